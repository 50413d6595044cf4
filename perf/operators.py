"""The operators of an expert layer, as cases to measure.

A layer of experts sends each token to the experts that a router chooses,
multiplies the tokens of every expert by that expert's matrix, and adds the
results up per token:

  route    logits -> the top experts of each token, their softmax weights, and
           the assignments sorted by expert (and the logits' gradient)
  grouped  products of ragged groups of rows, one matrix per group: forward, and
           backward with the gradients of the rows and of the matrices
  w4       the same product with 4-bit weights, one scale (and zero point) per
           group of K; with one matrix it is the dense product of a decode step
  combine  the weighted sum of each token's expert rows (and its gradients)

`own` chooses between the framework's kernels (the C ABI through
teamredbench_amd.native.capi) and the same operators in elementary torch
operations. Inputs are normal; expert loads are uneven, as a router's are.

  listed()               the fixed cases
  draw(rng)              one more case of the same ranges
  prepare(case, seed)    inputs, outputs, workspace
  run(state)             one pass; returns its outputs
  work(case)             bytes and operations it cannot do without
  exact(case, seed)      the outputs in 64 bits
"""
from __future__ import annotations

import functools

import numpy as np
import torch

own = False

BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
WORKSPACE_BYTES = 64 << 20     # the scratch a program keeps for all of these calls
FORWARD, GRAD_ROWS, GRAD_WEIGHTS = 0, 1, 2

MOST_FLOPS = 2 * 16384 * 4096 * 14336     # the largest listed product
MOST_WEIGHTS = 1 << 29                    # matrix elements of all experts together


def _route(name, tokens, experts, top_k, dtype, normalize, backward, padded):
    """`padded`: the share of tokens whose logits are all -inf (batch padding)."""
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "normalize": normalize, "backward": backward, "padded": padded}


def _grouped(name, tokens, top_k, experts, k, n, dtype, backward):
    return {"name": name, "kind": "grouped", "tokens": tokens, "top_k": top_k, "experts": experts, "k": k, "n": n,
            "dtype": dtype, "backward": backward}


def _w4(name, tokens, top_k, experts, k, n, group, dtype, zeros):
    return {"name": name, "kind": "w4", "tokens": tokens, "top_k": top_k, "experts": experts, "k": k, "n": n,
            "group": group, "dtype": dtype, "zeros": zeros}


def _combine(name, tokens, top_k, n, dtype, backward):
    return {"name": name, "kind": "combine", "tokens": tokens, "top_k": top_k, "n": n, "dtype": dtype,
            "backward": backward}


def listed() -> list[dict]:
    return [
        # A decode step's router: few tokens, latency alone.
        _route("route_decode_32", 32, 32, 4, "float32", True, False, 0.0),
        # A training step's router over a long padded batch, with its gradient.
        _route("route_train_16384", 16384, 128, 8, "bfloat16", False, True, 0.05),
        # Decode: every expert multiplies a few rows, so its matrix's bytes are what counts.
        _grouped("grouped_decode_32", 32, 4, 32, 4096, 2048, "bfloat16", False),
        # Prefill of a long prompt with wide experts: matrix cores alone.
        _grouped("grouped_prefill_8192", 8192, 2, 8, 4096, 14336, "bfloat16", False),
        # Many small experts, sizes off every tile, in fp16.
        _grouped("grouped_ragged_3001", 3001, 4, 60, 2056, 1416, "float16", False),
        # A training step's backward pass: both gradients.
        _grouped("grouped_backward_4096", 4096, 4, 16, 4096, 2048, "bfloat16", True),
        # One token through a dense 4-bit projection.
        _w4("w4_1x14336x4096", 1, 1, 1, 4096, 14336, 128, "bfloat16", False),
        # A batch of 16 tokens, zero points, small groups.
        _w4("w4_16x8192x8192", 16, 1, 1, 8192, 8192, 32, "float16", True),
        # A batch of 64 tokens through a vocabulary head of odd size.
        _w4("w4_64x50257x4096", 64, 1, 1, 4096, 50257, 64, "bfloat16", True),
        # Decode through 4-bit experts.
        _w4("w4_experts_64", 64, 4, 64, 4096, 2048, 128, "bfloat16", False),
        # Decode: four rows added for each of 32 tokens.
        _combine("combine_decode_32", 32, 4, 4096, "bfloat16", False),
        # A training step: forward and both gradients.
        _combine("combine_train_8192", 8192, 4, 4096, "bfloat16", True),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return int(round(lo * (hi / lo) ** rng.random()))


def _grained(rng, lo: int, hi: int) -> int:
    """Mostly multiples of 64 or 8; one in eight is odd."""
    v = _log_uniform(rng, lo, hi)
    grain = rng.choice((256, 64, 64, 64, 8, 8, 8, 1))
    return max(lo, v - v % grain) if grain > 1 else v | 1


def draw(rng) -> dict:
    kind = rng.choice(("route", "grouped", "grouped", "w4", "w4", "combine"))
    half = rng.choice(("bfloat16", "float16"))
    top_k = rng.randint(1, 8)
    if kind == "route":
        experts = _log_uniform(rng, 4, 256)
        case = _route("", _log_uniform(rng, 1, 16384), experts, min(top_k, experts),
                      rng.choice(("float32", "bfloat16", "float16")), rng.random() < 0.5, rng.random() < 0.5,
                      rng.choice((0.0, 0.1)))
    elif kind == "grouped":
        experts = _log_uniform(rng, 2, 64)
        k = _grained(rng, 256, 8192)
        n = _grained(rng, 256, max(256, min(14336, MOST_WEIGHTS // (experts * k))))
        top_k = min(top_k, experts)
        backward = rng.random() < 0.4
        most = MOST_FLOPS // (2 * k * n * (2 if backward else 1)) // top_k
        case = _grouped("", _log_uniform(rng, 1, max(1, min(8192, most))), top_k, experts, k, n, half, backward)
    elif kind == "w4":
        experts = rng.choice((1, 1, _log_uniform(rng, 2, 64)))
        k = 2 * _grained(rng, 256, 7168)
        n = _grained(rng, 256, max(256, min(32768, MOST_WEIGHTS // (experts * k))))
        case = _w4("", _log_uniform(rng, 1, 64), min(top_k, experts), experts, k, n, rng.choice((32, 64, 128)), half,
                   rng.random() < 0.5)
    else:
        case = _combine("", _log_uniform(rng, 1, 8192), min(top_k, 4), _grained(rng, 256, 4096), half,
                        rng.random() < 0.5)
    del case["name"]
    return case


# ---- one case ---------------------------------------------------------------

def _assignments(case: dict, g: torch.Generator) -> dict:
    """A router's choices with uneven loads: offsets (E + 1) and rows (R), int32, and the most rows of an expert."""
    tokens, k, experts = case["tokens"], case["top_k"], case["experts"]
    score = torch.randn(tokens, experts, generator=g, device="cuda")
    score += 0.3 * torch.randn(experts, generator=g, device="cuda")
    chosen = torch.topk(score, k, dim=1).indices.reshape(-1)
    by_expert, order = torch.sort(chosen, stable=True)
    offsets = torch.searchsorted(by_expert, torch.arange(experts + 1, device="cuda"))
    return {"offsets": offsets.to(torch.int32), "rows": (order // k).to(torch.int32),
            "longest": int(offsets.diff().max())}


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=None, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype or getattr(torch, case["dtype"]))

    def empty(*shape, dtype=None):
        return torch.zeros(*shape, dtype=dtype or getattr(torch, case["dtype"]), device="cuda")

    state = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    kind, tokens, top_k = case["kind"], case["tokens"], case["top_k"]
    if kind != "combine":
        state["workspace"] = empty(WORKSPACE_BYTES, dtype=torch.uint8)
    total = tokens * top_k
    if kind == "route":
        experts = case["experts"]
        logits = normal(tokens, experts)
        padded = int(case["padded"] * tokens)
        if padded:
            logits[tokens - padded:] = -torch.inf
        state.update(logits=logits, weights=empty(tokens, top_k, dtype=torch.float32),
                     ids=empty(tokens, top_k, dtype=torch.int32), offsets=empty(experts + 1, dtype=torch.int32),
                     rows=empty(total, dtype=torch.int32), slots=empty(tokens, top_k, dtype=torch.int32))
        if case["backward"]:
            state.update(grad_weights=normal(tokens, top_k, dtype=torch.float32), grad_logits=empty(tokens, experts))
        return state
    n = case["n"]
    if kind == "combine":
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        weights = torch.softmax(torch.randn(tokens, top_k, generator=g, device="cuda"), dim=1)
        state.update(y=normal(total, n), weights=weights, slots=order.view(tokens, top_k), out=empty(tokens, n))
        if case["backward"]:
            state.update(grad_out=normal(tokens, n), grad_y=empty(total, n),
                         grad_weights=empty(tokens, top_k, dtype=torch.float32))
        return state
    experts, k = case["experts"], case["k"]
    state["x"] = normal(tokens, k)
    if experts > 1:
        state.update(_assignments(case, g))
    if kind == "grouped":
        b = torch.empty(experts, k, n, dtype=getattr(torch, case["dtype"]), device="cuda")
        for e in range(experts):
            b[e] = normal(k, n, std=k ** -0.5)
        state["b"] = b
        if case["backward"]:
            state.update(grad_out=normal(total, n), grad_x=empty(total, k), grad_b=empty(experts, k, n))
        else:
            state["out"] = empty(total, n)
        return state
    groups = -(-k // case["group"])
    state["q"] = torch.randint(0, 256, (experts, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = 0.5 + torch.rand(experts, n, groups, generator=g, device="cuda")
    state["scales"] = (scales * (0.25 * k ** -0.5)).to(getattr(torch, case["dtype"]))
    if case["zeros"]:
        zeros = torch.randint(6, 11, (experts, n, groups), generator=g, device="cuda")
        state["zeros"] = zeros.to(getattr(torch, case["dtype"]))
    state["out"] = empty(total, n)
    return state


def run(state: dict):
    kind = state["case"]["kind"]
    return (_OWN if own else _PLAIN)[kind](state)


# ---- the framework's calls ----------------------------------------------------

@functools.cache
def _library():
    from teamredbench_amd.native import capi

    return capi.load_library(), capi.DTYPES


def _pointer(state: dict, name: str):
    return state[name].data_ptr() if name in state else None


def _own_route(s: dict):
    lib, dtypes = _library()
    c = s["case"]
    tokens, experts, top_k, dtype = c["tokens"], c["experts"], c["top_k"], dtypes[c["dtype"]]
    lib.route(dtype, s["logits"].data_ptr(), experts, tokens, experts, top_k, c["normalize"], s["weights"].data_ptr(),
              s["ids"].data_ptr(), s["offsets"].data_ptr(), s["rows"].data_ptr(), s["slots"].data_ptr(),
              s["workspace"].data_ptr(), WORKSPACE_BYTES, s["stream"])
    out = [s["weights"], s["ids"], s["offsets"], s["rows"], s["slots"]]
    if c["backward"]:
        lib.route_grad(dtype, s["logits"].data_ptr(), experts, s["ids"].data_ptr(), s["grad_weights"].data_ptr(),
                       tokens, experts, top_k, c["normalize"], s["grad_logits"].data_ptr(), experts, s["stream"])
        out.append(s["grad_logits"])
    return out


def _own_grouped(s: dict):
    lib, dtypes = _library()
    c = s["case"]
    tokens, experts, k, n, dtype = c["tokens"], c["experts"], c["k"], c["n"], dtypes[c["dtype"]]
    total = tokens * c["top_k"]
    offsets, rows, x, b = (s[name].data_ptr() for name in ("offsets", "rows", "x", "b"))
    rest = (total, n, k, s["workspace"].data_ptr(), WORKSPACE_BYTES, s["stream"])
    if not c["backward"]:
        lib.gemm_grouped(FORWARD, dtype, x, k, tokens, rows, b, n, s["out"].data_ptr(), n, offsets, experts, *rest)
        return s["out"]
    grad = s["grad_out"].data_ptr()
    lib.gemm_grouped(GRAD_ROWS, dtype, grad, n, total, None, b, n, s["grad_x"].data_ptr(), k, offsets, experts, *rest)
    lib.gemm_grouped(GRAD_WEIGHTS, dtype, x, k, tokens, rows, grad, n, s["grad_b"].data_ptr(), n, offsets, experts,
                     *rest)
    return [s["grad_x"], s["grad_b"]]


def _own_w4(s: dict):
    lib, dtypes = _library()
    c = s["case"]
    lib.gemm_w4(dtypes[c["dtype"]], s["x"].data_ptr(), c["k"], c["tokens"], _pointer(s, "rows"), s["q"].data_ptr(),
                s["scales"].data_ptr(), _pointer(s, "zeros"), c["group"], s["out"].data_ptr(), c["n"],
                _pointer(s, "offsets"), c["experts"], c["tokens"] * c["top_k"], c["n"], c["k"],
                s["workspace"].data_ptr(), WORKSPACE_BYTES, s["stream"])
    return s["out"]


def _own_combine(s: dict):
    lib, dtypes = _library()
    c = s["case"]
    tokens, top_k, n, dtype = c["tokens"], c["top_k"], c["n"], dtypes[c["dtype"]]
    total = tokens * top_k
    y, weights, slots = s["y"].data_ptr(), s["weights"].data_ptr(), s["slots"].data_ptr()
    lib.combine(dtype, y, n, total, weights, slots, tokens, top_k, n, s["out"].data_ptr(), n, s["stream"])
    if not c["backward"]:
        return s["out"]
    lib.combine_grad(dtype, s["grad_out"].data_ptr(), n, y, n, total, weights, slots, tokens, top_k, n,
                     s["grad_y"].data_ptr(), n, s["grad_weights"].data_ptr(), s["stream"])
    return [s["out"], s["grad_y"], s["grad_weights"]]


_OWN = {"route": _own_route, "grouped": _own_grouped, "w4": _own_w4, "combine": _own_combine}


# ---- the plain form: elementary operations in 32 bits ---------------------------

def _plain_route(s: dict):
    c = s["case"]
    experts, top_k = c["experts"], c["top_k"]
    logits = s["logits"].float()
    values, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    values, ids = values[:, :top_k], ids[:, :top_k]
    chosen = values > -torch.inf
    top = torch.where(chosen[:, :1], values[:, :1], 0.0)
    exps = torch.exp(values - top)
    total = exps.sum(1, keepdim=True) if c["normalize"] else torch.exp(logits - top).sum(1, keepdim=True)
    total = torch.where(chosen[:, :1], total, 1.0)
    weights = exps / total
    key = torch.where(chosen, ids, experts).reshape(-1)
    by_expert, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(by_expert, torch.arange(experts + 1, device=key.device))
    rows = torch.where(by_expert < experts, order // top_k, -1)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(key.numel(), device=key.device)
    slots = torch.where(key < experts, slots, -1).view_as(ids)
    out = [weights, torch.where(chosen, ids, -1).int(), offsets.int(), rows.int(), slots.int()]
    if c["backward"]:
        part = weights * s["grad_weights"]
        mean = part.sum(1, keepdim=True)
        if c["normalize"]:
            grad = torch.zeros_like(logits).scatter_add(1, ids, part - weights * mean)
        else:
            grad = (-(torch.exp(logits - top) / total) * mean).scatter_add(1, ids, part)
        out.append(grad.to(s["logits"].dtype))
    return out


def _padded(s: dict):
    """(E, P) row numbers of each expert's rows, R where it has no more, and each row's place among them."""
    c = s["case"]
    total, longest = c["tokens"] * c["top_k"], s["longest"]
    offsets = s["offsets"].long()
    at = offsets[:-1, None] + torch.arange(longest, device=offsets.device)
    at = torch.where(at < offsets[1:, None], at, total)
    row = torch.arange(total, device=offsets.device)
    expert = torch.searchsorted(offsets, row, right=True) - 1
    return at, expert * longest + row - offsets[expert]


def _with_zero_row(x: torch.Tensor) -> torch.Tensor:
    return torch.cat([x, x.new_zeros(1, x.shape[1])])


def _plain_grouped(s: dict):
    at, place = _padded(s)
    x = _with_zero_row(s["x"].float()[s["rows"].long()])[at]
    b = s["b"].float()
    if not s["case"]["backward"]:
        return torch.bmm(x, b).flatten(0, 1)[place].to(s["b"].dtype)
    grad = _with_zero_row(s["grad_out"].float())[at]
    grad_x = torch.bmm(grad, b.transpose(1, 2)).flatten(0, 1)[place]
    return [grad_x.to(s["b"].dtype), torch.bmm(x.transpose(1, 2), grad).to(s["b"].dtype)]


def _plain_w4(s: dict):
    c = s["case"]
    low, high = s["q"] & 15, s["q"] >> 4
    q = torch.stack([low, high], dim=-1).flatten(2).float()
    spread = torch.arange(c["k"], device=q.device) // c["group"]
    zeros = s["zeros"].float()[:, :, spread] if c["zeros"] else 8.0
    b = ((q - zeros) * s["scales"].float()[:, :, spread]).transpose(1, 2)
    x = s["x"].float()
    if c["experts"] == 1:
        return torch.matmul(x, b[0]).to(s["x"].dtype)
    at, place = _padded(s)
    return torch.bmm(_with_zero_row(x[s["rows"].long()])[at], b).flatten(0, 1)[place].to(s["x"].dtype)


def _plain_combine(s: dict):
    slots, weights = s["slots"].long(), s["weights"]
    y = s["y"].float()[slots]
    out = (weights[:, :, None] * y).sum(1).to(s["y"].dtype)
    if not s["case"]["backward"]:
        return out
    grad = s["grad_out"].float()[:, None, :]
    grad_y = torch.zeros_like(s["y"])
    grad_y[slots] = (weights[:, :, None] * grad).to(grad_y.dtype)
    return [out, grad_y, (grad * y).sum(2)]


_PLAIN = {"route": _plain_route, "grouped": _plain_grouped, "w4": _plain_w4, "combine": _plain_combine}


# ---- what a pass cannot do without ------------------------------------------------

def work(case: dict) -> dict:
    size, tokens, top_k = BYTES[case["dtype"]], case["tokens"], case["top_k"]
    total = tokens * top_k
    if case["kind"] == "route":
        logits = tokens * case["experts"] * size
        out = total * 16 + (case["experts"] + 1) * 4
        return {"bytes": logits + out + (logits + total * 4 if case["backward"] else 0),
                "flops": 4 * tokens * case["experts"]}
    n = case["n"]
    if case["kind"] == "combine":
        forward = (total + tokens) * n * size + total * 8
        backward = (total + tokens) * n * size + total * 4
        return {"bytes": forward + (backward if case["backward"] else 0),
                "flops": 2 * total * n * (3 if case["backward"] else 1)}
    experts, k = case["experts"], case["k"]
    hit = min(experts, total)    # experts with rows, at most
    if case["kind"] == "w4":
        groups = -(-k // case["group"])
        weights = hit * n * (k // 2 + groups * size * (2 if case["zeros"] else 1))
        return {"bytes": weights + (tokens * k + total * n) * size, "flops": 2 * total * n * k}
    if not case["backward"]:
        return {"bytes": (hit * k * n + tokens * k + total * n) * size, "flops": 2 * total * n * k}
    return {"bytes": (hit * k * n + experts * k * n + tokens * k + total * (n + k)) * size,
            "flops": 4 * total * n * k}


# ---- the definition in 64 bits ------------------------------------------------------

def _exact_route(case: dict, s: dict):
    logits = s["logits"].double().cpu().numpy()
    tokens, experts = logits.shape
    top_k = case["top_k"]
    order = np.argsort(-logits, axis=1, kind="stable")[:, :top_k]
    weights, slots = np.zeros((tokens, top_k)), np.full((tokens, top_k), -1, np.int32)
    ids = order.astype(np.int32)
    picked = np.take_along_axis(logits, order, 1)
    live = np.isfinite(picked)
    ids[~live] = -1
    some = live[:, 0]
    shifted = np.exp(logits[some] - picked[some, :1])
    top = np.take_along_axis(shifted, order[some], 1)
    over = top.sum(1) if case["normalize"] else shifted.sum(1)
    weights[some] = top / over[:, None]
    offsets, rows = np.zeros(experts + 1, np.int32), np.full(tokens * top_k, -1, np.int32)
    for e in range(experts):
        token, j = np.nonzero(ids == e)
        offsets[e + 1] = offsets[e] + len(token)
        rows[offsets[e]:offsets[e + 1]] = token
        slots[token, j] = np.arange(offsets[e], offsets[e + 1])
    out = [weights, ids, offsets, rows, slots]
    if case["backward"]:
        g = s["grad_weights"].double().cpu().numpy()[some]
        grad = np.zeros((tokens, experts))
        mean = (weights[some] * g).sum(1)[:, None]
        p = np.zeros_like(shifted)
        if case["normalize"]:
            np.put_along_axis(p, order[some], weights[some], 1)
        else:
            p = shifted / over[:, None]
        g_all = np.zeros_like(shifted)
        np.put_along_axis(g_all, order[some], g, 1)
        grad[some] = p * (g_all - mean)
        out.append(grad)
    return [torch.from_numpy(v) for v in out]


def _exact_grouped(case: dict, s: dict):
    b, rows, edges = s["b"], s["rows"].long(), s["offsets"].tolist()
    spans = list(zip(edges[:-1], edges[1:]))
    x = s["x"].double()
    if not case["backward"]:
        return torch.cat([x[rows[i:j]] @ b[e].double() for e, (i, j) in enumerate(spans)])
    grad = s["grad_out"].double()
    grad_x = torch.cat([grad[i:j] @ b[e].double().t() for e, (i, j) in enumerate(spans)])
    return [grad_x, torch.stack([x[rows[i:j]].t() @ grad[i:j] for i, j in spans])]


def _exact_w4(case: dict, s: dict):
    x, q, scales = s["x"].double(), s["q"], s["scales"].double()
    rows = s["rows"].long() if "rows" in s else torch.arange(case["tokens"], device=x.device)
    edges = s["offsets"].tolist() if "offsets" in s else [0, case["tokens"]]
    out, group = [], case["group"]
    for e, (i, j) in enumerate(zip(edges[:-1], edges[1:])):
        w = torch.empty(case["n"], case["k"], dtype=torch.float64, device=x.device)
        w[:, 0::2], w[:, 1::2] = (q[e] % 16).double(), (q[e] // 16).double()
        zero = s["zeros"][e].double().repeat_interleave(group, 1)[:, :case["k"]] if case["zeros"] else 8.0
        w = (w - zero) * scales[e].repeat_interleave(group, 1)[:, :case["k"]]
        out.append(x[rows[i:j]] @ w.t())
    return torch.cat(out)


def _exact_combine(case: dict, s: dict):
    y, w, slots = s["y"].double(), s["weights"].double(), s["slots"].long()
    out = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device=y.device)
    for j in range(case["top_k"]):
        out += w[:, j, None] * y[slots[:, j]]
    if not case["backward"]:
        return out
    grad, grad_y, grad_w = s["grad_out"].double(), torch.zeros_like(y), torch.zeros_like(w)
    for j in range(case["top_k"]):
        grad_y[slots[:, j]] = w[:, j, None] * grad
        grad_w[:, j] = torch.linalg.vecdot(grad, y[slots[:, j]])
    return [out, grad_y, grad_w]


_EXACT = {"route": _exact_route, "grouped": _exact_grouped, "w4": _exact_w4, "combine": _exact_combine}


def exact(case: dict, seed: int):
    return _EXACT[case["kind"]](case, prepare(case, seed))
