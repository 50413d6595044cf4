"""``experts`` benchmark: a layer of experts, operator by operator and whole.

A router sends each token to its top experts, every expert multiplies its
tokens by its two matrices (hidden = x W_up, out = hidden W_down, the second one
optionally with 4-bit weights), and the results are added up per token. The
reference has no such benchmark; its plugin interface, record fields and
metrics are the ones of its GEMM benchmark (src/teamredbench/benchmarks/mfu.py:33-181).

  params: backend ("native" only), dtypes (bfloat16, float16), layers: a list of
          {tokens, experts, top_k, k, n, group} (k: width of a token, n: width
          of the hidden row; group: with it W_down is 4-bit, one scale per group of n), warmup (10),
          iterations (50), seed (0), backward (default true where no layer is 4-bit), verify (default true),
          verify_max_tokens (default 64), operand_sets ("auto", or a count: the timed calls cycle through that
          many copies of the layer's buffers; "auto" takes enough that the smallest product bound by memory, by
          its arithmetic intensity, spans three times the 256 MB Infinity Cache, at most 1024 and half of the
          free memory)
  records, one per operator of a layer: case "experts_<operator>_t<tokens>e<experts>k<top_k>_<k>x<n>"
          with raw_metrics elapsed_s, achieved_ops / peak_tops and gemm_bytes for the products,
          moved_bytes / peak_bandwidth_gbps for the rest; operator "layer" is the whole forward pass. The
          backward operators are the gradients of the weighted sum, of the hidden rows, of W_up and of the
          logits (those of W_down and x are the same calls on other matrices).
          metadata: operand_sets, operand_footprint_bytes of the operator over all sets, cache_resident (they
          fit the Infinity Cache: the rate is the cache's, not HBM's) and parity, the in-run check after the timed
          calls, against torch on the same inputs: of the layer's output (records of the forward operators) or
          of the gradient itself, for up to verify_max_tokens tokens, and for W_up's gradient the experts
          with most and fewest rows. A record whose check fails is failed.

The calls go through libmi355bench.so (mb_route, mb_gemm_grouped, mb_gemm_w4,
mb_combine and their gradients) on torch's current stream; torch owns the memory.
"""
from __future__ import annotations

import copy
import itertools
from typing import Any

from teamredbench_amd.benchmarks.base import Benchmark, BenchmarkRecord
from teamredbench_amd.benchmarks.mfu import INFINITY_CACHE_BYTES, MAX_OPERAND_SETS, OPERAND_FOOTPRINT_TARGET
from teamredbench_amd.device import rocm_device_available
from teamredbench_amd.native import capi
from teamredbench_amd.parity import gemm_parity
from teamredbench_amd.registry import register_benchmark
from teamredbench_amd.utils import tensor_nbytes, timed_iterations

GRADIENTS = ("combine_grad", "rows_grad", "up_grad", "route_grad")
DEFAULT_LAYERS = [{"tokens": 4096, "experts": 16, "top_k": 4, "k": 4096, "n": 2048}]


class ExpertLayer:
    """The buffers of one layer and its operators' calls, forward and backward."""

    def __init__(self, torch: Any, lib: capi.NativeLibrary, dtype: str, layer: dict[str, int], device: Any, seed: int):
        self.torch, self.lib, self.dtype, self.dtype_name = torch, lib, capi.DTYPES[dtype], dtype
        self.tokens, self.experts, self.top_k, self.k, self.n = (
            int(layer[name]) for name in ("tokens", "experts", "top_k", "k", "n"))
        self.group = int(layer.get("group", 0))
        self.total = self.tokens * self.top_k
        self.stream = torch.cuda.current_stream(device).cuda_stream
        generator = torch.Generator(device=device).manual_seed(seed)
        half = getattr(torch, dtype)

        def normal(*shape: int, std: float = 1.0, of=half):
            return (torch.randn(*shape, generator=generator, device=device) * std).to(of)

        def empty(*shape: int, of=half):
            return torch.empty(*shape, device=device, dtype=of)

        tokens, experts, top_k, k, n, total = self.tokens, self.experts, self.top_k, self.k, self.n, self.total
        i32, f32 = torch.int32, torch.float32
        self.x, self.logits = normal(tokens, k), normal(tokens, experts, of=f32)
        self.up = torch.stack([normal(k, n, std=k**-0.5) for _ in range(experts)])
        if self.group:
            self.q = torch.randint(0, 256, (experts, k, (n + 1) // 2), generator=generator, device=device,
                                   dtype=torch.uint8)
            spread = torch.rand(experts, k, -(-n // self.group), generator=generator, device=device)
            self.scales = ((0.5 + spread) * (n**-0.5 / 4)).to(half)
        else:
            self.down = torch.stack([normal(n, k, std=n**-0.5) for _ in range(experts)])
        self.weights, self.ids = empty(tokens, top_k, of=f32), empty(tokens, top_k, of=i32)
        self.offsets, self.rows = empty(experts + 1, of=i32), empty(total, of=i32)
        self.slots = empty(tokens, top_k, of=i32)
        self.hidden, self.y, self.out = empty(total, n), empty(total, k), empty(tokens, k)
        self.workspace = empty(max(64 << 20, lib.route_workspace_size(tokens, experts, top_k)), of=torch.uint8)

    def prepare_backward(self) -> None:
        torch = self.torch
        self.grad_out = torch.randn_like(self.out)
        self.grad_y, self.grad_weights = torch.empty_like(self.y), torch.empty_like(self.weights)
        self.grad_hidden, self.grad_up = torch.empty_like(self.hidden), torch.empty_like(self.up)
        self.grad_logits = torch.empty_like(self.logits)

    def buffers(self) -> dict[str, Any]:
        """Every tensor of the layer but the workspace, by attribute."""
        return {name: value for name, value in vars(self).items()
                if isinstance(value, self.torch.Tensor) and name != "workspace"}

    def clone(self) -> "ExpertLayer":
        """The same layer on buffers of its own. The workspace, which no call leaves anything in, is shared."""
        other = copy.copy(self)
        for name, value in self.buffers().items():
            setattr(other, name, value.clone())
        return other

    def backward(self) -> None:
        for name in GRADIENTS:
            getattr(self, name)()

    def _workspace(self) -> tuple[int, int, int]:
        return self.workspace.data_ptr(), self.workspace.numel(), self.stream

    def route(self) -> None:
        self.lib.route(capi.DT_FLOAT32, self.logits.data_ptr(), 0, self.tokens, self.experts, self.top_k, True,
                       self.weights.data_ptr(), self.ids.data_ptr(), self.offsets.data_ptr(), self.rows.data_ptr(),
                       self.slots.data_ptr(), *self._workspace())

    def _grouped(self, op: int, x: Any, rows: Any, y: Any, out: Any, n: int, k: int) -> None:
        self.lib.gemm_grouped(op, self.dtype, x.data_ptr(), 0, x.shape[0], None if rows is None else rows.data_ptr(),
                              y.data_ptr(), 0, out.data_ptr(), 0, self.offsets.data_ptr(), self.experts, self.total,
                              n, k, *self._workspace())

    def up_product(self) -> None:
        self._grouped(capi.GROUPED_FORWARD, self.x, self.rows, self.up, self.hidden, self.n, self.k)

    def down_product(self) -> None:
        if not self.group:
            self._grouped(capi.GROUPED_FORWARD, self.hidden, None, self.down, self.y, self.k, self.n)
            return
        self.lib.gemm_w4(self.dtype, self.hidden.data_ptr(), 0, self.total, None, self.q.data_ptr(),
                         self.scales.data_ptr(), None, self.group, self.y.data_ptr(), 0, self.offsets.data_ptr(),
                         self.experts, self.total, self.k, self.n, *self._workspace())

    def combine(self) -> None:
        self.lib.combine(self.dtype, self.y.data_ptr(), 0, self.total, self.weights.data_ptr(), self.slots.data_ptr(),
                         self.tokens, self.top_k, self.k, self.out.data_ptr(), 0, self.stream)

    def forward(self) -> None:
        self.route()
        self.up_product()
        self.down_product()
        self.combine()

    def combine_grad(self) -> None:
        self.lib.combine_grad(self.dtype, self.grad_out.data_ptr(), 0, self.y.data_ptr(), 0, self.total,
                              self.weights.data_ptr(), self.slots.data_ptr(), self.tokens, self.top_k, self.k,
                              self.grad_y.data_ptr(), 0, self.grad_weights.data_ptr(), self.stream)

    def rows_grad(self) -> None:
        self._grouped(capi.GROUPED_GRAD_ROWS, self.grad_y, None, self.down, self.grad_hidden, self.k, self.n)

    def up_grad(self) -> None:
        self._grouped(capi.GROUPED_GRAD_WEIGHTS, self.x, self.rows, self.grad_hidden, self.grad_up, self.n, self.k)

    def route_grad(self) -> None:
        self.lib.route_grad(capi.DT_FLOAT32, self.logits.data_ptr(), 0, self.ids.data_ptr(),
                            self.grad_weights.data_ptr(), self.tokens, self.experts, self.top_k, True,
                            self.grad_logits.data_ptr(), 0, self.stream)

    def expected(self, tokens: int) -> Any:
        """The layer's output of the first `tokens` tokens by fp32 torch products, expert by expert."""
        torch = self.torch
        chosen, ids = torch.topk(self.logits[:tokens], self.top_k, dim=1)
        weights = torch.softmax(chosen, dim=1)
        out = torch.zeros(tokens, self.k, device=self.x.device)
        for e in range(self.experts):
            token, j = torch.nonzero(ids == e, as_tuple=True)
            if not token.numel():
                continue
            if self.group:
                q = torch.stack([self.q[e] & 15, self.q[e] >> 4], dim=-1).flatten(1)[:, :self.n].float() - 8.0
                scales = self.scales[e].float().repeat_interleave(self.group, 1)[:, :self.n]
                down = (q * scales).t()
            else:
                down = self.down[e].float()
            hidden = (self.x[token].float() @ self.up[e].float()).to(self.hidden.dtype).float()
            out.index_add_(0, token, weights[token, j, None] * (hidden @ down))
        return out


    # ---- checks: each gradient from the buffers its call read, in 64 bits (fp32 for a whole matrix) -------------
    def _sample(self, tokens: int) -> tuple[Any, Any, Any]:
        """The first tokens' assignments: token, choice and sorted row of each."""
        token, choice = self.torch.nonzero(self.slots[:tokens] >= 0, as_tuple=True)
        return token, choice, self.slots[token, choice].long()

    def check_forward(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        """Output name -> (dtype, what was computed, what it should be)."""
        return {"out": (self.dtype_name, self.out[:tokens].float(), self.expected(tokens))}

    def check_combine_grad(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        token, choice, row = self._sample(tokens)
        grad = self.grad_out[token].double()
        return {"grad_y": (self.dtype_name, self.grad_y[row], self.weights[token, choice, None].double() * grad),
                "grad_weights": ("float32", self.grad_weights[token, choice], (grad * self.y[row].double()).sum(1))}

    def check_rows_grad(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        token, choice, row = self._sample(tokens)
        expert = self.ids[token, choice]
        wanted = self.torch.empty(row.numel(), self.n, device=row.device)
        for e in expert.unique().tolist():
            at = expert == e
            wanted[at] = self.grad_y[row[at]].float() @ self.down[e].float().t().contiguous()
        return {"grad_hidden": (self.dtype_name, self.grad_hidden[row], wanted)}

    def check_up_grad(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        counts = self.offsets.diff()
        checked = {}
        for name, e in (("most", int(counts.argmax())), ("fewest", int(counts.argmin()))):
            lo, hi = int(self.offsets[e]), int(self.offsets[e + 1])
            x = self.x[self.rows[lo:hi].long()].float()
            checked[f"grad_up of the expert with {name} rows"] = (
                self.dtype_name, self.grad_up[e], x.t().contiguous() @ self.grad_hidden[lo:hi].float())
        return checked

    def check_route_grad(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        ids = self.ids[:tokens].long()
        chosen = self.torch.softmax(self.logits[:tokens].double().gather(1, ids), dim=1)
        g = self.grad_weights[:tokens].double()
        part = chosen * (g - (chosen * g).sum(1, keepdim=True))
        wanted = self.torch.zeros(tokens, self.experts, dtype=part.dtype, device=part.device).scatter_(1, ids, part)
        return {"grad_logits": ("float32", self.grad_logits[:tokens], wanted)}


def _bytes(work: dict[str, int]) -> int:
    return work.get("gemm_bytes", 0) or work.get("moved_bytes", 0)


def parity_of(torch: Any, checked: dict[str, tuple[str, Any, Any]]) -> dict[str, Any]:
    """The parity of the output that is nearest to its bound, or furthest over it, and every output's distance."""
    each = {name: gemm_parity(torch, dtype, got, want) if torch.count_nonzero(want) else
            {"rel_frobenius": 0.0, "bound": 0.0, "passed": not torch.count_nonzero(got)}
            for name, (dtype, got, want) in checked.items()}
    worst = max(each.values(), key=lambda p: (not p["passed"], p["rel_frobenius"] / p["bound"] if p["bound"] else 0.0))
    return {"vs": "torch", **{key: worst[key] for key in ("rel_frobenius", "bound")},
            "passed": all(p["passed"] for p in each.values()),
            "outputs": {name: p["rel_frobenius"] for name, p in each.items()}}


@register_benchmark("experts")
class ExpertsBenchmark(Benchmark):
    default_metrics = ["latency_us", "achieved_tops", "mfu_pct", "hbm_bandwidth_gbps", "gemm_bandwidth_gbps"]

    def _operators(self, layer: ExpertLayer, size: int, backward: bool) -> list[tuple[str, str, dict]]:
        """(name, the layer's method, what it computes and moves) of each operator, inputs read once and outputs
        written once."""
        tokens, experts, total, k, n = layer.tokens, layer.experts, layer.total, layer.k, layer.n
        hit = min(experts, total)
        product = {"achieved_ops": 2 * total * k * n}
        matrix = hit * k * n * size
        down = hit * k * ((n + 1) // 2 + -(-n // layer.group) * size) if layer.group else matrix
        assignments = total * 16 + (experts + 1) * 4
        operators = [
            ("route", "route", {"moved_bytes": tokens * experts * 4 + assignments}),
            ("up", "up_product", {**product, "gemm_bytes": matrix + (tokens * k + total * n) * size}),
            ("down", "down_product", {**product, "gemm_bytes": down + total * (n + k) * size}),
            ("combine", "combine", {"moved_bytes": (total + tokens) * k * size + total * 8}),
        ]
        moved = sum(_bytes(work) for _, _, work in operators)
        operators.append(("layer", "forward", {"achieved_ops": 4 * total * k * n, "gemm_bytes": moved}))
        if backward:
            operators += [
                ("combine_grad", "combine_grad", {"moved_bytes": (2 * total + tokens) * k * size + total * 12}),
                ("rows_grad", "rows_grad", {**product, "gemm_bytes": matrix + total * (n + k) * size}),
                ("up_grad", "up_grad",
                 {**product, "gemm_bytes": experts * k * n * size + (tokens * k + total * n) * size}),
                ("route_grad", "route_grad", {"moved_bytes": 2 * tokens * experts * 4 + total * 8}),
            ]
        return operators

    def _operand_sets(self, operators: list[tuple[str, str, dict]], peak_tops: float | None, set_bytes: int,
                      free_bytes: int) -> int:
        """Copies of the layer to cycle through (see the module's operand_sets)."""
        requested = self.params.get("operand_sets", "auto")
        if requested != "auto":
            return max(1, int(requested))
        hbm = self.context.hardware_profile.peak_hbm_bandwidth_gbps
        if not peak_tops or not hbm:
            return 1
        ridge = peak_tops * 1e12 / (hbm * 1e9)
        bound = [work["gemm_bytes"] for name, _, work in operators
                 if name != "layer" and "gemm_bytes" in work and work["achieved_ops"] < ridge * work["gemm_bytes"]]
        if not bound:
            return 1
        sets = -(-OPERAND_FOOTPRINT_TARGET // min(bound))
        return max(1, min(sets, MAX_OPERAND_SETS, free_bytes // 2 // set_bytes))

    def _cases(self, lib, torch, spec, shape: dict[str, int], peak_tops) -> list[BenchmarkRecord]:
        peak_hbm = self.context.hardware_profile.peak_hbm_bandwidth_gbps
        warmup, iterations = int(self.params.get("warmup", 10)), int(self.params.get("iterations", 50))
        layer = ExpertLayer(torch, lib, spec.name, shape, self.device, int(self.params.get("seed", 0)))
        backward = bool(self.params.get("backward", True)) and not layer.group
        layer.forward()
        if backward:
            layer.prepare_backward()
            layer.backward()
        suffix = f"t{layer.tokens}e{layer.experts}k{layer.top_k}_{layer.k}x{layer.n}"
        operators = self._operators(layer, spec.bytes_per_element, backward)
        set_bytes = sum(tensor_nbytes(value) for value in layer.buffers().values())
        sets = self._operand_sets(operators, peak_tops, set_bytes, torch.cuda.mem_get_info(self.device)[0])
        layers = [layer, *(layer.clone() for _ in range(sets - 1))]
        times = {}
        for name, method, _ in operators:
            calls = itertools.cycle([getattr(one, method) for one in layers])
            times[name] = timed_iterations(lambda: next(calls)(), torch_module=torch, warmup=warmup,
                                           iterations=iterations)
        del layers, calls
        rows = min(layer.tokens, int(self.params.get("verify_max_tokens", 64)))
        parity: dict[str, dict[str, Any]] = {}
        if bool(self.params.get("verify", True)):
            for name in ("forward", *(GRADIENTS if backward else ())):
                checked = getattr(layer, f"check_{name}")(rows)
                parity[name] = {**parity_of(torch, checked), "rows_checked": rows}
        records = []
        for name, _, work in operators:
            metadata = {"backend": "native", "kernel": "experts_gfx950", "operator": name, "timing": "wall_clock",
                        "operand_sets": sets, "operand_footprint_bytes": sets * _bytes(work),
                        "cache_resident": sets * _bytes(work) <= INFINITY_CACHE_BYTES,
                        **{key: int(value) for key, value in shape.items()}}
            check = name if name in GRADIENTS else "forward"
            if check in parity:
                metadata["parity"] = parity[check]
            raw = {"elapsed_s": times[name], **work}
            if "achieved_ops" in work:
                raw["peak_tops"] = peak_tops
            if "moved_bytes" in work:
                raw["peak_bandwidth_gbps"] = peak_hbm
            records.append(self.measured(case=f"experts_{name}_{suffix}", dtype=spec.name, raw_metrics=raw,
                                         metadata=metadata))
        return records

    def run(self) -> list[BenchmarkRecord]:
        backend = str(self.params.get("backend", "native")).lower()
        if backend != "native":
            raise KeyError(f"Unknown experts backend: {backend}")
        layers = [dict(layer) for layer in self.params.get("layers", DEFAULT_LAYERS)]
        specs = self.selected_dtype_specs()
        torch = self.context.torch_module
        why, lib = None, None
        try:
            lib = capi.load_library()
        except capi.NativeLibraryError as exc:
            why = str(exc)
        if why is None and not rocm_device_available(torch):
            why = "No ROCm device visible to PyTorch."
        if why is None:
            self.set_device()
        records: list[BenchmarkRecord] = []
        for spec in specs:
            peak_tops = self.context.hardware_profile.peak_compute_tops.get(spec.name)
            for shape in layers:
                case = "experts_" + "_".join(f"{key}{value}" for key, value in shape.items())
                unsupported = spec.name not in capi.EXPERT_DTYPES
                if why is not None or unsupported:
                    error = why or f"unsupported dtype for the expert layer: {spec.name}"
                    records.append(self.skip(case=case, dtype=spec.name, error=error, metadata={"backend": "native"}))
                    continue
                try:
                    records += self._cases(lib, torch, spec, shape, peak_tops)
                except (capi.NativeLibraryError, RuntimeError) as exc:
                    records.append(self.skip(case=case, dtype=spec.name, error=str(exc),
                                             metadata={"backend": "native"}))
                finally:
                    torch.cuda.empty_cache()
        return records
