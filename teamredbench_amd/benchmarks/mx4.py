"""``mx4`` benchmark: a linear layer in microscaled 4-bit floats (MX4), operator by operator and whole.

The layer multiplies its tokens by a matrix of weights, or every expert its tokens by a matrix of its own. x and
w are quantised to MX4, and the products run on those forms, in the backward pass too: the
gradients contract over other axes, so x, w and the output's gradient are also quantised along
their columns, in the same pass. The reference has no such benchmark (its narrowest type is fp8,
src/teamredbench/dtypes.py:23-24); its plugin interface, record fields and metrics are the ones of its GEMM benchmark
(src/teamredbench/benchmarks/mfu.py:33-181).

  params: backend ("native" only), dtypes (bfloat16, float16: of x, w and the outputs), layers: a list of
          {tokens, k, n} (k inputs, n outputs), with {experts, top_k} a router sends each token to its top experts;
          scale_rule ("floor", or "fit": no element saturates), and warmup, iterations, seed, backward (default
          true, layers without experts), verify, verify_max_tokens and operand_sets as in the experts benchmark
  records, one per operator of a layer: case "mx4_<operator>_t<tokens>_<k>x<n>", or "mx4_<operator>_t<tokens>e<experts>
          k<top_k>_<k>x<n>", with raw_metrics elapsed_s, achieved_ops / peak_tops (the profile's "mx4") and
          gemm_bytes for the products, moved_bytes / peak_bandwidth_gbps for the rest; operator "layer" is the
          forward pass on weights that are quantised already.
          metadata as in the experts benchmark; parity compares quantisation with its definition and products with
          torch's on the quantised values.

The calls go through libmi355bench.so (mb_mx4_quantize, mb_mx4_dequantize, mb_gemm_mx4, mb_route) on torch's
current stream; torch owns the memory.
"""
from __future__ import annotations

from typing import Any

from teamredbench_amd.benchmarks.layers import Layer, LayerBenchmark, moved_or_product_bytes
from teamredbench_amd.native import capi
from teamredbench_amd.registry import register_benchmark

GRADIENTS = ("quantize_grad", "x_grad", "w_grad")
CHECKS = ("quantize_x", "quantize_w", "dequantize_w", *GRADIENTS)
DEFAULT_LAYERS = [{"tokens": 4096, "k": 4096, "n": 14336}]
SCALE_RULES = {"floor": capi.MX4_SCALE_FLOOR, "fit": capi.MX4_SCALE_FIT}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def values_of(torch: Any, q: Any, scales: Any, columns: int) -> Any:
    """What rows of MX4 stand for, fp32."""
    table = torch.tensor([*E2M1, *(-v for v in E2M1)], device=q.device)
    codes = torch.stack([q & 15, q >> 4], dim=-1).flatten(1).int()
    power = torch.exp2(scales.double() - 127).float().masked_fill(scales == 255, torch.nan)
    return (table[codes] * power.repeat_interleave(32, 1))[:, :columns]


def quantized_values(torch: Any, x: Any, rule: int) -> Any:
    """x (fp32, rows along the blocks, finite) rounded to MX4 by the definition, fp32."""
    rows, columns = x.shape
    blocks = torch.nn.functional.pad(x, (0, -columns % 32)).view(rows, -1, 32)
    most = blocks.abs().amax(2, keepdim=True)
    mantissa, exponent = torch.frexp(most)   # most = mantissa 2^exponent, mantissa in [1/2, 1)
    power = exponent - 3 + (mantissa > 0.75) * (rule == capi.MX4_SCALE_FIT)
    power = torch.where(most > 0, power, -127).clamp(min=-127).double()
    v = (blocks.abs() * torch.exp2(-power)).clamp(max=6.0)
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    rounded = torch.round(v / step) * step   # a tie's even multiple is the even code
    return (rounded * torch.exp2(power) * blocks.sign()).float().view(rows, -1)[:, :columns]


class Mx4Layer(Layer):
    """The buffers of one layer and its operators' calls, forward and backward."""

    def __init__(self, torch: Any, lib: capi.NativeLibrary, dtype: str, layer: dict[str, int], device: Any, seed: int,
                 rule: int = capi.MX4_SCALE_FLOOR):
        self.torch, self.lib, self.dtype, self.dtype_name, self.rule = torch, lib, capi.DTYPES[dtype], dtype, rule
        self.tokens, self.k, self.n = (int(layer[name]) for name in ("tokens", "k", "n"))
        self.experts, self.top_k = int(layer.get("experts", 0)), int(layer.get("top_k", 1))
        tokens, k, n, experts = self.tokens, self.k, self.n, self.experts
        self.total = tokens * self.top_k if experts else tokens
        self.differentiable = not experts
        self.suffix = f"t{tokens}e{experts}k{self.top_k}_{k}x{n}" if experts else f"t{tokens}_{k}x{n}"
        self.stream = torch.cuda.current_stream(device).cuda_stream
        generator = torch.Generator(device=device).manual_seed(seed)
        half, i32, f32 = getattr(torch, dtype), torch.int32, torch.float32

        def normal(*shape: int, std: float = 1.0, of=half):
            return (torch.randn(*shape, generator=generator, device=device) * std).to(of)

        def empty(*shape: int, of=half):
            return torch.empty(*shape, device=device, dtype=of)

        self.x, self.w = normal(tokens, k), normal(max(experts, 1) * n, k, std=k**-0.5)
        self.x_q, self.x_s = self._form(tokens, k)
        self.w_q, self.w_s = self._form(max(experts, 1) * n, k)
        self.w_values, self.out = torch.empty_like(self.w), empty(self.total, n)
        if experts:
            self.logits, self.weights = normal(tokens, experts, of=f32), empty(tokens, self.top_k, of=f32)
            self.ids, self.slots = empty(tokens, self.top_k, of=i32), empty(tokens, self.top_k, of=i32)
            self.offsets, self.rows = empty(experts + 1, of=i32), empty(self.total, of=i32)
        size = lib.route_workspace_size(tokens, experts, self.top_k) if experts else 0
        self.workspace = empty(max(64 << 20, size), of=torch.uint8)
        self.backward_forms = False
        self.quantize_w()

    def _form(self, rows: int, columns: int) -> tuple[Any, Any]:
        def empty(width: int):
            return self.torch.empty(rows, width, dtype=self.torch.uint8, device=self.x.device)

        return empty(capi.mx4_row_bytes(columns)), empty(capi.mx4_row_scales(columns))

    def prepare_backward(self) -> None:
        tokens, k, n = self.tokens, self.k, self.n
        self.grad = self.torch.randn_like(self.out)
        self.grad_q, self.grad_s = self._form(tokens, n)
        self.xt_q, self.xt_s = self._form(k, tokens)         # along x's columns, and so on
        self.wt_q, self.wt_s = self._form(k, n)
        self.gradt_q, self.gradt_s = self._form(n, tokens)
        self.grad_x, self.grad_w = self.torch.empty_like(self.x), self.torch.empty_like(self.w)
        self.backward_forms = True
        self.quantize_x()
        self.quantize_w()

    def _quantize(self, x: Any, name: str) -> None:
        rows, columns = x.shape
        forms = [getattr(self, f"{name}_{part}").data_ptr() for part in "qs"]
        if self.backward_forms:
            forms += [getattr(self, f"{name}t_{part}").data_ptr() for part in "qs"]
        else:
            forms += [None, None]
        self.lib.mx4_quantize(self.dtype, x.data_ptr(), 0, rows, columns, self.rule, *forms, self.stream)

    def quantize_x(self) -> None:
        self._quantize(self.x, "x")

    def quantize_w(self) -> None:
        self._quantize(self.w, "w")

    def quantize_grad(self) -> None:
        self._quantize(self.grad, "grad")

    def dequantize_w(self) -> None:
        self.lib.mx4_dequantize(self.dtype, self.w_q.data_ptr(), self.w_s.data_ptr(), self.w.shape[0], self.k,
                                self.w_values.data_ptr(), 0, self.stream)

    def _product(self, left: str, right: str, out: Any, k: int) -> None:
        """out = left right^T, over k."""
        a, a_scales, b, b_scales = (getattr(self, f"{name}_{part}") for name in (left, right) for part in "qs")
        routed = self.experts > 0
        self.lib.gemm_mx4(self.dtype, a.data_ptr(), a_scales.data_ptr(), a.shape[0],
                          self.rows.data_ptr() if routed else None, b.data_ptr(), b_scales.data_ptr(), out.data_ptr(),
                          0, self.offsets.data_ptr() if routed else None, max(self.experts, 1), out.shape[0],
                          out.shape[1], k, self.workspace.data_ptr(), self.workspace.numel(), self.stream)

    def route(self) -> None:
        self.lib.route(capi.DT_FLOAT32, self.logits.data_ptr(), 0, self.tokens, self.experts, self.top_k, True,
                       self.weights.data_ptr(), self.ids.data_ptr(), self.offsets.data_ptr(), self.rows.data_ptr(),
                       self.slots.data_ptr(), self.workspace.data_ptr(), self.workspace.numel(), self.stream)

    def product(self) -> None:
        self._product("x", "w", self.out, self.k)

    def forward(self) -> None:
        if self.experts:
            self.route()
        self.quantize_x()
        self.product()

    def x_grad(self) -> None:
        self._product("grad", "wt", self.grad_x, self.n)

    def w_grad(self) -> None:
        self._product("gradt", "xt", self.grad_w, self.tokens)

    def backward(self) -> None:
        for name in GRADIENTS:
            getattr(self, name)()

    # ---- checks: output name -> (dtype, what was computed, what it should be) ------------------------------------
    def _values(self, name: str, columns: int, rows: Any = slice(None)) -> Any:
        """What (rows of) a form stand for."""
        return values_of(self.torch, getattr(self, f"{name}_q")[rows], getattr(self, f"{name}_s")[rows], columns)

    def check_forward(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        if not self.experts:
            wanted = self._values("x", self.k, slice(0, tokens)) @ self._values("w", self.k).t()
            return {"out": (self.dtype_name, self.out[:tokens], wanted)}
        token, choice = self.torch.nonzero(self.slots[:tokens] >= 0, as_tuple=True)
        row, expert = self.slots[token, choice].long(), self.ids[token, choice]
        x, wanted = self._values("x", self.k, token), self.torch.empty(row.numel(), self.n, device=row.device)
        for e in expert.unique().tolist():
            at = expert == e
            wanted[at] = x[at] @ self._values("w", self.k, slice(e * self.n, (e + 1) * self.n)).t()
        return {"out": (self.dtype_name, self.out[row], wanted)}

    def _check_forms(self, x: Any, name: str, count: int) -> dict[str, tuple[str, Any, Any]]:
        rows, columns = x.shape
        checked = {name: ("float32", self._values(name, columns, slice(0, count)),
                          quantized_values(self.torch, x[:count].float(), self.rule))}
        if self.backward_forms:
            checked[f"{name} along its columns"] = (
                "float32", self._values(f"{name}t", rows, slice(0, count)),
                quantized_values(self.torch, x[:, :count].float().t().contiguous(), self.rule))
        return checked

    def check_quantize_x(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        return self._check_forms(self.x, "x", tokens)

    def check_quantize_w(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        return self._check_forms(self.w, "w", tokens)

    def check_quantize_grad(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        return self._check_forms(self.grad, "grad", tokens)

    def check_dequantize_w(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        return {"w": (self.dtype_name, self.w_values[:tokens], self._values("w", self.k, slice(0, tokens)))}

    def check_x_grad(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        wanted = self._values("grad", self.n, slice(0, tokens)) @ self._values("wt", self.n).t()
        return {"grad_x": (self.dtype_name, self.grad_x[:tokens], wanted)}

    def check_w_grad(self, tokens: int) -> dict[str, tuple[str, Any, Any]]:
        wanted = self._values("gradt", self.tokens, slice(0, tokens)) @ self._values("xt", self.tokens).t()
        return {"grad_w": (self.dtype_name, self.grad_w[:tokens], wanted)}


@register_benchmark("mx4")
class Mx4Benchmark(LayerBenchmark):
    default_layers, what = DEFAULT_LAYERS, "the MX4 layer"
    checks, gradients, peak_name = CHECKS, GRADIENTS, "mx4"

    def layer_type(self, *args: Any) -> Mx4Layer:
        rule = str(self.params.get("scale_rule", "floor")).lower()
        if rule not in SCALE_RULES:
            raise KeyError(f"Unknown mx4 scale_rule: {rule}")
        return Mx4Layer(*args, rule=SCALE_RULES[rule])

    def _operators(self, layer: Mx4Layer, size: int, backward: bool) -> list[tuple[str, str, dict]]:
        tokens, k, n, total, experts = layer.tokens, layer.k, layer.n, layer.total, layer.experts

        def form(rows: int, columns: int) -> int:
            return rows * (capi.mx4_row_bytes(columns) + capi.mx4_row_scales(columns))

        def quantize(rows: int, columns: int) -> dict:
            both = form(columns, rows) if backward else 0
            return {"moved_bytes": rows * columns * size + form(rows, columns) + both}

        def product(rows: int, columns: int, depth: int, matrix: int, inputs: int) -> dict:
            return {"achieved_ops": 2 * rows * columns * depth,
                    "gemm_bytes": matrix + form(inputs, depth) + rows * columns * size}

        w_rows = max(experts, 1) * n
        hit = min(experts, total) * n if experts else n   # rows of w that a forward product reads
        operators = []
        if experts:
            operators.append(("route", "route", {"moved_bytes": tokens * experts * 4 + total * 16 + (experts + 1) * 4}))
        operators += [("quantize_x", "quantize_x", quantize(tokens, k)),
                      ("product", "product", product(total, n, k, form(hit, k), tokens))]
        moved = sum(moved_or_product_bytes(work) for _, _, work in operators)
        operators += [("layer", "forward", {"achieved_ops": 2 * total * n * k, "gemm_bytes": moved}),
                      ("quantize_w", "quantize_w", quantize(w_rows, k)),
                      ("dequantize_w", "dequantize_w", {"moved_bytes": form(w_rows, k) + w_rows * k * size})]
        if backward:
            operators += [("quantize_grad", "quantize_grad", quantize(tokens, n)),
                          ("x_grad", "x_grad", product(tokens, k, n, form(k, n), tokens)),
                          ("w_grad", "w_grad", product(n, k, tokens, form(k, tokens), n))]
        return operators
