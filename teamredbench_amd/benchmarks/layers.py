"""A layer of operators benchmarked one by one and whole: what the ``experts`` and ``mx4`` benchmarks share.

A layer holds its buffers and makes each operator's call; the benchmark times the calls over copies of the layer,
checks their outputs in the run and writes one record per operator.
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
from teamredbench_amd.utils import tensor_nbytes, timed_iterations


class Layer:
    """Buffers as attributes; `forward`, `prepare_backward` and `backward`, a method for each operator, and for each
    check a method check_<name>(rows)."""

    suffix: str            # of the records' cases: the layer's sizes
    tokens: int
    differentiable = True  # has a backward pass

    def buffers(self) -> dict[str, Any]:
        """Every tensor of the layer but the workspace, by attribute."""
        return {name: value for name, value in vars(self).items()
                if isinstance(value, self.torch.Tensor) and name != "workspace"}

    def clone(self) -> "Layer":
        """The same layer on buffers of its own. The workspace, which no call leaves anything in, is shared."""
        other = copy.copy(self)
        for name, value in self.buffers().items():
            setattr(other, name, value.clone())
        return other


def moved_or_product_bytes(work: dict[str, int]) -> int:
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


class LayerBenchmark(Benchmark):
    default_metrics = ["latency_us", "achieved_tops", "mfu_pct", "hbm_bandwidth_gbps", "gemm_bandwidth_gbps"]
    layer_type: type[Layer]
    default_layers: list[dict]
    what = ""                            # in the error of a dtype that the layer does not take
    checks: tuple[str, ...] = ()         # operators with a check of their own; the others take "forward"
    gradients: tuple[str, ...] = ()      # those of them that need the backward pass
    peak_name: str | None = None         # the profile's peak of the products, where it is not the dtype's

    def _operators(self, layer: Any, size: int, backward: bool) -> list[tuple[str, str, dict]]:
        """(name, the layer's method, what it computes and moves) of each operator, inputs read once and outputs
        written once."""
        raise NotImplementedError

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

    def _sets_by_operator(self, operators: list[tuple[str, str, dict]], peak_tops: float | None, set_bytes: int,
                          free_bytes: int, calls: int) -> dict[str, int]:
        """Copies that each operator's calls cycle through: `_operand_sets` for the products and the whole layer. What only
        moves bytes takes more where that is short of the footprint of its own, since its rate is reported as
        HBM's: up to the number of its calls, where those pass the cache at all."""
        sets = self._operand_sets(operators, peak_tops, set_bytes, free_bytes)
        by_operator = {name: sets for name, _, _ in operators}
        if self.params.get("operand_sets", "auto") == "auto":
            for name, _, work in operators:
                if "gemm_bytes" not in work:
                    own = min(-(-OPERAND_FOOTPRINT_TARGET // work["moved_bytes"]), MAX_OPERAND_SETS, calls,
                              free_bytes // 2 // set_bytes)
                    if own * work["moved_bytes"] > INFINITY_CACHE_BYTES:
                        by_operator[name] = max(sets, own)
        return by_operator

    def _cases(self, lib, torch, spec, shape: dict[str, int], peak_tops) -> list[BenchmarkRecord]:
        peak_hbm = self.context.hardware_profile.peak_hbm_bandwidth_gbps
        warmup, iterations = int(self.params.get("warmup", 10)), int(self.params.get("iterations", 50))
        layer = self.layer_type(torch, lib, spec.name, shape, self.device, int(self.params.get("seed", 0)))
        backward = bool(self.params.get("backward", True)) and layer.differentiable
        layer.forward()
        if backward:
            layer.prepare_backward()
            layer.backward()
        operators = self._operators(layer, spec.bytes_per_element, backward)
        set_bytes = sum(tensor_nbytes(value) for value in layer.buffers().values())
        sets = self._sets_by_operator(operators, peak_tops, set_bytes, torch.cuda.mem_get_info(self.device)[0],
                                      max(warmup, 0) + max(iterations, 1))
        layers = [layer, *(layer.clone() for _ in range(max(sets.values()) - 1))]
        times = {}
        for name, method, _ in operators:
            calls = itertools.cycle([getattr(one, method) for one in layers[:sets[name]]])
            times[name] = timed_iterations(lambda: next(calls)(), torch_module=torch, warmup=warmup,
                                           iterations=iterations)
        del layers, calls
        rows = min(layer.tokens, int(self.params.get("verify_max_tokens", 64)))
        parity: dict[str, dict[str, Any]] = {}
        if bool(self.params.get("verify", True)):
            for name in ("forward", *(c for c in self.checks if backward or c not in self.gradients)):
                checked = getattr(layer, f"check_{name}")(rows)
                parity[name] = {**parity_of(torch, checked), "rows_checked": rows}
        records = []
        for name, _, work in operators:
            footprint = sets[name] * moved_or_product_bytes(work)
            metadata = {"backend": "native", "kernel": f"{self.name}_gfx950", "operator": name, "timing": "wall_clock",
                        "operand_sets": sets[name], "operand_footprint_bytes": footprint,
                        "cache_resident": footprint <= INFINITY_CACHE_BYTES,
                        **{key: int(value) for key, value in shape.items()}}
            check = name if name in self.checks else "forward"
            if check in parity:
                metadata["parity"] = parity[check]
            raw = {"elapsed_s": times[name], **work}
            if "achieved_ops" in work:
                raw["peak_tops"] = peak_tops
            if "moved_bytes" in work:
                raw["peak_bandwidth_gbps"] = peak_hbm
            records.append(self.measured(case=f"{self.name}_{name}_{layer.suffix}", dtype=spec.name, raw_metrics=raw,
                                         metadata=metadata))
        return records

    def run(self) -> list[BenchmarkRecord]:
        backend = str(self.params.get("backend", "native")).lower()
        if backend != "native":
            raise KeyError(f"Unknown {self.name} backend: {backend}")
        layers = [dict(layer) for layer in self.params.get("layers", self.default_layers)]
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
            peak_tops = self.context.hardware_profile.peak_compute_tops.get(self.peak_name or spec.name)
            for shape in layers:
                case = f"{self.name}_" + "_".join(f"{key}{value}" for key, value in shape.items())
                unsupported = spec.name not in capi.EXPERT_DTYPES
                if why is not None or unsupported:
                    error = why or f"unsupported dtype for {self.what}: {spec.name}"
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
