"""The ``experts`` benchmark's own checks: every output it times is checked, and a wrong one fails its record."""
from __future__ import annotations

import pytest
import torch

from teamredbench_amd.benchmarks import experts

LAYER = {"tokens": 90, "experts": 12, "top_k": 3, "k": 264, "n": 200}


def test_the_worst_output_decides():
    good, want = torch.ones(8, 8), torch.ones(8, 8)
    off = good.clone()
    off[0, 0] = 3.0
    near = parity = experts.parity_of(torch, {"a": ("bfloat16", good, want), "b": ("bfloat16", good * 1.001, want)})
    assert near["passed"] and near["rel_frobenius"] == parity["outputs"]["b"] > 0
    bad = experts.parity_of(torch, {"a": ("bfloat16", good, want), "b": ("bfloat16", off, want)})
    assert not bad["passed"] and bad["rel_frobenius"] == bad["outputs"]["b"]
    nothing = experts.parity_of(torch, {"a": ("bfloat16", torch.zeros(2, 2), torch.zeros(2, 2))})
    assert nothing["passed"]
    stray = experts.parity_of(torch, {"a": ("bfloat16", torch.ones(2, 2), torch.zeros(2, 2))})
    assert not stray["passed"]


def test_a_nan_is_no_match():
    got = torch.ones(4, 4)
    got[1, 2] = torch.nan
    assert not experts.parity_of(torch, {"a": ("bfloat16", got, torch.ones(4, 4)),
                                         "b": ("bfloat16", torch.ones(2), torch.ones(2))})["passed"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_each_check_passes_and_notices_a_wrong_buffer(lib, dtype):
    layer = experts.ExpertLayer(torch, lib, dtype, LAYER, torch.device("cuda:0"), 0)
    layer.forward()
    layer.prepare_backward()
    for call in (layer.combine_grad, layer.rows_grad, layer.up_grad, layer.route_grad):
        call()
    tokens = 20

    def passed(name):
        return experts.parity_of(torch, getattr(layer, f"check_{name}")(tokens))["passed"]

    assert all(passed(name) for name in ("forward", *experts.GRADIENTS))
    # what each check reads, and a mistake in it: a result scaled, or rows in another's place
    for name, buffer in (("forward", "out"), ("combine_grad", "grad_y"), ("combine_grad", "grad_weights"),
                         ("rows_grad", "grad_hidden"), ("up_grad", "grad_up"), ("route_grad", "grad_logits")):
        right = getattr(layer, buffer)
        for wrong in (right * 1.05, right.roll(1, 0), torch.full_like(right, torch.nan)):
            setattr(layer, buffer, wrong)
            assert not passed(name), (name, buffer)
        setattr(layer, buffer, right)
        assert passed(name)


@pytest.mark.gpu
def test_every_record_carries_a_check(tmp_path, lib):
    from teamredbench_amd.runner import run_suite
    from test_experts_benchmark import LAYERS, _suite

    records = run_suite(_suite(tmp_path, LAYERS, ["bfloat16"])).records
    assert len(records) == 9 + 5
    for r in records:
        assert r.status == "ok" and r.metadata["parity"]["passed"], (r.case, r.metadata.get("parity"))
    gradients = {r.metadata["operator"]: set(r.metadata["parity"]["outputs"]) for r in records
                 if r.metadata["operator"] in experts.GRADIENTS}
    assert gradients["combine_grad"] == {"grad_y", "grad_weights"} and gradients["route_grad"] == {"grad_logits"}
    assert gradients["rows_grad"] == {"grad_hidden"} and len(gradients["up_grad"]) == 2


# ---- what the timed calls cycle through ------------------------------------------------


class _Sizes:
    def __init__(self, tokens, experts, top_k, k, n, group=0):
        self.tokens, self.experts, self.top_k, self.k, self.n, self.group = tokens, experts, top_k, k, n, group
        self.total = tokens * top_k


def _benchmark(**params):
    from types import SimpleNamespace

    context = SimpleNamespace(hardware_profile=SimpleNamespace(peak_hbm_bandwidth_gbps=8000.0))
    return experts.ExpertsBenchmark(context, params)


GIB = 1 << 30


def test_decode_weights_pass_the_cache():
    bench = _benchmark()
    decode = bench._operators(_Sizes(32, 32, 4, 4096, 2048, group=128), 2, False)
    work = {name: w for name, _, w in decode}
    # 32 matrices of 4096 x 2048 at 4 bits, a 16-bit scale for 128 of them, and 128 rows in and out
    assert work["down"]["gemm_bytes"] == 32 * 4096 * (1024 + 16 * 2) + 128 * (4096 + 2048) * 2
    sets = bench._operand_sets(decode, 2500.0, 700 << 20, 250 * GIB)
    assert sets * work["down"]["gemm_bytes"] >= 3 * (256 << 20) > (sets - 1) * work["down"]["gemm_bytes"]
    assert bench._operand_sets(decode, 2500.0, 100 * GIB, 250 * GIB) == 1      # no more than half of the free memory
    assert _benchmark(operand_sets=3)._operand_sets(decode, 2500.0, 700 << 20, 250 * GIB) == 3


def test_a_batch_bound_by_operations_takes_one_set():
    bench = _benchmark()
    batch = bench._operators(_Sizes(16384, 8, 2, 4096, 14336), 2, True)
    assert bench._operand_sets(batch, 2500.0, 4 * GIB, 250 * GIB) == 1
    work = {name: w for name, _, w in batch}
    assert work["layer"]["gemm_bytes"] == sum(w.get("gemm_bytes", 0) + w.get("moved_bytes", 0) for name, w in work.items()
                                              if name in ("route", "up", "down", "combine"))


def test_products_have_a_bandwidth():
    assert "gemm_bandwidth_gbps" in experts.ExpertsBenchmark.default_metrics


@pytest.mark.gpu
def test_copies_are_the_layer_on_buffers_of_their_own(lib):
    layer = experts.ExpertLayer(torch, lib, "bfloat16", LAYER, torch.device("cuda:0"), 0)
    layer.forward()
    other = layer.clone()
    mine, its = layer.buffers(), other.buffers()
    assert mine.keys() == its.keys() and {"x", "up", "down", "out", "slots"} <= mine.keys()
    assert all(mine[name].data_ptr() != its[name].data_ptr() for name in mine)
    assert other.workspace is layer.workspace
    other.out.fill_(7.0)
    other.forward()
    assert torch.equal(other.out, layer.out)


@pytest.mark.gpu
def test_records_say_how_large_their_operands_are(tmp_path, lib):
    from teamredbench_amd.runner import run_suite
    from test_experts_benchmark import LAYERS, _suite

    for r in run_suite(_suite(tmp_path, LAYERS, ["bfloat16"])).records:
        sets, footprint = r.metadata["operand_sets"], r.metadata["operand_footprint_bytes"]
        assert sets > 1 and footprint % sets == 0
        assert r.metadata["cache_resident"] == (footprint <= 256 << 20)
        if r.metadata["operator"] in ("up", "down", "rows_grad", "up_grad", "layer"):
            assert r.metrics["gemm_bandwidth_gbps"] > 0
