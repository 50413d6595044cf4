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
