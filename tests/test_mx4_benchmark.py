"""The ``mx4`` benchmark: registered, skipped cleanly without a GPU, run end to end with one; its plain forms and checks."""
from __future__ import annotations

import math
from pathlib import Path

import pytest
import torch
import yaml

import mx4_inputs
from teamredbench_amd.benchmarks import mx4
from teamredbench_amd.benchmarks.layers import parity_of
from teamredbench_amd.runner import PACKAGED_HARDWARE_DIR, run_suite

SUITE = PACKAGED_HARDWARE_DIR.parent.parent / "suites" / "mx4_layer.yaml"
LAYERS = [{"tokens": 70, "k": 264, "n": 200}, {"tokens": 20, "k": 256, "n": 72, "experts": 6, "top_k": 2}]


def _suite(tmp: Path, dtypes: list[str], **params) -> Path:
    params = {"backend": "native", "dtypes": dtypes, "layers": LAYERS, "warmup": 1, "iterations": 3, **params}
    doc = {"name": "mx4", "device": {"profile": str(PACKAGED_HARDWARE_DIR / "amd_instinct_mi355x.yaml")},
           "runtime": {"profile": str(PACKAGED_HARDWARE_DIR.parent / "rocm" / "rocm_7.yaml")},
           "outputs": {"directory": str(tmp / "results"), "formats": ["json", "csv"]},
           "benchmarks": [{"benchmark": "mx4", "params": params}]}
    path = tmp / "mx4.yaml"
    path.write_text(yaml.safe_dump(doc), encoding="utf-8")
    return path


def test_packaged_suite_names_the_benchmark():
    import teamredbench_amd.builtin  # noqa: F401
    from teamredbench_amd.registry import get_benchmark

    doc = yaml.safe_load(SUITE.read_text(encoding="utf-8"))
    assert [b["benchmark"] for b in doc["benchmarks"]] == ["mx4"]
    assert get_benchmark("mx4").default_metrics


def test_without_a_gpu_every_layer_is_skipped(tmp_path):
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    records = run_suite(_suite(tmp_path, ["bfloat16", "float16"])).records
    assert len(records) == 4 and all(r.status == "skipped" and "ROCm" in r.error for r in records)


@pytest.mark.parametrize("rule", [mx4_inputs.FLOOR, mx4_inputs.FIT])
def test_the_checks_own_quantisation_is_the_definition(rule):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(60, 200, generator=g) * 2.0 ** torch.randint(-130, 120, (60, 1), generator=g)
    x[7] = 0
    x[20:40] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])[torch.randint(0, 8, (20, 200), generator=g)]
    codes, scales = mx4_inputs.quantize(x.double().numpy(), rule)
    wanted = torch.from_numpy(mx4_inputs.values(codes, scales)[:, :200]).float()
    assert torch.equal(mx4.quantized_values(torch, x, rule), wanted)
    q, s = torch.from_numpy(mx4_inputs.pack(codes)), torch.from_numpy(scales)
    assert torch.equal(mx4.values_of(torch, q, s, 200), wanted)


def test_an_unknown_scale_rule_is_an_error():
    from types import SimpleNamespace

    bench = mx4.Mx4Benchmark(SimpleNamespace(), {"scale_rule": "round"})
    with pytest.raises(KeyError, match="scale_rule"):
        bench.layer_type(torch, None, "bfloat16", LAYERS[0], "cpu", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("rule", ["floor", "fit"])
def test_layers_run_end_to_end(tmp_path, lib, rule):
    records = run_suite(_suite(tmp_path, ["bfloat16", "float16", "float32"], scale_rule=rule)).records
    ran = [r for r in records if r.dtype != "float32"]
    assert len(ran) == 2 * (8 + 6)
    for r in ran:
        assert r.status == "ok", (r.case, r.dtype, r.error)
        assert r.metadata["parity"]["passed"] and r.metrics["latency_us"] > 0
        rate = r.metrics.get("achieved_tops") or r.metrics.get("hbm_bandwidth_gbps")
        assert rate is not None and math.isfinite(rate) and rate > 0
    assert {r.raw_metrics["peak_tops"] for r in ran if "peak_tops" in r.raw_metrics} == {10000.0}
    refused = [r for r in records if r.dtype == "float32"]
    assert len(refused) == 2 and all(r.status == "skipped" and "unsupported" in r.error for r in refused)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", LAYERS)
def test_each_check_passes_and_notices_a_wrong_buffer(lib, shape):
    layer = mx4.Mx4Layer(torch, lib, "bfloat16", shape, torch.device("cuda:0"), 0)
    layer.forward()
    layer.dequantize_w()
    names = [("forward", "out"), ("quantize_x", "x_q"), ("quantize_x", "x_s"), ("quantize_w", "w_q"),
             ("dequantize_w", "w_values")]
    if layer.differentiable:
        layer.prepare_backward()
        layer.backward()
        names += [("quantize_x", "xt_q"), ("quantize_w", "wt_s"), ("quantize_grad", "grad_q"),
                  ("quantize_grad", "gradt_q"), ("x_grad", "grad_x"), ("w_grad", "grad_w")]
    rows = min(layer.tokens, 20)

    def passed(name):
        return parity_of(torch, getattr(layer, f"check_{name}")(rows))["passed"]

    for name, buffer in names:
        assert passed(name), name
        right = getattr(layer, buffer)
        wrongs = [right ^ 1] if right.dtype == torch.uint8 else [right * 1.05, right.roll(1, 0),
                                                                 torch.full_like(right, torch.nan)]
        for wrong in wrongs:
            setattr(layer, buffer, wrong)
            assert not passed(name), (name, buffer)
        setattr(layer, buffer, right)
        assert passed(name)
