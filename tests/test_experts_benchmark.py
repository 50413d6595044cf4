"""The ``experts`` benchmark: registered, skipped cleanly without a GPU, and run end to end with one."""
from __future__ import annotations

import math
from pathlib import Path

import pytest
import yaml

from teamredbench_amd.runner import PACKAGED_HARDWARE_DIR, run_suite

SUITE = PACKAGED_HARDWARE_DIR.parent.parent / "suites" / "expert_layer.yaml"
LAYERS = [{"tokens": 300, "experts": 12, "top_k": 3, "k": 264, "n": 200},
          {"tokens": 20, "experts": 8, "top_k": 2, "k": 256, "n": 192, "group": 64}]


def _suite(tmp: Path, layers: list[dict], dtypes: list[str]) -> Path:
    params = {"backend": "native", "dtypes": dtypes, "layers": layers, "warmup": 1, "iterations": 3}
    doc = {"name": "experts", "device": {"profile": str(PACKAGED_HARDWARE_DIR / "amd_instinct_mi355x.yaml")},
           "runtime": {"profile": str(PACKAGED_HARDWARE_DIR.parent / "rocm" / "rocm_7.yaml")},
           "outputs": {"directory": str(tmp / "results"), "formats": ["json", "csv"]},
           "benchmarks": [{"benchmark": "experts", "params": params}]}
    path = tmp / "experts.yaml"
    path.write_text(yaml.safe_dump(doc), encoding="utf-8")
    return path


def test_packaged_suite_names_the_benchmark():
    import teamredbench_amd.builtin  # noqa: F401
    from teamredbench_amd.registry import get_benchmark

    doc = yaml.safe_load(SUITE.read_text(encoding="utf-8"))
    assert [b["benchmark"] for b in doc["benchmarks"]] == ["experts"]
    assert get_benchmark("experts").default_metrics


def test_without_a_gpu_every_layer_is_skipped(tmp_path):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    records = run_suite(_suite(tmp_path, LAYERS, ["bfloat16", "float16"])).records
    assert len(records) == 4 and all(r.status == "skipped" and "ROCm" in r.error for r in records)


@pytest.mark.gpu
def test_layers_run_end_to_end(tmp_path, lib):
    records = run_suite(_suite(tmp_path, LAYERS, ["bfloat16", "float16", "float32"])).records
    ran = [r for r in records if r.dtype != "float32"]
    assert len(ran) == 2 * (9 + 5)
    for r in ran:
        assert r.status == "ok", (r.case, r.dtype, r.error)
        assert r.metrics["latency_us"] > 0
        rate = r.metrics.get("achieved_tops") or r.metrics.get("hbm_bandwidth_gbps")
        assert rate is not None and math.isfinite(rate) and rate > 0
    layers = [r for r in ran if r.metadata["operator"] == "layer"]
    assert len(layers) == 4 and all(r.metadata["parity"]["passed"] for r in layers)
    refused = [r for r in records if r.dtype == "float32"]
    assert len(refused) == 2 and all(r.status == "skipped" and "unsupported" in r.error for r in refused)
