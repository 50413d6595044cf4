"""The copies of a layer that the ``experts`` and ``mx4`` benchmarks cycle through, operator by operator."""
from __future__ import annotations

from types import SimpleNamespace

import pytest

from teamredbench_amd.benchmarks import experts, mx4

GIB = 1 << 30
CACHE = 256 << 20
TARGET = 3 * CACHE
MOVERS = ("quantize_x", "quantize_w", "dequantize_w", "quantize_grad")


def _mx4(**params) -> mx4.Mx4Benchmark:
    return mx4.Mx4Benchmark(SimpleNamespace(hardware_profile=SimpleNamespace(peak_hbm_bandwidth_gbps=8000.0)), params)


def _operators(bench: mx4.Mx4Benchmark, tokens: int, k: int, n: int):
    return bench._operators(SimpleNamespace(tokens=tokens, k=k, n=n, total=tokens, experts=0), 2, True)


def test_what_only_moves_bytes_passes_the_cache_where_the_products_take_one_set():
    bench = _mx4()
    operators = _operators(bench, 4096, 4096, 14336)
    work = {name: w for name, _, w in operators}
    sets = bench._sets_by_operator(operators, 10000.0, 900 << 20, 250 * GIB, 60)
    assert {sets[name] for name in ("product", "layer", "x_grad", "w_grad")} == {1}
    for name in MOVERS:
        moved = work[name]["moved_bytes"]
        assert moved < CACHE   # one set lies in the Infinity Cache from call to call
        assert sets[name] * moved >= TARGET > (sets[name] - 1) * moved


def test_bounds_of_the_copies():
    bench = _mx4()
    operators = _operators(bench, 4096, 4096, 14336)
    assert set(bench._sets_by_operator(operators, 10000.0, 100 * GIB, 250 * GIB, 60).values()) == {1}   # half of the memory
    assert max(bench._sets_by_operator(operators, 10000.0, 900 << 20, 250 * GIB, 3).values()) == 3      # as many as calls
    assert set(_mx4(operand_sets=2)._sets_by_operator(operators, 10000.0, 900 << 20, 250 * GIB, 60).values()) == {2}
    few = bench._sets_by_operator(operators, 10000.0, 900 << 20, 250 * GIB, 2)   # 2 x 50 MB would not pass the cache
    assert few["quantize_x"] == 1 and few["dequantize_w"] == 2
    unknown = bench._sets_by_operator(operators, None, 900 << 20, 250 * GIB, 60)   # a profile without the type's peak
    assert unknown["product"] == 1 and unknown["quantize_x"] > 1


def test_a_layer_bound_by_memory_keeps_its_products_copies():
    bench = _mx4()
    operators = _operators(bench, 1, 4096, 14336)
    products = bench._operand_sets(operators, 10000.0, 300 << 20, 250 * GIB)
    sets = bench._sets_by_operator(operators, 10000.0, 300 << 20, 250 * GIB, 60)
    assert products > 1 and sets["product"] == sets["layer"] == products and min(sets.values()) == products


def test_the_experts_benchmark_too():
    context = SimpleNamespace(hardware_profile=SimpleNamespace(peak_hbm_bandwidth_gbps=8000.0))
    bench = experts.ExpertsBenchmark(context, {})
    layer = SimpleNamespace(tokens=4096, experts=8, top_k=2, k=4096, n=14336, total=8192, group=0)
    operators = bench._operators(layer, 2, True)
    work = {name: w for name, _, w in operators}
    sets = bench._sets_by_operator(operators, 2500.0, 3 * GIB, 250 * GIB, 60)
    assert sets["up"] == sets["layer"] == 1
    assert work["combine"]["moved_bytes"] < CACHE and sets["combine"] * work["combine"]["moved_bytes"] >= TARGET


@pytest.mark.gpu
def test_records_of_a_layer_bound_by_operations(tmp_path, lib):
    from teamredbench_amd.runner import run_suite
    from test_mx4_benchmark import _suite

    layer = {"tokens": 4096, "k": 4096, "n": 8192}
    records = run_suite(_suite(tmp_path, ["bfloat16"], layers=[layer], warmup=10, iterations=20)).records
    by_name = {r.metadata["operator"]: r for r in records}
    assert {"product", "w_grad", *MOVERS} <= by_name.keys()
    for name, r in by_name.items():
        assert r.status == "ok" and r.metadata["parity"]["passed"], (name, r.error)
        assert r.metadata["cache_resident"] == (r.metadata["operand_footprint_bytes"] <= CACHE)
    assert by_name["product"].metadata["operand_sets"] == 1
    for name in MOVERS:
        r = by_name[name]
        assert r.metadata["cache_resident"] is False and r.metadata["operand_sets"] > 1
        assert r.metadata["operand_footprint_bytes"] == r.metadata["operand_sets"] * r.raw_metrics["moved_bytes"]
        print(f"[sets] {name} {r.metadata['operand_sets']} {r.metrics['hbm_bandwidth_gbps']:.0f} GB/s", flush=True)
