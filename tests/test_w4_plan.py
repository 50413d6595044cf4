"""Which kernel a 4-bit product runs on (CPU): the plan compiled for the host."""
from __future__ import annotations

from pathlib import Path
import shutil
import subprocess

import pytest
import torch

import w4_inputs
from teamredbench_amd.native import capi

TESTS = Path(__file__).resolve().parent
# (total rows, experts, N) -> configuration, at 256 CUs: both sides of every bound, and the calls whose times are quoted
PICKS = [
    ((1, 1, 8160), 0), ((16, 1, 8160), 0), ((16, 1, 8161), 1), ((16, 1, 8192), 1), ((16, 1, 12256), 1),
    ((16, 1, 12257), 2), ((1, 1, 14336), 2), ((128, 16, 2048), 2), ((4, 1, 65504), 2), ((4, 1, 65505), 3),
    ((256, 64, 2048), 3), ((17, 1, 1920), 5), ((17, 1, 1921), 4), ((32, 1, 50257), 4), ((64, 1, 1920), 8),
    ((33, 1, 1921), 7), ((64, 1, 8192), 7), ((64, 1, 26112), 7), ((64, 1, 26113), 6), ((64, 1, 28672), 6),
    ((64, 1, 50257), 6), ((4096, 1, 512), 6),
]
# the shapes of test_gpu_experts_w4.py's test_kernels_as_picked
PICKED_THERE = [(16, 1, 4000), (16, 1, 8200), (16, 1, 12300), (256, 64, 1056), (32, 1, 2100), (32, 1, 100),
                (64, 1, 26500), (64, 1, 8192), (64, 1, 100)]


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    capi.load_library().set_tuning("w4_config", None)   # a call that succeeds clears the thread's last error


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "w4_plan_host"
    subprocess.run([shutil.which("g++") or "g++", "-O1", "-std=c++20", str(TESTS / "w4_plan_host.cpp"), "-o", str(exe)],
                   check=True)

    def run(shapes, cus=256):
        text = "".join(f"{rows} {experts} {n} {cus}\n" for rows, experts, n in shapes)
        return [int(v) for v in subprocess.run([str(exe)], input=text, capture_output=True, text=True,
                                               check=True).stdout.split()]

    return run


def test_picks(plan):
    assert plan([shape for shape, _ in PICKS]) == [config for _, config in PICKS]


def test_every_kernel_is_picked_by_a_tested_call(plan):
    assert sorted(set(plan(PICKED_THERE))) == list(range(9))


def test_the_knob_takes_every_configuration_and_no_other():
    lib = capi.load_library()
    for config in range(9):
        with lib.tuned(w4_config=config):
            assert lib.get_tuning("w4_config") == config
    for bad in (9, -2):
        with pytest.raises(capi.NativeLibraryError, match="cannot take"):
            lib.set_tuning("w4_config", bad)


# ---- the exact inputs of the GPU tests notice what a wrong kernel would do ----------------------


def _missed(c: dict, wrong: torch.Tensor) -> float:
    """Share of outputs that a mistake leaves as they are."""
    t = getattr(torch, c["dtype"])
    return float((w4_inputs.product(c).to(t) == wrong.to(t)).double().mean())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("k, group", [(838, 32), (2049, 128), (1300, 512), (16461, 128)])
def test_mistakes_show(dtype, k, group):
    # most outputs are others, even where the unit left out is a single k (one x in five is zero, one weight in sixteen)
    c = w4_inputs.case(dtype, [16], 64, k, group, True, seed=1)
    assert float(((c["x"].double().abs() @ torch.full((k, 1), 2.0 * 31, dtype=torch.float64)) * 2).max()) < 2**24
    x, w = w4_inputs.sorted_x(c), w4_inputs.weights(c, 0)
    scale = w4_inputs.spread(c, c["s"][0])
    for unit in (0, 256 * (k // 256)):                            # a unit of K left out, or taken twice
        for sign in (-1, 1):
            part = x[:, unit:unit + 256] @ w[:, unit:unit + 256].t()
            assert _missed(c, x @ w.t() + sign * part) < 0.5
    shifted = dict(c, s=c["s"].roll(1, 2))                        # the scale of the group before
    assert _missed(c, w4_inputs.product(shifted)) < 0.5
    neighbour = dict(c, s=c["s"].roll(1, 1))                      # of the column before
    assert _missed(c, w4_inputs.product(neighbour)) < 0.5
    assert _missed(c, x @ (w - scale).t()) < 0.5                 # every zero point one too large
    other = dict(c, z=c["z"].roll(1, 1))
    assert _missed(c, w4_inputs.product(other)) < 0.5
    swapped = x.clone()                                           # the two weights of a byte exchanged
    even = k - k % 2
    swapped[:, 0:even:2], swapped[:, 1:even:2] = x[:, 1:even:2], x[:, 0:even:2]
    assert _missed(c, swapped @ w.t()) < 0.5
