"""That the MX4 rounding tests' inputs reach every element code and every border between two (no GPU here)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mx4_inputs as mx4
from mx4_rounding_inputs import blocks

BORDERS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_value_every_code_and_every_tie(dtype):
    x = blocks(dtype)
    assert torch.isfinite(x).all() and x.shape[1] == 32
    all_bits = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16)
    finite = all_bits[torch.isfinite(all_bits.view(dtype))]
    assert torch.isin(finite, x.view(torch.int16)).all()
    for rule in (mx4.FLOOR, mx4.FIT):
        exact = x.double().numpy()
        codes, scales = mx4.quantize(exact, rule)
        codes, scales = codes[:, :32], scales[:, 0]
        counts = np.bincount(codes.ravel(), minlength=16)
        assert (counts >= 2000).all(), (rule, counts)
        v = np.abs(exact) * np.exp2(127.0 - scales.astype(np.float64))[:, None]
        for border in BORDERS:   # ties, which go to the even code
            assert (v == border).sum() >= 50, (rule, border)
        assert ((v > 6).sum() == 0) == (rule == mx4.FIT)


def test_a_rounding_mistake_shows():
    """Truncation, ties away from zero and ties to zero each give other codes."""
    x = blocks(torch.bfloat16).double().numpy()
    codes, scales = mx4.quantize(x, mx4.FLOOR)
    v = np.minimum(np.abs(x) * np.exp2(127.0 - scales[:, :1].astype(np.float64)), 6.0)
    right = codes[:, :32] & 7
    for wrong in (np.searchsorted(mx4.E2M1, v, side="right") - 1, np.searchsorted(BORDERS, v, side="right"),
                  np.searchsorted(BORDERS, v, side="left")):
        assert (wrong != right).sum() > 1000
