"""The tests' own MX4 definition: hand-made blocks, and mistakes that it would show (no GPU here)."""
from __future__ import annotations

import numpy as np

import mx4_inputs as mx4


def _block(*first: float) -> np.ndarray:
    return np.array([[*first, *[0.0] * (32 - len(first))]])


def test_ties_go_to_the_even_code():
    codes, scales = mx4.quantize(_block(4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -5, 6.5, 7.9), mx4.FLOOR)
    assert scales[0, 0] == 127
    assert list(codes[0, :12]) == [6, 0, 2, 2, 4, 4, 6, 6, 8, 14, 7, 7]
    assert list(mx4.values(codes, scales)[0, :8]) == [4, 0, 1, 1, 2, 2, 4, 4]


def test_scale_rules():
    for most, floor, fit in ((4, 127, 127), (6, 127, 127), (6.01, 127, 128), (7.99, 127, 128), (8, 128, 128),
                             (2.0**-126, 0, 0), (2.0**-149, 0, 0), (1.75 * 2.0**-125, 0, 1), (0, 0, 0),
                             (float(np.finfo(np.float32).max), 252, 253), (np.inf, 255, 255), (np.nan, 255, 255)):
        for rule, wanted in ((mx4.FLOOR, floor), (mx4.FIT, fit)):
            codes, scales = mx4.quantize(_block(0, most), rule)
            assert scales[0, 0] == wanted, (most, rule)
            assert wanted < 255 or not codes.any()


def test_packing_and_padding():
    codes, scales = mx4.random(3, 130, seed=0)
    assert codes.shape == (3, 256) and scales.shape == (3, 8) and not codes[:, 130:].any()
    q = mx4.pack(codes)
    assert q.shape == (3, 128) and (mx4.unpack(q) == codes).all()
    assert q[1, 2] == codes[1, 4] + 16 * codes[1, 5]


def test_products_of_the_random_matrices_are_exact_in_fp32():
    a, b = (mx4.values(*mx4.random(4, mx4.EXACT_COLUMNS, seed)) for seed in (1, 2))
    largest = (np.abs(a) @ np.abs(b).T).max()
    products = a[:, None] * b[None]
    assert (products * 16 == np.round(products * 16)).all() and largest < 2**20
    exact = a @ b.T
    # What a kernel could get wrong moves a sum: a unit left out or a block under its neighbour's scale.
    assert (a[:, :128] @ b[:, :128].T != 0).any()
    assert (np.roll(a.reshape(4, -1, 32), 1, 1).reshape(4, -1) @ b.T != exact).all()
