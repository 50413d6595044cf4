"""Microscaled 4-bit (MX4) matrices for the tests: the format by its definition, in 64 bits on the CPU.

A row is blocks of 32 e2m1 elements times 2^(scale - 127); rows are padded with zeros to whole units of 128.
"""
from __future__ import annotations

import numpy as np
import torch

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
VALUES = np.concatenate([E2M1, -E2M1])
FLOOR, FIT = 0, 1


def units(columns: int) -> int:
    return -(-columns // 128)


def quantize(x: np.ndarray, rule: int) -> tuple[np.ndarray, np.ndarray]:
    """fp64 (R, C), each value one that the source type holds -> codes (R, whole units of C) and scales, uint8.

    The nearest element is found among all of them; a tie takes the even code.
    """
    rows, columns = x.shape
    wide = np.zeros((rows, units(columns) * 128))
    wide[:, :columns] = x
    blocks = wide.reshape(rows, -1, 32)
    broken = ~np.isfinite(blocks).all(2)
    blocks = np.where(broken[:, :, None], 0.0, blocks)
    most = np.abs(blocks).max(2)
    exponent = np.frexp(most)[1] - 1            # most = m 2^exponent, 1 <= m < 2
    power = exponent - 2
    if rule == FIT:
        power = power + (most > 1.5 * np.exp2(exponent.astype(np.float64)))
    power = np.where(most == 0, -127, np.maximum(power, -127))
    v = np.abs(blocks) * np.exp2(-power.astype(np.float64))[:, :, None]
    distance = np.abs(np.minimum(v, 6.0)[..., None] - E2M1)
    nearest = distance.min(-1, keepdims=True)
    tied = distance == nearest                  # one, or two neighbours of which one code is even
    code = np.where(tied.sum(-1) == 1, tied.argmax(-1), (tied & (np.arange(8) % 2 == 0)).argmax(-1))
    code = code + 8 * np.signbit(blocks)
    code = np.where(broken[:, :, None], 0, code)
    return code.reshape(rows, -1).astype(np.uint8), np.where(broken, 255, power + 127).astype(np.uint8)


def pack(codes: np.ndarray) -> np.ndarray:
    """Codes -> bytes, the even column in the low half."""
    return codes[..., 0::2] | codes[..., 1::2] << 4


def unpack(q: np.ndarray) -> np.ndarray:
    codes = np.empty((*q.shape[:-1], 2 * q.shape[-1]), np.uint8)
    codes[..., 0::2], codes[..., 1::2] = q & 15, q >> 4
    return codes


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """fp64 values of whole units."""
    power = np.exp2(scales.astype(np.float64) - 127)
    power = np.where(scales == 255, np.nan, power)
    return VALUES[codes] * np.repeat(power, 32, axis=-1)


def random(rows: int, columns: int, seed: int, scales: tuple[int, int] = (126, 128)) -> tuple[np.ndarray, np.ndarray]:
    """Random codes (zeros past `columns`) and scale bytes from the inclusive range.

    With the default range, every product of two elements is a multiple of 2^-4 of at most 144, so
    sums over up to 7000 columns are exact in fp32 in any order.
    """
    rng = np.random.default_rng(seed)
    codes = np.zeros((rows, units(columns) * 128), np.uint8)
    codes[:, :columns] = rng.integers(0, 16, (rows, columns))
    return codes, rng.integers(scales[0], scales[1] + 1, (rows, units(columns) * 4)).astype(np.uint8)


EXACT_COLUMNS = 7000
assert 144 * EXACT_COLUMNS < 2**24 * 2.0**-4


def on_gpu(codes: np.ndarray, scales: np.ndarray) -> tuple[torch.Tensor, torch.Tensor]:
    return torch.from_numpy(pack(codes)).cuda(), torch.from_numpy(scales).cuda()
