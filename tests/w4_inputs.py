"""4-bit products whose sums are exact in fp32, so that every kernel has to give the same bits.

Shared by the tests of mb_gemm_w4. x and q - z are integers and the scales
powers of two. A sum of such products is exact in any order while the sum of
magnitudes, over the smallest step, stays below 2^24; weights may be held with
an offset of up to 16 beside |q - z|, group by group.
"""
from __future__ import annotations

import torch


def product(c: dict) -> torch.Tensor:
    """out[p][n] = sum over k of x[p][k] s (q - z) in 64 bits, sorted row by sorted row."""
    total, n = c["total"], c["n"]
    out = torch.zeros(total, n, dtype=torch.float64)
    for e in range(len(c["counts"])):
        lo, hi = sum(c["counts"][:e]), sum(c["counts"][:e + 1])
        out[lo:hi] = sorted_x(c)[lo:hi] @ weights(c, e).t()
    return out


def sorted_x(c: dict) -> torch.Tensor:
    x = c["x"].double()
    return x if c["rows"] is None else x[c["rows"].long()]


def spread(c: dict, v: torch.Tensor) -> torch.Tensor:
    """Per group -> per k."""
    return v.double().repeat_interleave(c["group"], -1)[..., :c["k"]]


def weights(c: dict, e: int) -> torch.Tensor:
    """Expert e's n x k matrix in 64 bits."""
    q = torch.stack([c["q"][e] & 15, c["q"][e] >> 4], dim=-1).flatten(1)[:, :c["k"]].double()
    return spread(c, c["s"][e]) * (q - (8.0 if c["z"] is None else spread(c, c["z"][e])))


def pack(q: torch.Tensor) -> torch.Tensor:
    """Integers 0 .. 15 in the last dimension, two a byte, the even one low; a last half is filled with ones."""
    if q.shape[-1] % 2:
        q = torch.cat([q, torch.full_like(q[..., :1], 15)], dim=-1)
    return (q[..., 0::2] | (q[..., 1::2] << 4)).to(torch.uint8)


def case(dtype: str, counts: list[int], n: int, k: int, group: int, zeros: bool, *, tokens: int | None = None,
         seed: int = 0) -> dict:
    """Random weights: x in -2 .. 2, s one of 1/2, 1, 2 by column and group, z in 0 .. 15. Sums of magnitudes
    are at most k * 2 * 2 * 31 in steps of 1/2: exact up to k = 67000."""
    g = torch.Generator().manual_seed(seed)
    t = getattr(torch, dtype)
    experts, total, groups = len(counts), sum(counts), -(-k // group)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=g)

    return {"dtype": dtype, "counts": counts, "n": n, "k": k, "group": group, "total": total,
            "x": ints(-2, 2, total if tokens is None else tokens, k).to(t),
            "rows": None if tokens is None else ints(0, tokens - 1, total).to(torch.int32),
            "q": pack(ints(0, 15, experts, n, k)), "s": (2.0 ** ints(-1, 1, experts, n, groups)).to(t),
            "z": ints(0, 15, experts, n, groups).to(t) if zeros else None}


def near_zero_point(dtype: str, rows: int, n: int, k: int, group: int, zeros: bool, powers: int, seed: int = 0) -> dict:
    """x all positive, and weights that are zero but for two of each column, which are one step of their scale: the
    result is small beside sums in which q, or q with an offset, stands for q - z. Scales 1 .. 2^powers."""
    g = torch.Generator().manual_seed(seed)
    t = getattr(torch, dtype)
    groups = -(-k // group)
    z = torch.randint(1, 15, (1, n, groups), generator=g) if zeros else torch.full((1, n, groups), 8)
    q = z.repeat_interleave(group, 2)[:, :, :k].clone()
    for _ in range(2):
        at = torch.randint(0, k, (1, n, 1), generator=g)
        q.scatter_(2, at, z.gather(2, at // group) + torch.randint(0, 2, (1, n, 1), generator=g) * 2 - 1)
    c = {"dtype": dtype, "counts": [rows], "n": n, "k": k, "group": group, "total": rows, "rows": None,
         "x": torch.randint(32, 64, (rows, k), generator=g).to(t), "q": pack(q),
         "s": (2.0 ** torch.randint(0, powers + 1, (1, n, groups), generator=g)).to(t), "z": z.to(t) if zeros else None}
    return c
