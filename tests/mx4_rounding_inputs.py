"""Blocks that hold every finite 16-bit value under scales other than its own (for the MX4 rounding tests).

A row is one block: 31 values of one sign-and-exponent range and, somewhere among them, the anchor that sets the scale:
the smallest value of a binade 0 to 5 above them, 1.5 times that, or the binade's largest.
"""
from __future__ import annotations

import torch

EACH = 31
ABOVE = range(6)


def blocks(dtype: torch.dtype) -> torch.Tensor:
    """Rows of 32 values of `dtype`: every finite value under every anchor that is finite and no smaller than it."""
    mantissa_bits = 7 if dtype == torch.bfloat16 else 10
    exponents = 1 << (15 - mantissa_bits)
    g = torch.Generator().manual_seed(mantissa_bits)
    rows = []
    for exponent in range(exponents - 1):              # the last is infinity and NaN; 0: zeros and subnormals
        mantissas = torch.arange(1 << mantissa_bits)
        bits = (exponent << mantissa_bits) + torch.cat([mantissas, mantissas + (1 << 15)])
        for above in ABOVE:
            for mantissa in (0, 1 << (mantissa_bits - 1), (1 << mantissa_bits) - 1):
                if not 0 < exponent + above < exponents - 1:
                    continue
                anchor = ((exponent + above) << mantissa_bits) + mantissa
                values = bits[(bits & 0x7FFF) <= anchor]
                values = values[torch.randperm(values.numel(), generator=g)]
                values = torch.cat([values, torch.zeros(-values.numel() % EACH, dtype=values.dtype)]).view(-1, EACH)
                signs = torch.randint(0, 2, (values.shape[0], 1), generator=g) << 15
                at = exponent * 7 % 32
                rows.append(torch.cat([values[:, :at], anchor + signs, values[:, at:]], dim=1))
    bits = torch.cat(rows)
    return torch.where(bits >= 1 << 15, bits - (1 << 16), bits).to(torch.int16).view(dtype)
