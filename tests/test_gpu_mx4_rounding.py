"""MX4 rounding of every finite 16-bit value under scales of its own and of larger neighbours (-m gpu)."""
from __future__ import annotations

import pytest
import torch

import mx4_inputs as mx4
from mx4_rounding_inputs import blocks
from test_gpu_mx4 import _check_form, _quantize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rule", [mx4.FLOOR, mx4.FIT])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value_under_other_scales(lib, dtype, rule):
    x = blocks(dtype)
    print(f"[rounding] {dtype} rule {rule} {tuple(x.shape)}", flush=True)
    _check_form(_quantize(lib, x.cuda(), rule, "r")["r"], x.double().numpy(), rule)
    columns = _quantize(lib, x.t().contiguous().cuda(), rule, "c")["c"]
    _check_form(columns, x.double().numpy(), rule)


@pytest.mark.parametrize("rule", [mx4.FLOOR, mx4.FIT])
def test_the_same_values_and_their_neighbours_in_fp32(lib, rule):
    for step in (-1, 0, 1):   # the fp32 values below, at and above them; the anchors stay
        x = blocks(torch.float16).float()
        anchor = x.abs().amax(1, keepdim=True)
        near = (x.view(torch.int32) + step).view(torch.float32)
        x = torch.where((x != 0) & (x.abs() < anchor), near, x)
        print(f"[rounding] fp32 step {step} rule {rule}", flush=True)
        _check_form(_quantize(lib, x.cuda(), rule, "r")["r"], x.double().numpy(), rule)
        _check_form(_quantize(lib, x.t().contiguous().cuda(), rule, "c")["c"], x.double().numpy(), rule)
