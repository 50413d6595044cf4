"""MX4 products in fp16 on every kernel, and by expert on x without a list (-m gpu).

Sums are exact in fp32 in any order (tests/mx4_inputs.py), so every result has to match bit for bit.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mx4_inputs as mx4
from teamredbench_amd.benchmarks.mx4 import values_of
from teamredbench_amd.native import capi
from test_gpu_mx4 import (CANARY, CONFIGS, DENSE, EXPERTS, HALF, _exact_product, _product, _rounded, _strided)
from test_gpu_mx4_large import _random

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("config, splits", CONFIGS)
def test_every_kernel_in_fp16(lib, tune, config, splits):
    tune(mx4_config=config, mx4_splits=splits)
    for m, n, k in [*DENSE, (70, 130, 6000)]:
        print(f"[kernel] fp16 {config} splits {splits} {m}x{n}x{k}", flush=True)
        a, b = mx4.random(m, k, m + k), mx4.random(n, k, n * 3 + k)
        wanted = _rounded(_exact_product(a, b), "float16")
        x, w = mx4.on_gpu(*a), mx4.on_gpu(*b)
        out = _strided(torch.full((m + 1, n), CANARY, dtype=wanted.dtype), n + 5, 0, CANARY)
        _product(lib, "float16", x, w, out, total=m, n=n, k=k)
        assert torch.equal(out[:m].cpu(), wanted)
        assert (out[m:] == CANARY).all()
        assert (torch.as_strided(out, (m, 5), (n + 5, 1), n) == CANARY).all()


@pytest.mark.parametrize("config, splits", [(None, None), *CONFIGS])
def test_by_expert_without_a_list(lib, tune, config, splits):
    """x has every sorted row and some of no expert: experts of none, of one row, and 70 of them."""
    tune(mx4_config=config, mx4_splits=splits)
    for counts, _ in EXPERTS:
        experts, total, spare = len(counts), sum(counts), 5
        offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        for n, k in ((70, 300), (264, 1500)):
            a, b = mx4.random(total + spare, k, 3), mx4.random(experts * n, k, 4)
            va, vb = mx4.values(*a), mx4.values(*b).reshape(experts, n, -1)
            exact = np.concatenate([va[offsets[e]:offsets[e + 1]] @ vb[e].T for e in range(experts)])
            x, w, d_offsets = mx4.on_gpu(*a), mx4.on_gpu(*b), torch.from_numpy(offsets).cuda()
            for dtype in HALF:
                print(f"[experts] {config} splits {splits} {dtype} {counts} {n}x{k}", flush=True)
                wanted = _rounded(exact, dtype)
                out = torch.full((total + spare, n), CANARY, dtype=wanted.dtype, device="cuda")
                _product(lib, dtype, x, w, out, offsets=d_offsets, experts=experts, n=n, k=k)
                assert torch.equal(out[:total].cpu(), wanted)
                assert (out[total:] == CANARY).all()


def _gemm(lib, dtype, x, w, out, n, k, *, rows=None, offsets=None, experts=1, workspace=None):
    lib.gemm_mx4(capi.DTYPES[dtype], x[0].data_ptr(), x[1].data_ptr(), x[0].shape[0],
                 None if rows is None else rows.data_ptr(), w[0].data_ptr(), w[1].data_ptr(), out.data_ptr(),
                 out.stride(0), None if offsets is None else offsets.data_ptr(), experts, out.shape[0], n, k,
                 None if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.numel(),
                 torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows, n, k, ld", [(8192, 6144, 384, 6144), (4100, 4360, 512, 4360),
                                            (5000, 4100, 1152, 4161)])
def test_blocks_that_make_several_dense_tiles(lib, tune, dtype, rows, n, k, ld):
    """Tiles of 256, one block a CU: whole ones stored among the next one's loads, others behind a full wait."""
    tune(mx4_config=0)
    x, w = _random(rows, k, 1), _random(n, k, 2)
    whole = torch.full((rows + 1, ld), CANARY, dtype=getattr(torch, dtype), device="cuda")
    out = whole[:rows, :n]
    for _ in range(2):
        _gemm(lib, dtype, x, w, out, n, k)
    wanted = values_of(torch, *x, k) @ values_of(torch, *w, k).t().contiguous()
    assert torch.equal(out, wanted.to(out.dtype))
    assert (whole[rows] == CANARY).all() and (whole[:, n:] == CANARY).all()


@pytest.mark.parametrize("listed", [False, True])
def test_blocks_that_make_several_tiles_by_expert_in_fp16(lib, tune, listed):
    tune(mx4_config=0)
    n, k, experts = 2050, 384, 60
    g = torch.Generator().manual_seed(9)
    counts = torch.randint(0, 900, (experts,), generator=g)
    counts[torch.rand(experts, generator=g) < 0.3] = 0
    counts[10:14] = torch.tensor([256, 512, 1, 257])
    total = int(counts.sum()) + 9
    offsets = torch.cat([torch.tensor([4]), counts.cumsum(0) + 4]).int()
    x, w = _random(total, k, 1), _random(experts * n, k, 2)
    rows = torch.randint(-1, total + 1, (total,), generator=g).int()
    out = torch.full((total, n), CANARY, dtype=torch.float16, device="cuda")
    _gemm(lib, "float16", x, w, out, n, k, rows=rows.cuda() if listed else None, offsets=offsets.cuda(), experts=experts)
    values = values_of(torch, *x, k)
    if listed:
        there = ((rows >= 0) & (rows < total)).cuda()
        values = values[rows.clamp(0, total - 1).long().cuda()] * there[:, None]
    for e in range(experts):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        wv = values_of(torch, w[0][e * n:(e + 1) * n], w[1][e * n:(e + 1) * n], k)
        assert torch.equal(out[lo:hi], (values[lo:hi].contiguous() @ wv.t().contiguous()).half()), e
    assert (out[:4] == CANARY).all() and (out[int(offsets[-1]):] == CANARY).all()


@pytest.mark.parametrize("config, splits", [(None, None), (1, 1), (2, 3), (3, 2), (4, 1), (5, None), (6, None)])
def test_streamed_w_in_fp16(lib, tune, config, splits):
    """96 MB of w and more, read once, are loaded past the caches."""
    tune(mx4_config=config, mx4_splits=splits)
    n, k = 31003, 6016
    w = _random(n, k, 2)
    wv = values_of(torch, *w, k).t().contiguous()
    workspace = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    for m in (1, 8, 30, 64, 100):
        x, out = _random(m, k, m), torch.full((m + 1, n), CANARY, dtype=torch.float16, device="cuda")
        _gemm(lib, "float16", x, w, out[:m], n, k, workspace=workspace)
        assert torch.equal(out[:m], (values_of(torch, *x, k) @ wv).half()), m
        assert (out[m] == CANARY).all()
