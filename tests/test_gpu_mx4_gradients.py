"""A linear layer's gradients through mb_mx4_quantize and mb_gemm_mx4: against differences, and by expert (-m gpu).

Values of the e2m1 grid itself are held exactly along both axes, so the products are the exact gradients rounded once.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mx4_inputs as mx4
from gemm_bounds import elementwise_bound
from teamredbench_amd.native import capi
from test_gpu_mx4 import CANARY, HALF, _product, _quantize, _rounded

pytestmark = pytest.mark.gpu


def _grid(rows: int, columns: int, seed: int) -> np.ndarray:
    return mx4.VALUES[np.random.default_rng(seed).integers(0, 16, (rows, columns))]


def _form(lib, values: np.ndarray, along: str, dtype=torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    form = _quantize(lib, torch.from_numpy(values).to(dtype).cuda(), mx4.FLOOR, along)[along]
    return tuple(t[:-1].contiguous() for t in form)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tokens, n, k", [(3, 5, 8), (40, 33, 70), (129, 130, 257)])
def test_gradients_are_the_layers_differences(lib, dtype, tokens, n, k):
    """dx and dw from the calls against central differences of sum(grad * (x w^T)), which is linear in x and in w."""
    x, w, grad = _grid(tokens, k, 1), _grid(n, k, 2), _grid(tokens, n, 3)
    got = {}
    for which, left, right, depth, shape in ((0, (grad, "r"), (w, "c"), n, (tokens, k)),
                                             (1, (grad, "c"), (x, "c"), tokens, (n, k))):
        out = torch.empty(shape, dtype=getattr(torch, dtype), device="cuda")
        _product(lib, dtype, _form(lib, *left), _form(lib, *right), out, n=shape[1], k=depth)
        got[which] = out.cpu()
    loss = lambda p, q: float((grad * (p @ q.T)).sum())   # noqa: E731 -- multiples of 1/8 below 2^40: exact
    rng = np.random.default_rng(4)
    for which, operand in ((0, x), (1, w)):
        every = [(i, j) for i in range(operand.shape[0]) for j in range(operand.shape[1])]
        chosen = every if len(every) <= 64 else [every[i] for i in rng.choice(len(every), 64, replace=False)]
        for i, j in chosen:
            up, down = [x.copy(), w.copy()], [x.copy(), w.copy()]
            up[which][i, j] += 0.5
            down[which][i, j] -= 0.5
            difference = torch.tensor(loss(*up) - loss(*down), dtype=torch.float64).float().to(getattr(torch, dtype))
            assert got[which][i, j] == difference, (which, i, j)
    assert torch.equal(got[0], _rounded(grad @ w, dtype)) and torch.equal(got[1], _rounded(grad.T @ x, dtype))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("counts, n, k", [([5, 0, 130, 33], 72, 200), ([1] * 9, 264, 96), ([300, 7], 130, 257)])
def test_gradient_of_x_by_expert(lib, dtype, counts, n, k):
    """dx[p] = grad[p] w[e]: the product by expert on each expert's w along its columns, one quantisation an expert."""
    experts, total, spare = len(counts), sum(counts), 3
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    g = torch.Generator().manual_seed(n)
    w = torch.randn(experts, n, k, generator=g).to(getattr(torch, dtype)).cuda()
    grad = torch.randn(total + spare, n, generator=g).to(getattr(torch, dtype)).cuda()
    units = mx4.units(n)
    wt = (torch.empty(experts * k, 64 * units, dtype=torch.uint8, device="cuda"),
          torch.empty(experts * k, 4 * units, dtype=torch.uint8, device="cuda"))
    stream = torch.cuda.current_stream().cuda_stream
    for e in range(experts):
        lib.mx4_quantize(capi.DTYPES[dtype], w[e].data_ptr(), 0, n, k, mx4.FLOOR, None, None,
                         wt[0][e * k].data_ptr(), wt[1][e * k].data_ptr(), stream)
    form = tuple(t[:-1].contiguous() for t in _quantize(lib, grad, mx4.FLOOR, "r")["r"])
    out = torch.full((total + spare, k), CANARY, dtype=grad.dtype, device="cuda")
    _product(lib, dtype, form, wt, out, offsets=torch.from_numpy(offsets).cuda(), experts=experts, n=k, k=n)
    left = torch.from_numpy(mx4.values(*mx4.quantize(grad.double().cpu().numpy(), mx4.FLOOR)))
    for e in range(experts):
        lo, hi = offsets[e], offsets[e + 1]
        right = torch.from_numpy(mx4.values(*mx4.quantize(w[e].double().cpu().numpy().T, mx4.FLOOR)))
        exact, magnitude = left[lo:hi] @ right.T, left[lo:hi].abs() @ right.abs().T
        assert ((out[lo:hi].double().cpu() - exact).abs() <= elementwise_bound(dtype, n, exact.abs(), magnitude)).all(), e
    assert (out[total:] == CANARY).all()
