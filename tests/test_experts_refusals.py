"""What the expert layer's entry points refuse, before any device is touched (no GPU here)."""
from __future__ import annotations

import pytest

from teamredbench_amd.native import capi

P = 1 << 20   # an address that is never read: every call below is refused first
BF, F32, F8 = capi.DT_BFLOAT16, capi.DT_FLOAT32, capi.DT_FLOAT8_E4M3FN
INVALID, UNSUPPORTED, SHAPE, WORKSPACE = (capi.MB_ERR_INVALID_ARG, capi.MB_ERR_UNSUPPORTED, capi.MB_ERR_SHAPE,
                                          capi.MB_ERR_WORKSPACE)

ROUTE = dict(dtype=F32, logits=P, ld=0, tokens=10, experts=8, top_k=2, normalize=True, weights=P, expert_ids=P,
             offsets=P, rows=P, slots=P)
ROUTE_GRAD = dict(dtype=F32, logits=P, ld=0, expert_ids=P, grad_weights=P, tokens=10, experts=8, top_k=2,
                  normalize=True, grad_logits=P, ld_grad=0)
GROUPED = dict(op=0, dtype=BF, x=P, ldx=0, x_rows=10, rows=None, y=P, ldy=0, out=P, ldo=0, offsets=P, experts=4,
               total_rows=10, n=16, k=24)
W4 = dict(dtype=BF, x=P, ldx=0, x_rows=10, rows=None, q=P, scales=P, zeros=None, group=32, out=P, ldo=0, offsets=P,
          experts=4, total_rows=10, n=16, k=64)
COMBINE = dict(dtype=BF, y=P, ldy=0, y_rows=20, weights=P, slots=P, tokens=10, top_k=2, n=16, out=P, ldo=0)
COMBINE_GRAD = dict(dtype=BF, grad_out=P, ldg=0, y=P, ldy=0, y_rows=20, weights=P, slots=P, tokens=10, top_k=2, n=16,
                    grad_y=P, ld_grad_y=0, grad_weights=P)

REFUSED = [
    ("route", ROUTE, dict(dtype=F8), UNSUPPORTED), ("route", ROUTE, dict(dtype=99), UNSUPPORTED),
    ("route", ROUTE, dict(tokens=-1), INVALID), ("route", ROUTE, dict(experts=0), INVALID),
    ("route", ROUTE, dict(experts=1025), INVALID), ("route", ROUTE, dict(top_k=0), INVALID),
    ("route", ROUTE, dict(top_k=9), INVALID), ("route", ROUTE, dict(experts=100, top_k=65), INVALID),
    ("route", ROUTE, dict(ld=7), INVALID), ("route", ROUTE, dict(tokens=1 << 30), SHAPE),
    ("route", ROUTE, dict(logits=None), INVALID), ("route", ROUTE, dict(offsets=None), INVALID),
    ("route", ROUTE, dict(slots=None), INVALID), ("route", ROUTE, dict(logits=P + 2), SHAPE),
    ("route", ROUTE, dict(rows=P + 1), SHAPE), ("route", ROUTE, dict(tokens=1000), WORKSPACE),
    ("route", ROUTE, dict(tokens=1000, workspace=P, workspace_bytes=8), WORKSPACE),
    ("route", ROUTE, dict(tokens=1000, workspace=P + 2, workspace_bytes=1 << 20), WORKSPACE),
    ("route_grad", ROUTE_GRAD, dict(dtype=F8), UNSUPPORTED), ("route_grad", ROUTE_GRAD, dict(ld_grad=5), INVALID),
    ("route_grad", ROUTE_GRAD, dict(expert_ids=None), INVALID), ("route_grad", ROUTE_GRAD, dict(top_k=9), INVALID),
    ("route_grad", ROUTE_GRAD, dict(grad_weights=P + 2), SHAPE),
    ("gemm_grouped", GROUPED, dict(op=3), INVALID), ("gemm_grouped", GROUPED, dict(op=-1), INVALID),
    ("gemm_grouped", GROUPED, dict(dtype=F32), UNSUPPORTED), ("gemm_grouped", GROUPED, dict(experts=0), INVALID),
    ("gemm_grouped", GROUPED, dict(experts=1025), INVALID), ("gemm_grouped", GROUPED, dict(total_rows=-1), INVALID),
    ("gemm_grouped", GROUPED, dict(total_rows=1 << 31), INVALID), ("gemm_grouped", GROUPED, dict(x_rows=9), INVALID),
    ("gemm_grouped", GROUPED, dict(n=0), INVALID), ("gemm_grouped", GROUPED, dict(k=-3), INVALID),
    ("gemm_grouped", GROUPED, dict(ldx=23), INVALID), ("gemm_grouped", GROUPED, dict(ldy=15), INVALID),
    ("gemm_grouped", GROUPED, dict(ldo=15), INVALID), ("gemm_grouped", GROUPED, dict(op=1, ldx=15), INVALID),
    ("gemm_grouped", GROUPED, dict(op=1, ldo=23), INVALID), ("gemm_grouped", GROUPED, dict(x=None), INVALID),
    ("gemm_grouped", GROUPED, dict(offsets=None), INVALID), ("gemm_grouped", GROUPED, dict(op=2, out=None), INVALID),
    ("gemm_grouped", GROUPED, dict(y=P + 1), SHAPE), ("gemm_grouped", GROUPED, dict(rows=P + 2), SHAPE),
    ("gemm_grouped", GROUPED, dict(n=1 << 16, k=1 << 15), SHAPE),
    ("gemm_w4", W4, dict(dtype=F32), UNSUPPORTED), ("gemm_w4", W4, dict(group=16), SHAPE),
    ("gemm_w4", W4, dict(group=48), SHAPE), ("gemm_w4", W4, dict(group=0), SHAPE),
    ("gemm_w4", W4, dict(offsets=None), INVALID), ("gemm_w4", W4, dict(q=None), INVALID),
    ("gemm_w4", W4, dict(scales=None), INVALID), ("gemm_w4", W4, dict(n=0), INVALID),
    ("gemm_w4", W4, dict(ldx=63), INVALID), ("gemm_w4", W4, dict(ldo=3), INVALID),
    ("gemm_w4", W4, dict(scales=P + 1), SHAPE), ("gemm_w4", W4, dict(x_rows=4), INVALID),
    ("combine", COMBINE, dict(dtype=F32), UNSUPPORTED), ("combine", COMBINE, dict(top_k=65), INVALID),
    ("combine", COMBINE, dict(tokens=-1), INVALID), ("combine", COMBINE, dict(n=0), INVALID),
    ("combine", COMBINE, dict(ldy=15), INVALID), ("combine", COMBINE, dict(slots=None), INVALID),
    ("combine", COMBINE, dict(out=P + 1), SHAPE), ("combine", COMBINE, dict(weights=P + 2), SHAPE),
    ("combine_grad", COMBINE_GRAD, dict(dtype=F32), UNSUPPORTED), ("combine_grad", COMBINE_GRAD, dict(ldg=3), INVALID),
    ("combine_grad", COMBINE_GRAD, dict(y=None), INVALID), ("combine_grad", COMBINE_GRAD, dict(grad_out=None), INVALID),
    ("combine_grad", COMBINE_GRAD, dict(grad_weights=P + 1), SHAPE),
]


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    capi.load_library().set_tuning("gemm_splits", None)   # a call that succeeds clears the thread's last error


@pytest.mark.parametrize("name, base, change, status", REFUSED,
                         ids=[f"{n}-{'-'.join(f'{k}={v}' for k, v in c.items())}" for n, _, c, _ in REFUSED])
def test_refused(name, base, change, status):
    lib = capi.load_library()
    with pytest.raises(capi.NativeLibraryError, match=f"mb_{name}") as err:
        getattr(lib, name)(**{**base, **change})
    assert err.value.status == status
    assert lib.handle.mb_last_error()


def test_route_workspace_size():
    lib = capi.load_library()
    assert lib.route_workspace_size(0, 8, 2) == lib.route_workspace_size(64, 8, 2) == 0
    assert lib.route_workspace_size(1 << 20, 1024, 64) <= 256 * 1024 * 4
    assert lib.route_workspace_size(100, 8, 9) == lib.route_workspace_size(-1, 8, 1) == 0


def test_limits_match_the_header():
    import re

    from teamredbench_amd.native import build

    text = (build.PACKAGE_DIR.parent / "include" / "mi355bench.h").read_text(encoding="utf-8")
    consts = {k: int(v) for k, v in re.findall(r"#define (MB_(?:ROUTE|GROUPED)_\w+) (\d+)", text)}
    assert consts == {"MB_ROUTE_MAX_EXPERTS": capi.ROUTE_MAX_EXPERTS, "MB_ROUTE_MAX_TOP_K": capi.ROUTE_MAX_TOP_K,
                      "MB_GROUPED_FORWARD": capi.GROUPED_FORWARD, "MB_GROUPED_GRAD_ROWS": capi.GROUPED_GRAD_ROWS,
                      "MB_GROUPED_GRAD_WEIGHTS": capi.GROUPED_GRAD_WEIGHTS}
