"""What the microscaled 4-bit entry points refuse, before any device is touched (no GPU here)."""
from __future__ import annotations

import re

import pytest

from teamredbench_amd.native import build, capi

P = 1 << 20   # an address that is never read: every call below is refused first
BF, F32, F64, F8 = capi.DT_BFLOAT16, capi.DT_FLOAT32, capi.DT_FLOAT64, capi.DT_FLOAT8_E4M3FN
INVALID, UNSUPPORTED, SHAPE = capi.MB_ERR_INVALID_ARG, capi.MB_ERR_UNSUPPORTED, capi.MB_ERR_SHAPE

QUANTIZE = dict(dtype=BF, x=P, ldx=0, rows=10, columns=40, scale_rule=0, q=P, scales=P, qt=P, scales_t=P)
DEQUANTIZE = dict(dtype=BF, q=P, scales=P, rows=10, columns=40, out=P, ldo=0)
GEMM = dict(dtype=BF, x=P, x_scales=P, x_rows=10, rows=None, w=P, w_scales=P, out=P, ldo=0, offsets=P, experts=4,
            total_rows=10, n=16, k=64)

REFUSED = [
    ("mx4_quantize", QUANTIZE, dict(dtype=F64), UNSUPPORTED), ("mx4_quantize", QUANTIZE, dict(dtype=F8), UNSUPPORTED),
    ("mx4_quantize", QUANTIZE, dict(dtype=99), UNSUPPORTED), ("mx4_quantize", QUANTIZE, dict(scale_rule=2), INVALID),
    ("mx4_quantize", QUANTIZE, dict(scale_rule=-1), INVALID), ("mx4_quantize", QUANTIZE, dict(rows=-1), INVALID),
    ("mx4_quantize", QUANTIZE, dict(rows=1 << 31), INVALID), ("mx4_quantize", QUANTIZE, dict(columns=0), INVALID),
    ("mx4_quantize", QUANTIZE, dict(columns=1 << 31), INVALID), ("mx4_quantize", QUANTIZE, dict(ldx=39), INVALID),
    ("mx4_quantize", QUANTIZE, dict(rows=(1 << 31) - 1, columns=1 << 10), SHAPE),
    ("mx4_quantize", QUANTIZE, dict(q=None), INVALID), ("mx4_quantize", QUANTIZE, dict(scales=None), INVALID),
    ("mx4_quantize", QUANTIZE, dict(qt=None), INVALID), ("mx4_quantize", QUANTIZE, dict(scales_t=None), INVALID),
    ("mx4_quantize", QUANTIZE, dict(q=None, scales=None, qt=None, scales_t=None), INVALID),
    ("mx4_quantize", QUANTIZE, dict(x=None), INVALID), ("mx4_quantize", QUANTIZE, dict(x=P + 1), SHAPE),
    ("mx4_quantize", QUANTIZE, dict(dtype=F32, x=P + 2), SHAPE), ("mx4_quantize", QUANTIZE, dict(q=P + 8), SHAPE),
    ("mx4_quantize", QUANTIZE, dict(qt=P + 4), SHAPE), ("mx4_quantize", QUANTIZE, dict(scales=P + 2), SHAPE),
    ("mx4_quantize", QUANTIZE, dict(scales_t=P + 1), SHAPE),
    ("mx4_dequantize", DEQUANTIZE, dict(dtype=F64), UNSUPPORTED), ("mx4_dequantize", DEQUANTIZE, dict(rows=-1), INVALID),
    ("mx4_dequantize", DEQUANTIZE, dict(columns=0), INVALID), ("mx4_dequantize", DEQUANTIZE, dict(ldo=39), INVALID),
    ("mx4_dequantize", DEQUANTIZE, dict(q=None), INVALID), ("mx4_dequantize", DEQUANTIZE, dict(scales=None), INVALID),
    ("mx4_dequantize", DEQUANTIZE, dict(out=None), INVALID), ("mx4_dequantize", DEQUANTIZE, dict(out=P + 1), SHAPE),
    ("mx4_dequantize", DEQUANTIZE, dict(q=P + 8), SHAPE), ("mx4_dequantize", DEQUANTIZE, dict(scales=P + 2), SHAPE),
    ("gemm_mx4", GEMM, dict(dtype=F32), UNSUPPORTED), ("gemm_mx4", GEMM, dict(dtype=F8), UNSUPPORTED),
    ("gemm_mx4", GEMM, dict(experts=0), INVALID), ("gemm_mx4", GEMM, dict(experts=1025), INVALID),
    ("gemm_mx4", GEMM, dict(offsets=None), INVALID), ("gemm_mx4", GEMM, dict(total_rows=-1), INVALID),
    ("gemm_mx4", GEMM, dict(total_rows=1 << 31), INVALID), ("gemm_mx4", GEMM, dict(x_rows=9), INVALID),
    ("gemm_mx4", GEMM, dict(x_rows=-1, rows=P), INVALID), ("gemm_mx4", GEMM, dict(n=0), INVALID),
    ("gemm_mx4", GEMM, dict(n=1 << 30), INVALID), ("gemm_mx4", GEMM, dict(k=0), INVALID),
    ("gemm_mx4", GEMM, dict(k=capi.MX4_MAX_K + 1), SHAPE), ("gemm_mx4", GEMM, dict(ldo=15), INVALID),
    ("gemm_mx4", GEMM, dict(total_rows=(1 << 31) - 1, x_rows=(1 << 31) - 1, n=1 << 20), SHAPE),
    ("gemm_mx4", GEMM, dict(total_rows=(1 << 31) - 255, x_rows=(1 << 31) - 255, n=1, k=1), SHAPE),
    ("gemm_mx4", GEMM, dict(x=None), INVALID), ("gemm_mx4", GEMM, dict(x_scales=None), INVALID),
    ("gemm_mx4", GEMM, dict(w=None), INVALID), ("gemm_mx4", GEMM, dict(w_scales=None), INVALID),
    ("gemm_mx4", GEMM, dict(out=None), INVALID), ("gemm_mx4", GEMM, dict(out=P + 1), SHAPE),
    ("gemm_mx4", GEMM, dict(x=P + 8), SHAPE), ("gemm_mx4", GEMM, dict(x_scales=P + 2), SHAPE),
    ("gemm_mx4", GEMM, dict(w=P + 4), SHAPE), ("gemm_mx4", GEMM, dict(w_scales=P + 1), SHAPE),
    ("gemm_mx4", GEMM, dict(rows=P + 2), SHAPE), ("gemm_mx4", GEMM, dict(offsets=P + 1), SHAPE),
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


def test_constants_match_the_header():
    text = (build.PACKAGE_DIR.parent / "include" / "mi355bench.h").read_text(encoding="utf-8")
    consts = dict(re.findall(r"#define (MB_MX4_[A-Z_]+) (\d+)", text))
    assert int(consts["MB_MX4_SCALE_FLOOR"]) == capi.MX4_SCALE_FLOOR
    assert int(consts["MB_MX4_SCALE_FIT"]) == capi.MX4_SCALE_FIT
    assert int(consts["MB_MX4_MAX_K"]) == capi.MX4_MAX_K
    for columns in (1, 31, 127, 128, 129, 4096, 50257):
        assert capi.mx4_row_bytes(columns) == (columns + 127) // 128 * 64
        assert capi.mx4_row_scales(columns) == (columns + 127) // 128 * 4
