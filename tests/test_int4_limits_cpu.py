"""Calls at the end of the range of 32-bit row numbers are refused before anything is launched."""
import ctypes

import pytest

from vq_gemm_b200 import _lib

LAST = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib():
    from vq_gemm_b200.build import build
    build()
    return _lib.load()


@pytest.mark.parametrize("rows", [LAST, LAST - 15, LAST - 300])
def test_rows_that_32_bits_do_not_hold_rounded_up_to_a_tile(lib, rows):
    p = ctypes.c_void_p(4096)
    ws = 1 << 30
    assert lib.vqg_int4_gemm(p, p, p, None, p, 1, rows, 32, 32, 0, p, ws, None) == _lib.ERR_UNSUPPORTED
    assert lib.vqg_int4_gemm(p, p, p, None, p, rows, 16, 32, 32, 0, p, ws, None) == _lib.ERR_UNSUPPORTED
    assert lib.vqg_int4_dequant(p, p, None, p, 1, rows, 32, 32, 0, None) == _lib.ERR_UNSUPPORTED
    assert lib.vqg_int4_quantize(p, p, p, None, 1, rows, 32, 32, 0, None) == _lib.ERR_UNSUPPORTED
    assert lib.vqg_route_experts(p, None, p, p, rows, 1, 1, 0, 1, 1, 0, 0, 1.0, 0, None) == _lib.ERR_UNSUPPORTED
    assert lib.vqg_int4_experts(p, p, p, p, p, None, p, p, None, p, rows, 1, 1, 32, 32, 32, 32, 0, p, ws, None) == _lib.ERR_UNSUPPORTED
    inner = 0x3fffffe0
    assert lib.vqg_int4_experts(p, p, p, p, p, None, p, p, None, p, 1, 1, 1, 32, inner, 32, inner, 0, p, ws, None) == _lib.ERR_UNSUPPORTED
