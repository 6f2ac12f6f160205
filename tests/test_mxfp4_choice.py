"""Which kernel a 4-bit product runs on, on the host: the shapes that the GPU tests mean for one kernel do reach it."""
import ctypes

import pytest

from amos_amd import _lib
from mxfp4_reach import FEW, FUSED, LONG

NAMES = {"float32": ("f32", _lib.AMOS_F32), "float16": ("f16", _lib.AMOS_F16), "bfloat16": ("bf16", _lib.AMOS_BF16)}


def chosen(M, N, K, a=_lib.AMOS_MXFP4):
    name = _lib.load().amos_mxfp4_gemm_kernel_name(ctypes.byref(_lib.Mxfp4GemmDesc(M, N, K, a, _lib.AMOS_F32)))
    return name and name.decode()


@pytest.mark.parametrize("kernel, M, N, K", LONG)
def test_tiles(kernel, M, N, K):
    assert K >= 9 * 256 and chosen(M, N, K) == kernel
    for _, dtype in NAMES.values():   # many dense rows: the same, behind their quantisation
        assert chosen(M, N, K, dtype) == kernel


@pytest.mark.parametrize("rt, M, N, K", FEW)
def test_few_rows(rt, M, N, K):
    assert chosen(M, N, K) == "amos_mx_gemm_few<mxfp4,%d,1>" % rt
    for dtype, (name, code) in NAMES.items():
        assert chosen(M, N, K, code) == "amos_mx_gemm_few<%s,%d,1>" % (name if FUSED[dtype](M, K) else "mxfp4", rt)


def test_few_rows_cover_both_ways_in():
    for dtype in FUSED:
        for rt in (1, 2, 3):
            assert any(FUSED[dtype](M, K) for r, M, N, K in FEW if r == rt)
    assert any(not FUSED["bfloat16"](M, K) for r, M, N, K in FEW if r == 3)


def test_others():
    assert chosen(17, 48, 384) == "amos_mx_gemm_few<mxfp4,1,2>"
    assert chosen(70, 1100, (1 << 23) + 300) == "amos_mx_gemm_few<mxfp4,1,2>"      # 32-bit offsets of the tiles
    assert chosen(9, 30000, 1 << 24) == "amos_mx_gemm_few<mxfp4,1,1>"
    assert chosen(0, 5, 5) is None and chosen(5, 5, 5, _lib.AMOS_I8) is None
