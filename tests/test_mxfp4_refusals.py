"""What the microscaled 4-bit operators and group norm refuse, and the layouts of their structs, on the
host: no call here reaches a launch."""
import ctypes

import pytest
import torch

from amos_amd import _lib, ops

BUF = ctypes.create_string_buffer(4096 + 256)
AT = (ctypes.addressof(BUF) + 255) // 256 * 256


def test_struct_layouts():
    assert ctypes.sizeof(_lib.Mxfp4Desc) == 24 and ctypes.sizeof(_lib.Mxfp4GemmDesc) == 32
    assert ctypes.sizeof(_lib.Mxfp4Epilogue) == 24 and ctypes.sizeof(_lib.GroupNormDesc) == 5 * 8 + 8 * 4
    assert _lib.GroupNormDesc.eps.offset == 64


def test_pitch():
    lib = _lib.load()
    for cols, want in ((1, 64), (32, 64), (127, 64), (128, 64), (129, 128), (4096, 2048), (1 << 30, 1 << 29)):
        assert lib.amos_mxfp4_pitch(cols) == want == ops.mxfp4_pitch(cols)
    assert lib.amos_mxfp4_pitch(0) == 0
    with pytest.raises(ValueError):
        ops.mxfp4_pitch(0)


@pytest.mark.parametrize("change, code, text", [
    (dict(rows=0), _lib.AMOS_ERR_BAD_ARG, "0 x 64"),
    (dict(cols=-1), _lib.AMOS_ERR_BAD_ARG, "x -1"),
    (dict(rows=1 << 31), _lib.AMOS_ERR_UNSUPPORTED, "2^31"),
    (dict(dtype=_lib.AMOS_I8), _lib.AMOS_ERR_UNSUPPORTED, "dtype 2"),
    (dict(axis=2), _lib.AMOS_ERR_BAD_ARG, "axis 2"),
    (dict(x=None), _lib.AMOS_ERR_BAD_ARG, "null"),
    (dict(codes=AT + 8), _lib.AMOS_ERR_BAD_ARG, "16-byte"),
    (dict(scales=AT + 2), _lib.AMOS_ERR_BAD_ARG, "4-byte"),
    (dict(x=AT + 1), _lib.AMOS_ERR_BAD_ARG, "misaligned"),
    (dict(axis=0, rows=65536 * 256), _lib.AMOS_ERR_UNSUPPORTED, "axis 0"),
])
def test_quantize_refuses(change, code, text):
    lib = _lib.load()
    a = dict(rows=4, cols=64, dtype=_lib.AMOS_F32, axis=1, x=AT, codes=AT, scales=AT)
    a.update(change)
    d = _lib.Mxfp4Desc(a["rows"], a["cols"], a["dtype"], a["axis"])
    assert lib.amos_mxfp4_quantize(ctypes.byref(d), a["x"], a["codes"], a["scales"], None) == code
    assert text in lib.amos_last_error().decode()
    if a["axis"] != 0:
        assert lib.amos_mxfp4_dequantize(ctypes.byref(d), a["codes"], a["scales"], a["x"], None) == code
    assert lib.amos_mxfp4_quantize(None, AT, AT, AT, None) == _lib.AMOS_ERR_BAD_ARG


def test_dequantize_refuses_the_other_axis():
    lib = _lib.load()
    d = _lib.Mxfp4Desc(4, 64, _lib.AMOS_F32, 0)
    assert lib.amos_mxfp4_dequantize(ctypes.byref(d), AT, AT, AT, None) == _lib.AMOS_ERR_BAD_ARG


@pytest.mark.parametrize("change, code, text", [
    (dict(M=0), _lib.AMOS_ERR_BAD_ARG, "extents"),
    (dict(K=1 << 31), _lib.AMOS_ERR_UNSUPPORTED, "2^31"),
    (dict(N=1 << 30), _lib.AMOS_ERR_UNSUPPORTED, "2^30"),
    (dict(a_dtype=_lib.AMOS_I8), _lib.AMOS_ERR_UNSUPPORTED, "A of dtype"),
    (dict(out_dtype=_lib.AMOS_I32), _lib.AMOS_ERR_UNSUPPORTED, "output dtype"),
    (dict(A=None), _lib.AMOS_ERR_BAD_ARG, "null"),
    (dict(a_scales=None), _lib.AMOS_ERR_BAD_ARG, "null"),
    (dict(C=None), _lib.AMOS_ERR_BAD_ARG, "null"),
    (dict(B=AT + 4), _lib.AMOS_ERR_BAD_ARG, "16-byte"),
    (dict(b_scales=AT + 1), _lib.AMOS_ERR_BAD_ARG, "4-byte"),
    (dict(C=AT + 2), _lib.AMOS_ERR_BAD_ARG, "misaligned"),
    (dict(N=(1 << 30) - 1), _lib.AMOS_ERR_UNSUPPORTED, "results"),          # grids of 2^32 threads and more
    (dict(N=1 << 28, K=1 << 24), _lib.AMOS_ERR_UNSUPPORTED, "results"),
    (dict(bias_dtype=_lib.AMOS_I8), _lib.AMOS_ERR_UNSUPPORTED, "bias"),
    (dict(add_dtype=_lib.AMOS_I32), _lib.AMOS_ERR_UNSUPPORTED, "added operand"),
])
def test_product_refuses(change, code, text):
    lib = _lib.load()
    a = dict(M=4, N=8, K=64, a_dtype=_lib.AMOS_MXFP4, out_dtype=_lib.AMOS_F32, A=AT, a_scales=AT, B=AT, b_scales=AT, C=AT, bias_dtype=_lib.AMOS_F32, add_dtype=_lib.AMOS_F32)
    a.update(change)
    d = _lib.Mxfp4GemmDesc(a["M"], a["N"], a["K"], a["a_dtype"], a["out_dtype"])
    e = _lib.Mxfp4Epilogue(AT, AT, a["bias_dtype"], a["add_dtype"])
    assert lib.amos_mxfp4_gemm(ctypes.byref(d), ctypes.byref(e), a["A"], a["a_scales"], a["B"], a["b_scales"], a["C"], None, 0, None) == code
    assert text in lib.amos_last_error().decode()


def test_product_wants_its_workspace():
    lib = _lib.load()
    d = _lib.Mxfp4GemmDesc(500, 8, 200, _lib.AMOS_BF16, _lib.AMOS_F32)
    need = lib.amos_mxfp4_gemm_workspace_bytes(ctypes.byref(d))
    assert need >= 500 * (128 + 8)     # A's codes and scales
    for ptr, size in ((None, need), (AT, need - 1), (AT + 16, need)):
        assert lib.amos_mxfp4_gemm(ctypes.byref(d), None, AT, None, AT, AT, AT, ptr, size, None) == _lib.AMOS_ERR_WORKSPACE
        assert b"workspace" in lib.amos_last_error()
    bad = _lib.Mxfp4GemmDesc(0, 8, 200, _lib.AMOS_BF16, _lib.AMOS_F32)
    assert lib.amos_mxfp4_gemm_workspace_bytes(ctypes.byref(bad)) == 0


def norm_desc(**change):
    a = dict(N=2, C=32, D=1, H=4, W=4, groups=4, activation=_lib.AMOS_ACT_NONE, x_dtype=_lib.AMOS_F32, y_dtype=_lib.AMOS_F32,
             affine_dtype=_lib.AMOS_F32, layout=_lib.AMOS_LAYOUT_NHWC, eps=1e-5)
    a.update(change)
    return _lib.GroupNormDesc(**a)


@pytest.mark.parametrize("change, code, text", [
    (dict(N=0), _lib.AMOS_ERR_BAD_ARG, "extents"),
    (dict(groups=5), _lib.AMOS_ERR_BAD_ARG, "5 groups"),
    (dict(groups=0), _lib.AMOS_ERR_BAD_ARG, "0 groups"),
    (dict(layout=_lib.AMOS_LAYOUT_NCHW), _lib.AMOS_ERR_UNSUPPORTED, "layout"),
    (dict(activation=7), _lib.AMOS_ERR_UNSUPPORTED, "activation"),
    (dict(x_dtype=_lib.AMOS_I8), _lib.AMOS_ERR_UNSUPPORTED, "dtypes"),
    (dict(y_dtype=_lib.AMOS_MXFP4), _lib.AMOS_ERR_UNSUPPORTED, "dtypes"),
    (dict(eps=-1.0), _lib.AMOS_ERR_BAD_ARG, "eps"),
    (dict(eps=float("nan")), _lib.AMOS_ERR_BAD_ARG, "eps"),
    (dict(H=1 << 20, W=1 << 20), _lib.AMOS_ERR_UNSUPPORTED, "2^28"),
    (dict(N=1 << 20, H=1 << 12, C=1 << 12), _lib.AMOS_ERR_UNSUPPORTED, "2^40"),
    (dict(N=1 << 26, H=1, W=1), _lib.AMOS_ERR_UNSUPPORTED, "images"),       # a grid of 2^32 threads
])
def test_group_norm_refuses(change, code, text):
    lib = _lib.load()
    d = norm_desc(**change)
    assert lib.amos_group_norm_workspace_bytes(ctypes.byref(d), 0) == 0
    assert lib.amos_group_norm(ctypes.byref(d), AT, AT, AT, AT, AT, AT, AT, 1 << 30, None) == code
    assert text in lib.amos_last_error().decode()
    assert lib.amos_group_norm_backward(ctypes.byref(d), AT, AT, AT, AT, AT, AT, AT, AT, AT, AT, 1 << 30, None) == code


def test_group_norm_refuses_pointers():
    lib = _lib.load()
    d = norm_desc()
    assert lib.amos_group_norm(ctypes.byref(d), None, None, None, AT, None, None, AT, 1 << 30, None) == _lib.AMOS_ERR_BAD_ARG
    assert lib.amos_group_norm(ctypes.byref(d), AT + 2, None, None, AT, None, None, AT, 1 << 30, None) == _lib.AMOS_ERR_BAD_ARG
    assert lib.amos_group_norm_backward(ctypes.byref(d), AT, AT, None, None, None, AT, AT, None, None, AT, 1 << 30, None) == _lib.AMOS_ERR_BAD_ARG
    big = norm_desc(N=4, H=64, W=64, C=256, groups=32)
    need = lib.amos_group_norm_workspace_bytes(ctypes.byref(big), 1)
    assert need > 0
    for ptr, size in ((None, need), (AT, 8)):
        assert lib.amos_group_norm_backward(ctypes.byref(big), AT, AT, AT, AT, AT, AT, AT, AT, AT, ptr, size, None) == _lib.AMOS_ERR_WORKSPACE
        assert b"workspace" in lib.amos_last_error()


def test_host_tensors_are_refused():
    x = torch.zeros(4, 64)
    u = torch.zeros(4, 64, dtype=torch.uint8)
    n = torch.zeros(1, 2, 2, 8)
    for call in (lambda: ops.mxfp4_quantize(x), lambda: ops.Mxfp4(u, u[:, :4].contiguous(), 64), lambda: ops.group_norm(n, 2),
                 lambda: ops.group_norm_backward(n, n, x, x, 2)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    for call in (lambda: ops.mxfp4_gemm(x, x), lambda: ops.mxfp4_dequantize(x)):
        with pytest.raises(ValueError, match="Mxfp4"):
            call()
