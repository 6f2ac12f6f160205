"""Group norm and its gradient on tensors that start anywhere: the plan does not look at addresses, so the results have the
bits that aligned tensors give, and the elements around them stay."""
import pytest
import torch

from test_gpu_group_norm import DTYPES, coefficients, make

pytestmark = pytest.mark.gpu


def moved(t, by):
    """t's values in a view that starts `by` elements into its memory"""
    room = torch.zeros(t.numel() + 8, dtype=t.dtype, device="cuda")
    view = room[by:by + t.numel()].view(t.shape)
    view.copy_(t)
    return view


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape, groups", [((2, 12, 11, 64), 8), ((1, 40, 50, 24), 3), ((4, 64, 64, 128), 32), ((3, 5, 7, 30), 5), ((1, 66, 65, 30), 3), ((1, 9, 8, 4104), 1)])
def test_misaligned(gpu, shape, groups, dt):
    from amos_amd import ops
    w, b = [t.cuda() for t in coefficients(shape[-1], 1)]
    x, dy = make("nhwc", shape, 3, dt).cuda(), make("nhwc", shape, 4, dt).cuda()
    y, mean, rstd = ops.group_norm(x, groups, w, b, activation="silu", stats=True)
    grads = ops.group_norm_backward(dy, x, mean, rstd, groups, w, b, activation="silu")
    for i, j, k in ((1, 3, 2), (3, 1, 5), (2, 7, 1)):
        out = torch.full((x.numel() + 8,), 7.0, dtype=dt, device="cuda")
        got = ops.group_norm(moved(x, i), groups, moved(w, j), moved(b, k), activation="silu", out=out[j:j + x.numel()].view(shape), stats=True)
        for p, q in zip(got, (y, mean, rstd)):
            assert torch.equal(p, q)
        assert (out[:j] == 7).all() and (out[j + x.numel():] == 7).all()
        back = ops.group_norm_backward(moved(dy, j), moved(x, i), moved(mean, k), moved(rstd, i), groups, moved(w, k), moved(b, j), activation="silu")
        for p, q in zip(back, grads):
            assert torch.equal(p, q)


@pytest.mark.parametrize("over", ["dy", "x"])
@pytest.mark.parametrize("shape, groups", [((2, 12, 11, 64), 8), ((4, 64, 64, 128), 32), ((1, 66, 65, 30), 3), ((1, 9, 8, 4104), 1)])
def test_gradient_in_place(gpu, shape, groups, over):
    """the C call's dx may be dy or x: one launch and two, several chunks and tiles"""
    import ctypes
    from amos_amd import _lib, ops
    lib = _lib.load()
    w, b = [t.cuda() for t in coefficients(shape[-1], 1)]
    x, dy = make("nhwc", shape, 3).cuda(), make("nhwc", shape, 4).cuda()
    _, mean, rstd = ops.group_norm(x, groups, w, b, activation="silu", stats=True)
    want = ops.group_norm_backward(dy, x, mean, rstd, groups, w, b, activation="silu")
    n, h, wide, c = shape
    d = _lib.GroupNormDesc(N=n, C=c, D=1, H=h, W=wide, groups=groups, activation=_lib.AMOS_ACT_SILU, x_dtype=_lib.AMOS_F32, y_dtype=_lib.AMOS_F32,
                           affine_dtype=_lib.AMOS_F32, layout=_lib.AMOS_LAYOUT_NHWC, eps=1e-5)
    need = lib.amos_group_norm_workspace_bytes(ctypes.byref(d), 1)
    ws = torch.empty(need + 8, dtype=torch.uint8, device="cuda")
    dw, db = torch.empty_like(w), torch.empty_like(b)
    dx = dict(dy=dy, x=x)[over]
    at = [t.data_ptr() for t in (dy, x, w, b, mean, rstd, dx, dw, db, ws)]
    _lib.check(lib.amos_group_norm_backward(ctypes.byref(d), *at, need, torch.cuda.current_stream().cuda_stream))
    for p, q in zip((dx, dw, db), want):
        assert torch.equal(p, q)
