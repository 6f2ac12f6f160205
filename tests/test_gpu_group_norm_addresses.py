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
