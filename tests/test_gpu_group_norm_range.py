"""Group norm at the ends of fp32's range: what its sums hold is right, what they do not hold is NaN -- never a finite
result that the input has no part in."""
import pytest
import torch

from test_gpu_group_norm import check_forward, coefficients, make

pytestmark = pytest.mark.gpu
SHAPES = [(3, 6, 7, 32), (2, 64, 64, 256), (2, 6, 5, 2304), (1, 66, 65, 30)]       # one launch, two launches, odd channels


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sums_beyond_the_range_are_nan(gpu, shape, dt):
    """group 0 of the last image has deviations of 2^66, whose squares fp32 does not hold: that group is NaN, every other
    element has the bits it has without it"""
    from amos_amd import ops
    x = make("nhwc", shape, 2, dt).cuda()
    w, b = (t.cuda() for t in coefficients(shape[-1], 2))
    clean = ops.group_norm(x, 2, w, b, activation="silu", stats=True)
    x[-1, :, :, :shape[-1] // 2] *= 2.0 ** 66
    got = ops.group_norm(x, 2, w, b, activation="silu", stats=True)
    for t, plain in zip(got[::2], clean[::2]):     # y, rstd
        bad = torch.zeros_like(t, dtype=torch.bool)
        if t.dim() == 2:
            bad[-1, 0] = True
        else:
            bad[-1, :, :, :shape[-1] // 2] = True
        assert torch.equal(t.isnan(), bad) and torch.equal(t[~bad], plain[~bad])
    dx, dw, db = ops.group_norm_backward(torch.ones_like(x), x, got[1], got[2], 2, w, b, activation="silu")
    assert dx[-1, :, :, :shape[-1] // 2].isnan().all() and dx[:-1].isfinite().all() and dx[-1, :, :, shape[-1] // 2:].isfinite().all()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("power", [-70, 40])
def test_sums_inside_the_range(gpu, shape, power):
    """values of 2^40 (squares of 2^80 times some 2^20 elements) and of 2^-70 (squares of 2^-140 beside eps): the formula's"""
    w, b = coefficients(shape[-1], 4)
    check_forward(make("nhwc", shape, 3) * 2.0 ** power, 2, w, b, "silu", "nhwc", torch.float32)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("value", [2.0 ** 70, -2.0 ** 90])
def test_large_equal_values(gpu, shape, value):
    """a mean whose square fp32 does not hold, and no deviation: h is 0, whichever kernel runs"""
    from amos_amd import ops
    w, b = (t.cuda() for t in coefficients(shape[-1], 4))
    y, mean, rstd = ops.group_norm(torch.full(shape, value, device="cuda"), 2, w, b, stats=True)
    assert (mean == value).all() and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5), rtol=1e-6)
    assert torch.equal(y, b.expand(shape))


@pytest.mark.parametrize("shape", [(1, 12, 12, 64), (3, 12, 12, 64), (2, 64, 64, 256), (1, 66, 65, 30)])
def test_sums_of_coefficient_gradients_that_cancel(gpu, shape):
    """three neighbouring pixels, which three rows of threads take, with dy = 2^26, 1 and -2^26 and h = 1: every share is
    exact, and their sum is 1 where it is taken in more than fp32's 24 bits"""
    from amos_amd import ops
    c = shape[-1]
    dy = torch.zeros(shape, device="cuda")
    dy[0, 0, 0], dy[0, 0, 1], dy[0, 0, 2] = 2.0 ** 26, 1.0, -2.0 ** 26
    zero, one = torch.zeros(shape[0], 2, device="cuda"), torch.ones(shape[0], 2, device="cuda")
    dx, dw, db = ops.group_norm_backward(dy, torch.ones(shape, device="cuda"), zero, one, 2, torch.ones(c, device="cuda"), torch.zeros(c, device="cuda"))
    assert (dw == 1).all() and (db == 1).all() and dx.isfinite().all()
