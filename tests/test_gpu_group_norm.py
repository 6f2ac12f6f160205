"""Group norm with an activation, channels last, and its gradient, against their formulas in 64 bits.

Tolerances count roundings of 2^-24.  The mean of a group is a tree of means: L = 64 covers the sequential
additions of a lane, a team and a join at the sizes here, so it is off by L 2^-24 max|x|, the deviation's
factor rstd by L 2^-24 relative, h by L 2^-24 (max|x| rstd + |h|); an output is one more rounding to its
type.  exp(-z) is off by (|z| + 4) 2^-23 relative."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 2.0 ** -24
L = 64
LAYOUTS = {"nhwc": (0, 3, 1, 2), "ndhwc": (0, 4, 1, 2, 3), "hwnc": (2, 3, 0, 1), "dhwnc": (3, 4, 0, 1, 2)}   # -> NC...


def back(layout, t):
    return t.permute(*np.argsort(LAYOUTS[layout]).tolist())


def formula(x, groups, w, b, eps, act, layout):
    """x in 64 bits in `layout` -> y in `layout`, mean, rstd [N, G], z and h in NC..."""
    v = x.permute(*LAYOUTS[layout])
    n, c = v.shape[:2]
    g = v.reshape(n, groups, -1)
    mean, var = g.mean(-1), g.var(-1, unbiased=False)
    rstd = (var + eps) ** -0.5
    h = ((g - mean[..., None]) * rstd[..., None]).reshape(v.shape)
    shape = (1, c) + (1,) * (v.dim() - 2)
    z = h * w.reshape(shape) + b.reshape(shape)
    y = z if act is None else z.clamp(min=0) if act == "relu" else z * torch.sigmoid(z)
    return back(layout, y), mean, rstd, z, h


def make(layout, shape, seed, dtype=torch.float32, offset=0.5):
    """values whose mean differs by channel, in `layout`"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    c = shape[-1]
    return (x * torch.exp(0.3 * torch.randn(c, generator=g)) + offset * torch.randn(c, generator=g)).to(dtype)


def coefficients(c, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed + 1)
    return (1 + 0.2 * torch.randn(c, generator=g)).to(dtype), (0.3 * torch.randn(c, generator=g)).to(dtype)


def check_forward(x, groups, w, b, act, layout, out, eps=1e-5):
    from amos_amd import ops
    dev = lambda t: None if t is None else t.cuda()
    y, mean, rstd = ops.group_norm(x.cuda(), groups, dev(w), dev(b), eps=eps, activation=act, layout=layout, out_dtype=out, stats=True)
    c = x.shape[-1]
    wd = torch.ones(c, dtype=torch.float64) if w is None else w.double()
    bd = torch.zeros(c, dtype=torch.float64) if b is None else b.double()
    want, m, r, z, h = formula(x.double(), groups, wd, bd, eps, act, layout)
    top = x.double().permute(*LAYOUTS[layout]).reshape(m.shape[0], groups, -1).abs().amax(-1)
    assert y.dtype == out and mean.dtype == rstd.dtype == torch.float32
    assert ((mean.cpu().double() - m).abs() <= L * E * top).all()
    # the deviation is of x - mean: the mean's own error enters squared, and by the rounding of x - mean
    assert ((rstd.cpu().double() - r).abs() <= r * (L * E + (L * E * top * r) ** 2 + 2 * E * top * r)).all()
    zabs = z.abs()
    spread = (top * r).amax()
    err_z = L * E * (spread + h.abs() * (1 + 2 * E * spread / E / L)) * wd.abs().amax() + 3 * E * (zabs + bd.abs().amax())
    slope = 1.1   # the steepest that silu gets
    err = back(layout, err_z * slope + (2 * (zabs + 4) * 2 * E * zabs if act == "silu" else 0))
    half = torch.finfo(out).eps / 2
    assert ((y.cpu().double() - want).abs() <= err * (1 + half) + half * want.abs() + torch.finfo(out).tiny).all()
    return y, mean, rstd


# layout, shape, groups: single elements, one pixel, one channel a group, odd widths, groups across vectors, many
# channels (several tiles, groups wider than a tile), long images (many chunks), all layouts
SHAPES = [("nhwc", (1, 1, 1, 1), 1), ("nhwc", (2, 1, 1, 64), 4), ("nhwc", (1, 7, 7, 512), 32), ("nhwc", (3, 13, 17, 120), 24),
          ("nhwc", (2, 5, 3, 7), 7), ("nhwc", (2, 33, 31, 48), 16), ("nhwc", (1, 64, 65, 8), 8), ("nhwc", (2, 56, 56, 64), 32),
          ("nhwc", (2, 6, 5, 2304), 32), ("nhwc", (1, 4, 9, 4100), 1), ("nhwc", (2, 3, 3, 2500), 5), ("nhwc", (1, 3, 5, 6144), 2),
          ("nhwc", (5, 9, 8, 40), 5), ("ndhwc", (2, 3, 5, 7, 24), 3), ("hwnc", (9, 8, 3, 64), 16), ("dhwnc", (2, 4, 5, 3, 33), 11),
          ("nhwc", (2, 128, 130, 16), 2), ("hwnc", (40, 41, 6, 128), 4), ("nhwc", (8, 40, 40, 64), 8), ("nhwc", (1, 70, 66, 512), 32),
          ("nhwc", (2, 71, 67, 360), 15), ("hwnc", (67, 71, 1, 330), 11), ("nhwc", (1, 66, 65, 4224), 3)]


@pytest.mark.parametrize("layout, shape, groups", SHAPES)
@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_forward(gpu, layout, shape, groups, act):
    for i, (dt, out) in enumerate([(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)]):
        w, b = coefficients(shape[-1], i, [torch.float32, torch.bfloat16, torch.float32, torch.float16][i])
        check_forward(make(layout, shape, i, dt), groups, w, b, act, layout, out)
    check_forward(make(layout, shape, 9), groups, None, None, act, layout, torch.float16)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("out", DTYPES)
def test_every_pair_of_types(gpu, dt, out):
    for shape in ((2, 9, 7, 32), (2, 9, 7, 30)):
        w, b = coefficients(shape[-1], 3)
        check_forward(make("nhwc", shape, 4, dt), 2, w, None, "silu", "nhwc", out)
        check_forward(make("nhwc", shape, 4, dt), 2, None, b, "silu", "nhwc", out)
        check_gradient(make("nhwc", shape, 4, dt), 2, w, b, "silu", "nhwc", out)


def test_large_mean(gpu):
    """a mean a thousand times the deviation, which a difference of large sums would lose"""
    x = make("nhwc", (2, 40, 41, 32), 1) + 1000
    w, b = coefficients(32, 1)
    check_forward(x, 4, w, b, "silu", "nhwc", torch.float32)
    x = torch.full((1, 12, 12, 16), 3.25)          # no deviation at all: h is 0
    from amos_amd import ops
    y, mean, rstd = ops.group_norm(x.cuda(), 2, stats=True)
    assert not y.any() and (mean == 3.25).all() and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5), rtol=1e-6)


def check_gradient(x, groups, w, b, act, layout, ytype, eps=1e-5):
    from amos_amd import ops
    c = x.shape[-1]
    g = torch.Generator().manual_seed(77)
    dy = torch.randn(x.shape, generator=g).to(ytype)
    leaves = [x.double().requires_grad_(), (torch.ones(c) if w is None else w).double().requires_grad_(),
              (torch.zeros(c) if b is None else b).double().requires_grad_()]
    y, mean, rstd, z, h = formula(leaves[0], groups, leaves[1], leaves[2], eps, act, layout)
    if act == "relu":   # an element on the corner's other side than in 64 bits has another gradient: keep away from it
        near = back(layout, z.abs() < 1e-4)
        dy = torch.where(near, torch.zeros_like(dy), dy).contiguous()
    want = torch.autograd.grad(y, leaves, dy.double())
    dev = lambda t: None if t is None else t.cuda()
    dx, dw, db = ops.group_norm_backward(dy.cuda(), x.cuda(), mean.detach().float().cuda(), rstd.detach().float().cuda(), groups, dev(w), dev(b),
                                         activation=act, layout=layout)
    assert dx.dtype == x.dtype and (dw is None) == (w is None) and (db is None) == (b is None)
    with torch.no_grad():
        rows = lambda t: t.permute(*LAYOUTS[layout])
        d = rows(dy.double()).abs() * 1.1                      # |act'| <= 1.1
        top = rows(x.double()).reshape(mean.shape[0], groups, -1).abs().amax(-1)
        spread = float((top * rstd).amax())                    # mean and rstd were rounded to fp32: h is off by spread + |h|
        err_h = 4 * E * (spread + h.abs())
        err_d = d * (E * (8 + 4 * (z.abs() + 4)) + err_h * leaves[1].abs().amax())   # |act''| <= 1/2, and the factors' own
        sums = lambda t: t.sum([i for i in range(t.dim()) if i != 1])
        if db is not None:
            assert ((db.cpu().double() - want[2]).abs() <= sums(err_d + L * E * d)).all()
        if dw is not None:
            assert ((dw.cpu().double() - want[1]).abs() <= sums(err_d * h.abs() + d * err_h + L * E * d * h.abs())).all()
        wide = lambda t: t.reshape(mean.shape[0], groups, -1).mean(-1)
        ww = leaves[1].abs().reshape((1, c) + (1,) * (z.dim() - 2))
        spreadout = lambda t: t[..., None].expand(-1, -1, z[0].numel() // groups).reshape(z.shape)
        e1 = spreadout(wide((err_d + (L + 2) * E * d) * ww))
        e2 = spreadout(wide((err_d * h.abs() + d * err_h + (L + 2) * E * d * h.abs()) * ww))
        m2 = spreadout(wide(d * h.abs() * ww))
        r = spreadout(rstd)
        err = back(layout, r * (err_d * ww + e1 + h.abs() * e2 + err_h * m2 + 8 * E * (d * ww + spreadout(wide(d * ww)) + h.abs() * m2)))
        half = torch.finfo(x.dtype).eps / 2
        assert ((dx.cpu().double() - want[0]).abs() <= err * (1 + half) + half * want[0].abs() + torch.finfo(x.dtype).tiny).all()
    return dy, dx, dw, db


@pytest.mark.parametrize("layout, shape, groups", SHAPES)
@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_gradient(gpu, layout, shape, groups, act):
    for i, (dt, out) in enumerate([(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)]):
        w, b = coefficients(shape[-1], i, [torch.float32, torch.bfloat16, torch.float32, torch.float16][i])
        check_gradient(make(layout, shape, i, dt), groups, w, b, act, layout, out)
    check_gradient(make(layout, shape, 9), groups, None, None, act, layout, torch.float32)


@pytest.mark.parametrize("act", [None, "silu"])
def test_gradient_against_differences(gpu, act):
    """the change of sum(y dy) along a direction, from the formula at both ends of a short step: its error is of
    the step's square (1e-8 of values near 1) against the gradient's roundings, 1e-5 of the same sums"""
    shape, groups = (2, 9, 11, 24), 6
    x, (w, b) = make("nhwc", shape, 5), coefficients(24, 5)
    dy, dx, dw, db = check_gradient(x, groups, w, b, act, "nhwc", torch.float32)
    g = torch.Generator().manual_seed(8)
    step = 1e-4
    v = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (x, w, b)]
    total = lambda s: (formula(x.double() + s * v[0], groups, w.double() + s * v[1], b.double() + s * v[2], 1e-5, act, "nhwc")[0] * dy.double()).sum()
    change = (total(step) - total(-step)) / (2 * step)
    ours = sum((t.cpu().double() * d).sum() for t, d in zip((dx, dw, db), v))
    size = sum((t.cpu().double() * d).abs().sum() for t, d in zip((dx, dw, db), v))
    assert abs(float(change - ours)) <= 1e-5 * float(size)


def test_infinities_and_nan_stay_in_their_group(gpu):
    from amos_amd import ops
    x = make("nhwc", (3, 6, 7, 32), 2)
    clean = ops.group_norm(x.cuda(), 4, activation="relu")
    x[0, 2, 3, 5] = float("nan")       # group 0 of image 0
    x[2, 0, 0, 31] = float("inf")      # group 3 of image 2
    y = ops.group_norm(x.cuda(), 4, activation="relu")
    bad = torch.zeros(3, 6, 7, 32, dtype=torch.bool)
    bad[0, :, :, :8] = True
    bad[2, :, :, 24:] = True
    assert torch.equal(y.isnan().cpu(), bad)
    assert torch.equal(y.cpu()[~bad], clean.cpu()[~bad])


@pytest.mark.parametrize("shape", [(2, 6, 7, 32), (2, 64, 64, 256)])       # one launch, two launches
def test_gradient_without_an_activation_ignores_the_bias(gpu, shape):
    """y's gradient by x does not know the bias, whatever it holds; relu stops at -infinity and passes NaN on"""
    from amos_amd import ops
    x, dy = make("nhwc", shape, 3).cuda(), make("nhwc", shape, 4).cuda()
    w, b = (t.cuda() for t in coefficients(shape[-1], 3))
    odd = b.clone()
    odd[3], odd[17], odd[25] = float("nan"), float("-inf"), float("inf")
    _, mean, rstd = ops.group_norm(x, 4, w, b, stats=True)
    for one, two in zip(ops.group_norm_backward(dy, x, mean, rstd, 4, w, b), ops.group_norm_backward(dy, x, mean, rstd, 4, w, odd)):
        assert torch.equal(one, two)
    _, dw, db = ops.group_norm_backward(dy, x, mean, rstd, 4, w, odd, activation="relu")
    plain, plain_b = ops.group_norm_backward(dy, x, mean, rstd, 4, w, b)[1:]
    assert db[17] == 0 and dw[17] == 0
    for c in (3, 25):
        assert db[c] == plain_b[c] and dw[c] == plain[c]


@pytest.mark.parametrize("shape, groups", [((2, 12, 11, 64), 8), ((1, 40, 50, 24), 3), ((4, 64, 64, 128), 32)])
def test_in_place_misaligned_stream_and_repetition(gpu, shape, groups):
    from amos_amd import ops
    w, b = [t.cuda() for t in coefficients(shape[-1], 1)]
    for dt in DTYPES:
        x = make("nhwc", shape, 3, dt).cuda()
        want, mean, rstd = ops.group_norm(x, groups, w, b, activation="silu", stats=True)
        dy = make("nhwc", shape, 4, dt).cuda()
        grads = ops.group_norm_backward(dy, x, mean, rstd, groups, w, b, activation="silu")
        # again: the same bits
        assert torch.equal(ops.group_norm(x, groups, w, b, activation="silu"), want)
        for p, q in zip(ops.group_norm_backward(dy, x, mean, rstd, groups, w, b, activation="silu"), grads):
            assert torch.equal(p, q)
        # on another stream
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        y = ops.group_norm(x, groups, w, b, activation="silu", stream=s)
        g = ops.group_norm_backward(dy, x, mean, rstd, groups, w, b, activation="silu", stream=s)
        s.synchronize()
        assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(g, grads))
        # off the 16-byte grid (the element-wise kernels, sums in another order): a few roundings of values near 1,
        # amplified at most tenfold, and one of the type; the elements around the result stay
        room, out = torch.zeros(x.numel() + 8, dtype=dt, device="cuda"), torch.full((x.numel() + 8,), 7.0, dtype=dt, device="cuda")
        view = room[1:1 + x.numel()].view(shape)
        view.copy_(x)
        y = ops.group_norm(view, groups, w, b, activation="silu", out=out[3:3 + x.numel()].view(shape))
        assert torch.allclose(y.float(), want.float(), rtol=2 * torch.finfo(dt).eps, atol=1e-5)
        assert (out[:3] == 7).all() and (out[3 + x.numel():] == 7).all()
        # in place
        same = x.clone()
        assert ops.group_norm(same, groups, w, b, activation="silu", out=same) is same and torch.equal(same, want)


def test_captured(gpu):
    """forward and gradient in a graph, replayed on changing inputs between eager calls; the workspaces of two
    graphs are their own"""
    from amos_amd import ops
    shape, groups = (2, 30, 31, 64), 16
    w, b = [t.cuda() for t in coefficients(64, 1)]

    def both(x, dy):
        y, mean, rstd = ops.group_norm(x, groups, w, b, activation="silu", out_dtype=torch.float32, stats=True)
        return (y,) + ops.group_norm_backward(dy, x, mean, rstd, groups, w, b, activation="silu")

    ins = [(torch.zeros(shape, dtype=torch.bfloat16, device="cuda"), torch.zeros(shape, device="cuda")) for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for i in ins:
            both(*i)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for i in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both(*i))
        graphs.append(g)
    for turn in range(3):
        for k, (x, dy) in enumerate(ins):
            x.copy_(make("nhwc", shape, 10 * turn + k))
            dy.copy_(make("nhwc", shape, 10 * turn + k + 5))
        for g in graphs:
            g.replay()
        for i, got in zip(ins, outs):
            for p, q in zip(got, both(*i)):
                assert torch.equal(p, q)
        torch.cuda.synchronize()


def test_more_than_32_bits_of_bytes(gpu):
    """the last image of a batch beyond 2^32 bytes"""
    from amos_amd import ops
    n, shape = 2100, (64, 64, 256)
    x = torch.zeros((n,) + shape, dtype=torch.bfloat16, device="cuda")
    last = make("nhwc", (1,) + shape, 3, torch.bfloat16).cuda()
    x[-1] = last[0]
    w, b = [t.cuda() for t in coefficients(256, 1)]
    want, m, r = ops.group_norm(last, 32, w, b, activation="silu", stats=True)
    y, mean, rstd = ops.group_norm(x, 32, w, b, activation="silu", stats=True)
    # (another number of chunks: sums in another order)
    assert torch.allclose(mean[-1], m[0], rtol=1e-5, atol=1e-6) and torch.allclose(rstd[-1], r[0], rtol=1e-5)
    assert torch.allclose(y[-1].float(), want[0].float(), rtol=2 ** -7, atol=1e-5)
    dy = torch.zeros_like(x)
    dy[-1] = 1.5
    dx, dw, db = ops.group_norm_backward(dy, x, mean, rstd, 32, w, b, activation="silu")
    one = ops.group_norm_backward(dy[-1:], last, mean[-1:], rstd[-1:], 32, w, b, activation="silu")
    assert torch.allclose(dx[-1].float(), one[0][0].float(), rtol=2 ** -7, atol=1e-5)
    assert torch.allclose(dw, one[1], rtol=1e-4, atol=1e-2) and torch.allclose(db, one[2], rtol=1e-4, atol=1e-2)
    assert not dx[:-1].any()


def test_refusals_on_device_tensors(gpu):
    from amos_amd import ops
    x = torch.zeros(2, 3, 3, 8, device="cuda")
    s = torch.zeros(2, 2, device="cuda")
    for bad in (lambda: ops.group_norm(x, 3), lambda: ops.group_norm(x, 0), lambda: ops.group_norm(x, 2, layout="nchw"), lambda: ops.group_norm(x, 2, layout="ndhwc"),
                lambda: ops.group_norm(x, 2, activation="gelu"), lambda: ops.group_norm(x.transpose(1, 3), 2), lambda: ops.group_norm(x[:0], 2),
                lambda: ops.group_norm(x.long(), 2), lambda: ops.group_norm(x, 2, out_dtype=torch.int8), lambda: ops.group_norm(x, 2, x[0, 0, 0, :4]),
                lambda: ops.group_norm(x, 2, torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda", dtype=torch.float16)),
                lambda: ops.group_norm(x, 2, out=x[:1]), lambda: ops.group_norm(x, 2, out=x, out_dtype=torch.float16),
                lambda: ops.group_norm_backward(x[:1], x, s, s, 2), lambda: ops.group_norm_backward(x, x, s[:1], s, 2), lambda: ops.group_norm_backward(x, x, s, s.double(), 2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(Exception):
        ops.group_norm(x, 2, eps=-1.0)
