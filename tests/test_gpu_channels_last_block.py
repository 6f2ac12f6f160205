"""A channels-last block as a network runs it: a convolution's fp32 output through group norm + silu to 16
bits, quantised rows through a 4-bit pointwise product with bias and residual, and a convolution on its output;
forward and the products of its backward pass.  Every stage is checked in 64 bits on the inputs it was given."""
import pytest
import torch

import mxfp4_reference as ref
from test_gpu_group_norm import check_forward, check_gradient, coefficients, make

pytestmark = pytest.mark.gpu


def close_product(got, a, b, more=0.0):
    """a, b in 64 bits; fp32 sums of K products, one rounding to the result's type"""
    want, mag = a @ b.t() + more, a.abs() @ b.abs().t() + (more.abs() if torch.is_tensor(more) else 0)
    half = torch.finfo(got.dtype).eps / 2
    assert ((got.cpu().double() - want).abs() <= (a.shape[1] + 18) * 2.0 ** -23 * mag * (1 + half) + half * want.abs()).all()


@pytest.mark.parametrize("n, h, w, c, k, groups", [(2, 9, 7, 64, 96, 8), (1, 1, 1, 128, 64, 4), (3, 12, 13, 160, 72, 16)])
def test_block(gpu, n, h, w, c, k, groups):
    from amos_amd import ops
    x32 = make("nhwc", (n, h, w, c), 1)                                     # what a convolution leaves
    gamma, beta = coefficients(c, 2)
    y, mean, rstd = check_forward(x32, groups, gamma, beta, "silu", "nhwc", torch.bfloat16)
    g = torch.Generator().manual_seed(3)
    weight = (torch.randn(k, c, generator=g) / c ** 0.5).bfloat16().cuda()
    bias, rest = torch.randn(k, generator=g).cuda(), torch.randn(n * h * w, k, generator=g).bfloat16().cuda()
    q = ops.mxfp4_quantize(weight)
    rows = y.reshape(-1, c)
    z = ops.mxfp4_gemm(rows, q, out_dtype=torch.float16, bias=bias, add=rest)
    value = lambda t: ref.values(*ref.quantize(t.float()), t.shape[1])
    close_product(z, value(rows), value(weight), bias.cpu().double() + rest.cpu().double())
    # the convolution on it, channels last
    cw = (torch.randn(3, 3, k, 32, generator=g) / (3 * k ** 0.5)).half().cuda()
    out = ops.conv2d(z.reshape(n, h, w, k), cw, 1, 1, layout="nhwc")
    zz, ww = z.reshape(n, h, w, k).cpu().double().permute(0, 3, 1, 2), cw.cpu().double().permute(3, 2, 0, 1)
    want = torch.nn.functional.conv2d(zz, ww, padding=1).permute(0, 2, 3, 1)
    mag = torch.nn.functional.conv2d(zz.abs(), ww.abs(), padding=1).permute(0, 2, 3, 1)
    assert ((out.cpu().double() - want).abs() <= (9 * k + 16) * 2.0 ** -23 * mag).all()
    # backward: gradients of the product on operands quantised along what each sums over, then of the norm
    dz = (torch.randn(n * h * w, k, generator=g) * 1e-2).bfloat16().cuda()
    dy = ops.mxfp4_gemm(dz, ops.mxfp4_quantize(weight, axis=0), out_dtype=torch.bfloat16)
    close_product(dy, value(dz), value(weight.t()))
    dw = ops.mxfp4_gemm(ops.mxfp4_quantize(dz, axis=0), ops.mxfp4_quantize(rows.contiguous(), axis=0))
    close_product(dw, value(dz.t()), value(rows.t()))
    check_gradient(x32, groups, gamma, beta, "silu", "nhwc", torch.bfloat16)
    dx, dgamma, dbeta = ops.group_norm_backward(dy.reshape(n, h, w, c), x32.cuda(), mean, rstd, groups, gamma.cuda(), beta.cuda(), activation="silu")
    assert dx.shape == x32.shape and dx.isfinite().all() and dgamma.isfinite().all() and dbeta.isfinite().all()


def every_call():
    """(name, call with a stream or None, tensors of its result) of each operator, with and without its options"""
    from amos_amd import ops
    g = torch.Generator().manual_seed(3)
    r = lambda *shape: torch.randn(*shape, generator=g).cuda()
    x, add, bias = r(24, 200).bfloat16(), r(24, 72), r(72).half()
    w = ops.mxfp4_quantize(r(72, 200))
    q = ops.mxfp4_quantize(x)
    image, dy, weight, shift = r(2, 3, 5, 6, 24), r(2, 3, 5, 6, 24).bfloat16(), r(24), r(24)
    _, mean, rstd = ops.group_norm(image, 6, weight, shift, stats=True, layout="ndhwc")
    mx = lambda t: (t.codes, t.scales)
    yield "quantize", lambda s: ops.mxfp4_quantize(x, axis=0, stream=s), mx
    yield "quantize, other names of the axes", lambda s: ops.mxfp4_quantize(x, axis=-1, stream=s), mx
    yield "quantize into", lambda s: ops.mxfp4_quantize(x, out=q, stream=s), mx
    yield "dequantize", lambda s: ops.mxfp4_dequantize(q, torch.float16, stream=s), lambda t: (t,)
    yield "dequantize into", lambda s: ops.mxfp4_dequantize(q, torch.bfloat16, out=torch.empty_like(x), stream=s), lambda t: (t,)
    yield "product", lambda s: ops.mxfp4_gemm(q, w, stream=s), lambda t: (t,)
    yield "product, dense rows", lambda s: ops.mxfp4_gemm(x, w, out_dtype=torch.bfloat16, add=add, bias=bias, stream=s), lambda t: (t,)
    yield "product into", lambda s: ops.mxfp4_gemm(x, w, out=torch.empty_like(add), bias=bias, stream=s), lambda t: (t,)
    yield "norm", lambda s: ops.group_norm(image, 6, layout="ndhwc", activation="silu", stream=s), lambda t: (t,)
    yield "norm, statistics", lambda s: ops.group_norm(image[0], 3, weight, shift, 1e-3, "relu", "hwnc", torch.float16, stats=True, stream=s), lambda t: t
    yield "norm into", lambda s: ops.group_norm(image, 6, weight, out=torch.empty_like(dy), layout="ndhwc", stream=s), lambda t: (t,)
    yield "gradient", lambda s: ops.group_norm_backward(dy, image, mean, rstd, 6, weight, shift, "silu", "ndhwc", stream=s), lambda t: t
    yield "gradient, no coefficients", lambda s: ops.group_norm_backward(dy, image, mean, rstd, 6, layout="ndhwc", stream=s)[:1], lambda t: t


def test_native_and_long_way_agree(gpu):
    """a named stream goes the long way through the interpreter, the current one the native way"""
    for name, call, tensors in every_call():
        one, two = tensors(call(None)), tensors(call(torch.cuda.current_stream()))
        assert len(one) == len(two)
        for a, b in zip(one, two):
            assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b), name


def test_calls_keep_nothing(gpu):
    """no memory and no references stay behind, refused calls included"""
    import sys
    from amos_amd import ops
    bad = torch.zeros(4, 6, device="cuda")
    for name, call, tensors in every_call():
        call(None)
        before = torch.cuda.memory_allocated(), sys.getrefcount(None), sys.getrefcount(torch.float16), sys.getrefcount(ops.Mxfp4)
        for _ in range(300):
            call(None)
        after = torch.cuda.memory_allocated(), sys.getrefcount(None), sys.getrefcount(torch.float16), sys.getrefcount(ops.Mxfp4)
        assert before[0] == after[0] and all(abs(b - a) < 50 for a, b in zip(before[1:], after[1:])), name
    before = torch.cuda.memory_allocated(), sys.getrefcount(bad)
    for _ in range(100):
        with pytest.raises(ValueError):
            ops.group_norm(bad, 2)
        with pytest.raises(ValueError):
            ops.mxfp4_quantize(bad, axis=0, out=bad)
    assert torch.cuda.memory_allocated() == before[0] and abs(sys.getrefcount(bad) - before[1]) < 10


def test_calls_from_threads(gpu):
    """several threads at once, each on a stream of its own"""
    import threading
    want = [[t.clone() for t in tensors(call(None))] for _, call, tensors in every_call()]
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                for ours, (name, call, tensors) in zip(want, every_call()):
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(ours, tensors(call(None)))):
                        wrong.append(name)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
