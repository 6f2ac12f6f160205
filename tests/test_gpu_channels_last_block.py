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
