"""The kernels of the 4-bit product over long K and over several row blocks, and quantisation over every scale, against
their definition in 64 bits.  Where all scales are alike, the operands are multiples of 1/2 and every partial sum is a whole
number of quarters below 2^24 of them: equal, whatever the order.  Else each of the K + 16 additions (one more for the bias)
rounds by at most 2^-23 of the sum of magnitudes (truncation allowed)."""
import pytest
import torch

import mxfp4_reference as ref
from mxfp4_reach import FEW, LONG
from test_gpu_mxfp4 import DTYPES, awkward, put, same_codes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel, M, N, K", LONG)
def test_long_k(gpu, kernel, M, N, K):
    from amos_amd import ops
    g = torch.Generator().manual_seed(M + 5 * N + K)
    a, b = ref.random_codes(g, M, K), ref.random_codes(g, N, K)
    want = ref.values(*a, K) @ ref.values(*b, K).t()
    first = ops.mxfp4_gemm(put(a, K), put(b, K))
    assert torch.equal(first.cpu(), want.float())
    for _ in range(3):
        assert torch.equal(ops.mxfp4_gemm(put(a, K), put(b, K)), first)
    # every block's scale at its own place, in both operands
    a, b = (a[0], ref.random_codes(g, M, K, 115, 139)[1]), (b[0], ref.random_codes(g, N, K, 120, 134)[1])
    av, bv = ref.values(*a, K), ref.values(*b, K)
    got = ops.mxfp4_gemm(put(a, K), put(b, K)).cpu().double()
    assert ((got - av @ bv.t()).abs() <= (K + 16) * 2.0 ** -23 * (av.abs() @ bv.abs().t())).all()


@pytest.mark.parametrize("rt, M, N, K", FEW)
def test_few_rows(gpu, rt, M, N, K):
    from amos_amd import ops
    g = torch.Generator().manual_seed(M + N + K)
    a, b = ref.random_codes(g, M, K), ref.random_codes(g, N, K)
    want = ref.values(*a, K) @ ref.values(*b, K).t()
    assert torch.equal(ops.mxfp4_gemm(put(a, K), put(b, K)).cpu(), want.float())
    # scales of all sizes, bias and D, every type of the rows
    b = (b[0], ref.random_codes(g, N, K, 120, 134)[1])
    bv, q = ref.values(*b, K), put(b, K)
    bias, add = torch.randn(N, generator=g), torch.randn(M, N, generator=g)
    for dtype in DTYPES:
        x = awkward(M, K, dtype, M + K)
        codes = ref.quantize(x)
        av = ref.values(*codes, K)
        want = av @ bv.t() + bias.double() + add.double()
        bound = (K + 18) * 2.0 ** -23 * (av.abs() @ bv.abs().t() + bias.double().abs() + add.double().abs())
        for rows in (x.cuda(), put(codes, K)):
            got = ops.mxfp4_gemm(rows, q, bias=bias.cuda(), add=add.cuda())
            assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_scale(gpu, dtype):
    """a block for every power of two of the type, subnormal ones among them: its largest magnitude with a random
    fraction, ties of every pair of neighbouring codes, their neighbours on both sides, and smaller values"""
    from amos_amd import ops
    info = torch.finfo(dtype)
    low = int(torch.tensor(info.smallest_normal * info.eps, dtype=torch.float64).log2())
    high = int(torch.frexp(torch.tensor(info.max, dtype=torch.float64))[1]) - 1
    g = torch.Generator().manual_seed(1)
    e = torch.arange(low, high + 1)
    unit = torch.exp2(e.double() - 2)[:, None]      # what the scale is where it is not clamped
    x = torch.zeros(len(e), 96, dtype=torch.float64)
    x[:, :1] = unit * (4 + 3.999 * torch.rand(len(e), 1, generator=g).double())
    ties = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7], dtype=torch.float64)
    x[:, 1:9], x[:, 9:17] = unit * ties, -unit * ties
    x[:, 17:32] = unit * (8 * torch.rand(len(e), 15, generator=g).double() - 4)
    x[:, 32], x[:, 33:41], x[:, 41:49] = unit[:, 0] * 4, unit * ties * (1 + info.eps), unit * ties * (1 - info.eps)
    x[:, 49:64] = unit * torch.exp2(-20 * torch.rand(len(e), 15, generator=g).double())
    x[:, 64:] = unit * 7.9 * torch.randn(len(e), 32, generator=g).double().clamp(-1, 1)
    x = x.clamp(-info.max, info.max).to(dtype)
    want = ref.quantize(x)
    q = ops.mxfp4_quantize(x.cuda())
    same_codes(q, want)
    assert len(want[1][:, 0].unique()) >= (250 if dtype != torch.float16 else 38)
    same_codes(ops.mxfp4_quantize(x.t().contiguous().cuda(), axis=0), want)
    for back in DTYPES:
        assert torch.equal(ops.mxfp4_dequantize(q, back).cpu(), ref.values(*want, 96).float().to(back))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_more_than_31_bits_of_results(gpu, out):
    """a product of 2^31 and more results: its first, middle and last rows"""
    from amos_amd import ops
    M, N, K = 46400, 46500, 96
    g = torch.Generator().manual_seed(3)
    a, b = ref.random_codes(g, M, K), ref.random_codes(g, N, K)
    assert M * N > 1 << 31
    c = ops.mxfp4_gemm(put(a, K), put(b, K), out_dtype=out)
    av, bv = ref.values(*a, K), ref.values(*b, K)
    rows = torch.cat([torch.arange(3), torch.arange(23100, 23110), torch.arange(M - 300, M, 7), torch.tensor([M - 1])])
    assert torch.equal(c[rows.cuda()].cpu(), (av[rows] @ bv.t()).float().to(out))
