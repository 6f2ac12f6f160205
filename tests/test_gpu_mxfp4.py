"""Microscaled 4-bit quantisation and product against their definition in 64 bits.

Quantisation is compared code for code.  Products: where all scales are alike the operands are multiples
of 1/2 and every partial sum is a whole number of quarters below 2^24 of them, so any order of fp32
additions is exact and the result has to be equal (after its one rounding); for scales of all sizes each
of the K + 16 additions of a sum rounds by at most 2^-23 of the sum of magnitudes (truncation allowed)."""
import pytest
import torch

import mxfp4_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def put(codes_scales, cols):
    from amos_amd import ops
    return ops.Mxfp4(codes_scales[0].cuda(), codes_scales[1].cuda(), cols)


def same_codes(q, want):
    assert torch.equal(q.scales.cpu(), want[1])
    assert torch.equal(q.codes.cpu(), want[0])


def awkward(rows, cols, dtype, seed=0):
    """normal values of many sizes with zeros, ties, saturating and tiny ones among them"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, dtype=torch.float64)
    x = x * torch.exp2(torch.randint(-9, 5, (rows, (cols + 31) // 32), generator=g).double()).repeat_interleave(32, 1)[:, :cols]
    ties = torch.randint(-32, 33, (rows, cols), generator=g).double() / 4
    x = torch.where(torch.rand(rows, cols, generator=g) < 0.3, ties, x)
    x = torch.where(torch.rand(rows, cols, generator=g) < 0.1, 0.0, x)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 127), (4, 128), (9, 200), (300, 264), (257, 1000), (64, 4096)])
def test_quantize(gpu, dtype, rows, cols):
    from amos_amd import ops
    x = awkward(rows, cols, dtype, rows + cols)
    same_codes(ops.mxfp4_quantize(x.cuda()), ref.quantize(x))
    same_codes(ops.mxfp4_quantize(x.cuda(), axis=0), ref.quantize(x.t()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_extremes(gpu, dtype):
    """blocks at both ends of the type, subnormal ones, signed zeros, infinities and NaN: those make their
    own block NaN and no other"""
    from amos_amd import ops
    info = torch.finfo(dtype)
    x = torch.zeros(12, 96, dtype=torch.float64)
    x[0, :40] = info.max
    x[1, ::3] = -info.max
    x[2, :] = info.tiny
    x[3, 5] = info.smallest_normal * info.eps            # the smallest subnormal
    x[4, :] = torch.linspace(-1, 1, 96, dtype=torch.float64) * info.tiny * 3
    x[5, 1::2] = -0.0
    x[6, 40] = float("inf")
    x[7, 70] = float("nan")
    x[8, 0], x[8, 95] = float("-inf"), 1.0
    x[9, :32], x[9, 32:64] = 1.75, 1.7499
    x[10, :] = torch.arange(96) * 2.0 ** -20
    x = x.to(dtype)
    q = ops.mxfp4_quantize(x.cuda())
    same_codes(q, ref.quantize(x))
    same_codes(ops.mxfp4_quantize(x.t().contiguous().cuda(), axis=0), ref.quantize(x))
    back = ops.mxfp4_dequantize(q).cpu()
    assert back[6, 32:64].isnan().all() and back[7, 64:].isnan().all() and back[8, :32].isnan().all() and int(back.isnan().sum()) == 96
    # a matrix-core product takes the scale 255 as NaN: the row, and no other row
    ones = put(ref.quantize(torch.ones(3, 96)), 96)
    c = ops.mxfp4_gemm(q, ones).cpu()
    nan_rows = torch.tensor([6, 7, 8])
    assert c[nan_rows].isnan().all() and int(c.isnan().sum()) == 9


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 37), (130, 256), (65, 1003)])
def test_dequantize(gpu, dtype, rows, cols):
    from amos_amd import ops
    g = torch.Generator().manual_seed(rows)
    packed = ref.random_codes(g, rows, cols, 0, 255)
    got = ops.mxfp4_dequantize(put(packed, cols), dtype).cpu()
    want = ref.values(*packed, cols).float().to(dtype)   # (fp32 holds them all)
    assert got.dtype == dtype and torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_unaligned_storage_and_outputs(gpu, dtype):
    """tensors that start off the 16-byte grid; results written into the caller's tensors, whose
    neighbours stay as they were"""
    from amos_amd import ops
    rows, cols = 33, 264
    x = awkward(rows, cols, dtype)
    room = torch.zeros(rows * cols + 3, dtype=dtype, device="cuda")
    view = room[1:1 + rows * cols].view(rows, cols)
    view.copy_(x)
    want = ref.quantize(x)
    codes = torch.full((rows + 2, ref.pitch(cols)), 7, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows + 2, ref.pitch(cols) // 16), 9, dtype=torch.uint8, device="cuda")
    q = ops.Mxfp4(codes[1:-1], scales[1:-1], cols)
    assert ops.mxfp4_quantize(view, out=q) is q
    same_codes(q, want)
    assert (codes[0] == 7).all() and (codes[-1] == 7).all() and (scales[0] == 9).all() and (scales[-1] == 9).all()
    same_codes(ops.mxfp4_quantize(view, axis=0), ref.quantize(x.t()))
    back = torch.full((rows * cols + 3,), 5.0, dtype=dtype, device="cuda")
    ops.mxfp4_dequantize(q, dtype, out=back[1:1 + rows * cols].view(rows, cols))
    assert torch.equal(back[1:1 + rows * cols].view(rows, cols).cpu(), ref.values(*want, cols).float().to(dtype))
    assert back[0] == 5 and (back[1 + rows * cols:] == 5).all()
    # the product from and into such tensors
    c = torch.full((rows * rows + 3,), 5.0, dtype=dtype, device="cuda")
    out = c[1:1 + rows * rows].view(rows, rows)
    assert ops.mxfp4_gemm(view, q, out=out) is out
    assert torch.equal(out, ops.mxfp4_gemm(q, q, out_dtype=dtype))
    assert c[0] == 5 and (c[1 + rows * rows:] == 5).all()


# M, N, K: single tokens, every row count class, sizes that fill no tile, one tile exactly, K of one element,
# odd counts of K steps, more K than the waves take in one turn
PRODUCTS = [(1, 1, 1), (1, 17, 33), (1, 1000, 4096), (2, 130, 640), (5, 64, 129), (16, 16, 128), (17, 48, 384), (24, 257, 1000),
            (33, 31, 2050), (64, 64, 256), (65, 100, 511), (100, 300, 513), (127, 129, 128), (128, 128, 1024), (130, 260, 640),
            (255, 257, 1152), (256, 256, 512), (300, 520, 2304), (512, 384, 768), (513, 1023, 96), (1025, 70, 4352), (700, 1300, 32), (40, 4500, 900),
            (300, 9000, 200), (24, 8300, 700), (9, 12400, 1100), (31, 8290, 1536), (1500, 1700, 1152), (1530, 1666, 1024), (2310, 2250, 640), (2304, 2304, 512), (520, 1100, 2700), (60, 17000, 1200), (1000, 700, 4480), (3100, 3005, 1100), (3005, 3100, 512), (3000, 2900, 300), (4100, 4097, 384), (4096, 4098, 512)]


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("M, N, K", PRODUCTS)
def test_product_exact(gpu, out, M, N, K):
    """multiples of 1/2 on both sides: equal, whatever the order of the sums"""
    from amos_amd import ops
    g = torch.Generator().manual_seed(M * 7 + N * 3 + K)
    a, b = ref.random_codes(g, M, K), ref.random_codes(g, N, K)
    want = ref.values(*a, K) @ ref.values(*b, K).t()
    got = ops.mxfp4_gemm(put(a, K), put(b, K), out_dtype=out)
    assert torch.equal(got.cpu(), want.float().to(out))
    bias = torch.randint(-20, 20, (N,), generator=g).float() / 2
    add = torch.randint(-40, 40, (M, N), generator=g).float() / 4
    for bt, at in ((torch.float32, torch.bfloat16), (torch.float16, torch.float32)):
        got = ops.mxfp4_gemm(put(a, K), put(b, K), out_dtype=out, bias=bias.to(bt).cuda(), add=add.to(at).cuda())
        assert torch.equal(got.cpu(), (want + bias.double() + add.double()).float().to(out))
    c = add.to(out).cuda()   # the added operand is the output
    assert ops.mxfp4_gemm(put(a, K), put(b, K), out=c, add=c) is c
    assert torch.equal(c.cpu(), (want + add.to(out).double()).float().to(out))


@pytest.mark.parametrize("M, N, K", PRODUCTS)
def test_product_scales(gpu, M, N, K):
    """scales of many sizes, each block's at its own place"""
    from amos_amd import ops
    g = torch.Generator().manual_seed(M + N + K)
    a, b = ref.random_codes(g, M, K, 115, 139), ref.random_codes(g, N, K, 120, 134)
    av, bv = ref.values(*a, K), ref.values(*b, K)
    got = ops.mxfp4_gemm(put(a, K), put(b, K)).cpu().double()
    assert ((got - av @ bv.t()).abs() <= (K + 16) * 2.0 ** -23 * (av.abs() @ bv.abs().t())).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M, N, K", [(1, 17, 33), (1, 1000, 4096), (3, 40, 200), (4, 64, 1024), (7, 33, 2050), (16, 50, 999), (24, 257, 1000), (100, 300, 520), (300, 520, 2304),
                                     (2, 5000, 600), (8, 12200, 300), (16, 40, 1024), (3, 13000, 700), (1, 100, 5000)])
def test_dense_rows_are_quantised_as_mxfp4_quantize_does(gpu, dtype, M, N, K):
    from amos_amd import ops
    a = awkward(M, K, dtype, M).cuda()
    g = torch.Generator().manual_seed(N)
    b = put(ref.random_codes(g, N, K, 120, 134), K)
    q = ops.mxfp4_quantize(a)
    bias = torch.randn(N, generator=g).cuda()
    for out in DTYPES:
        one = ops.mxfp4_gemm(a, b, out_dtype=out, bias=bias).double()
        two = ops.mxfp4_gemm(q, b, out_dtype=out, bias=bias).double()
        # (the same blocks, by the definition; the sums may be taken in another order)
        av, bv = ref.values(q.codes, q.scales, K), ref.values(b.codes, b.scales, K)
        mag = (av.abs() @ bv.abs().t() + bias.cpu().double().abs())
        half = torch.finfo(out).eps / 2
        near = (one - two).abs().cpu() <= 2 * (K + 17) * 2.0 ** -23 * mag + 2 * half * one.abs().cpu() + torch.finfo(out).tiny
        assert (near | (one == two).cpu()).all()   # (equal infinities, where fp16 ends, among them)
    a[0, K // 2] = float("nan")   # its block: row 0 and nothing else
    c = ops.mxfp4_gemm(a, b)
    assert c[0].isnan().all() and not c[1:].isnan().any()


def test_largest_and_smallest_scales(gpu):
    """scale bytes at both ends: products that fp32 holds are right, too large ones are infinite"""
    from amos_amd import ops
    K = 128
    g = torch.Generator().manual_seed(3)
    for M in (1, 200):
        for ea, eb in ((0, 254), (254, 0), (10, 200), (127, 1), (250, 3)):
            a, b = ref.random_codes(g, M, K, ea, ea), ref.random_codes(g, 40, K, eb, eb)
            want = ref.values(*a, K) @ ref.values(*b, K).t()
            assert torch.equal(ops.mxfp4_gemm(put(a, K), put(b, K)).cpu(), want.float())
        one = torch.full((M, K), 1.0)
        a = ref.quantize(one)
        a[1][:, :4] = 254
        assert torch.isinf(ops.mxfp4_gemm(put(a, K), put(a, K))).all()


def test_other_stream_and_repetition(gpu):
    """launched on a stream of the caller's, and twice: the same bits"""
    from amos_amd import ops
    for M in (3, 40, 300):
        x = awkward(M, 1000, torch.bfloat16).cuda()
        w = ops.mxfp4_quantize(awkward(200, 1000, torch.float32, 5).cuda())
        want = ops.mxfp4_gemm(x, w)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = [ops.mxfp4_gemm(x, w, stream=s) for _ in range(3)]
        q = ops.mxfp4_quantize(x, axis=0, stream=s)
        back = ops.mxfp4_dequantize(q, torch.bfloat16, stream=s)
        s.synchronize()
        for c in got:
            assert torch.equal(c, want)
        same_codes(q, ref.quantize(x.cpu().t()))
        assert back.shape == (1000, M)


@pytest.mark.parametrize("M", [1, 24, 130])
def test_captured_calls(gpu, M):
    """quantisation, product and dequantisation in a graph, replayed on changing inputs between eager
    calls; two graphs have workspaces of their own"""
    from amos_amd import ops
    N, K = 300, 1030
    w = ops.mxfp4_quantize(awkward(N, K, torch.float32, 5).cuda())
    xs = [torch.zeros(M, K, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    graphs, outs = [], []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for x in xs:
            ops.mxfp4_gemm(x, w)
    torch.cuda.current_stream().wait_stream(s)
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            q = ops.mxfp4_quantize(x, axis=0)
            outs.append((ops.mxfp4_gemm(x, w), ops.mxfp4_dequantize(q, torch.float32)))
        graphs.append(g)
    for turn in range(3):
        for i, x in enumerate(xs):
            x.copy_(awkward(M, K, torch.bfloat16, 10 * turn + i))
        for g in graphs:
            g.replay()
        for x, (c, back) in zip(xs, outs):
            assert torch.equal(c, ops.mxfp4_gemm(x, w))
            assert torch.equal(back, ops.mxfp4_dequantize(ops.mxfp4_quantize(x, axis=0)))
        torch.cuda.synchronize()


def test_more_than_32_bits_of_elements(gpu):
    """offsets beyond 2^32: the last rows of a matrix of 2^32 and some elements"""
    from amos_amd import ops
    rows, cols = 65600, 65536
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    tail = awkward(40, cols, torch.bfloat16)
    x[-40:] = tail.cuda()
    q = ops.mxfp4_quantize(x)
    want = ref.quantize(tail)
    assert torch.equal(q.scales[-40:].cpu(), want[1]) and torch.equal(q.codes[-40:].cpu(), want[0])
    assert not q.codes[:-40].any()
    back = ops.mxfp4_dequantize(q, torch.bfloat16, out=x)
    assert torch.equal(back[-40:].cpu(), ref.values(*want, cols).float().bfloat16())
    del x, back
    c = ops.mxfp4_gemm(q, ops.Mxfp4(q.codes[-40:], q.scales[-40:], cols), out_dtype=torch.float32)
    v = ref.values(*want, cols)
    mag = v.abs() @ v.abs().t()
    assert ((c[-40:].cpu().double() - v @ v.t()).abs() <= (cols + 16) * 2.0 ** -23 * mag).all() and not c[:-40].any()
    big = ops.mxfp4_quantize(torch.zeros(64, 1 << 20, dtype=torch.bfloat16, device="cuda"), axis=0)
    assert big.shape == (1 << 20, 64) and not big.codes.any() and not big.scales.any()


@pytest.mark.parametrize("M, N", [(9, 20), (70, 1100)])
def test_very_long_sums(gpu, M, N):
    """K past what the tiles' 32-bit offsets reach: zeros but for its first and last elements"""
    from amos_amd import ops
    K, ends = (1 << 23) + 300, 520
    g = torch.Generator().manual_seed(M)
    parts = []
    for rows in (M, N):
        c = torch.randint(0, 16, (rows, 2 * ends), generator=g)
        packed = torch.zeros(rows, ref.pitch(K), dtype=torch.uint8)
        packed[:, :ends // 2] = (c[:, 0:ends:2] + 16 * c[:, 1:ends:2]).to(torch.uint8)
        packed[:, (K - ends) // 2:K // 2] = (c[:, ends::2] + 16 * c[:, ends + 1::2]).to(torch.uint8)
        parts.append((ops.Mxfp4(packed.cuda(), torch.full((rows, ref.pitch(K) // 16), 127, dtype=torch.uint8, device="cuda"), K), ref.GRID[c]))
    want = parts[0][1] @ parts[1][1].t()        # multiples of 1/4 below 2^17: exact
    assert torch.equal(ops.mxfp4_gemm(parts[0][0], parts[1][0]).cpu(), want.float())


def test_columns_in_several_launches(gpu):
    """axis 0 of a matrix wider than one launch takes"""
    from amos_amd import ops
    cols = (1 << 24) + 130
    at = [0, 1, 63, (1 << 24) - 1, 1 << 24, (1 << 24) + 1, cols - 1]
    x = torch.zeros(3, cols, dtype=torch.float16, device="cuda")
    part = awkward(3, len(at), torch.float16)
    x[:, at] = part.cuda()
    q = ops.mxfp4_quantize(x, axis=0)
    codes, scales = ref.quantize(part.t())
    assert torch.equal(q.codes[at].cpu(), codes) and torch.equal(q.scales[at].cpu(), scales)
    q.codes[at] = 0
    q.scales[at] = 0
    assert not q.codes.any() and not q.scales.any()


def test_refusals_on_device_tensors(gpu):
    from amos_amd import ops
    x = torch.zeros(4, 64, device="cuda")
    q = ops.mxfp4_quantize(x)
    for bad in (lambda: ops.mxfp4_quantize(x.long()), lambda: ops.mxfp4_quantize(x.t()), lambda: ops.mxfp4_quantize(x[None]),
                lambda: ops.mxfp4_quantize(x, axis=2), lambda: ops.mxfp4_quantize(x[:0]), lambda: ops.mxfp4_quantize(x, out=x),
                lambda: ops.mxfp4_quantize(x, axis=0, out=q), lambda: ops.Mxfp4(q.codes, q.scales, 200), lambda: ops.Mxfp4(q.codes.float(), q.scales, 64),
                lambda: ops.Mxfp4(q.codes[:, :32], q.scales, 64), lambda: ops.Mxfp4(q.codes, q.scales[:3], 64),
                lambda: ops.mxfp4_gemm(q, ops.mxfp4_quantize(torch.zeros(4, 32, device="cuda"))), lambda: ops.mxfp4_gemm(x[0], q),
                lambda: ops.mxfp4_gemm(q, q, out_dtype=torch.int8), lambda: ops.mxfp4_gemm(q, q, bias=x[0]), lambda: ops.mxfp4_gemm(q, q, add=x),
                lambda: ops.mxfp4_gemm(q, q, out=x), lambda: ops.mxfp4_gemm(x.long(), q), lambda: ops.mxfp4_dequantize(q, torch.int8),
                lambda: ops.mxfp4_dequantize(q, torch.float16, out=x)):
        with pytest.raises(ValueError):
            bad()
