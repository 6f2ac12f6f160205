"""The operators of the channels-last block -- normalise and activate, quantise, multiply -- as
cases to measure: microscaled 4-bit quantisation and product, group norm with an activation and
its gradient.

`own` False: their plain form in elementary torch operations; True: the calls of `amos_amd.ops`.
`exact` gives the same results from the definitions in 64 bits.
"""
import math

import torch

own = False

_DTYPE = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_BLOCK, _PAD = 32, 128   # elements behind one scale; what a row of codes is padded to


def listed():
    return [
        # a large activation matrix on its way into a 4-bit product, and back (a round trip is also
        # how the rounding is imitated at 16 bits)
        dict(name="quantize 8192x8192 bf16", op="quantize", rows=8192, cols=8192, dtype="bfloat16", axis=1),
        # a ragged gradient, quantised along its rows' index for a product that sums over rows
        dict(name="quantize 1003x777 fp32 axis 0", op="quantize", rows=1003, cols=777, dtype="float32", axis=0),
        # the benchmark's square product, both operands held in 4 bits
        dict(name="product 8192^3", op="product", m=8192, n=8192, k=8192, a="mxfp4", out="float32", bias=False, add=False),
        # one token through a projection: the activations arrive at 16 bits
        dict(name="product 1x4096x4096", op="product", m=1, n=4096, k=4096, a="bfloat16", out="bfloat16", bias=False, add=False),
        # a batch of tokens through a wide layer, weights streamed once
        dict(name="product 24x10240x8192", op="product", m=24, n=10240, k=8192, a="bfloat16", out="bfloat16", bias=True, add=False),
        # a ragged batch with bias and residual, sizes that fill no tile
        dict(name="product 333x1000x2050", op="product", m=333, n=1000, k=2050, a="float16", out="float32", bias=True, add=True),
        # a layer's training step: forward, input gradient, weight gradient, each product on
        # operands quantised along what it sums over
        dict(name="step 4096x2048x1024", op="step", m=4096, n=2048, k=1024),
        # a stage of a residual network on a batch of 32, channels last
        dict(name="norm 32x56x56x256 silu", op="norm", n=32, d=1, h=56, w=56, groups=32, per=8, dtype="bfloat16", out="bfloat16", act="silu", affine=True),
        # one small image's deep stage as a convolution leaves it (fp32), handed on at 16 bits
        dict(name="norm 1x7x7x512 fp32", op="norm", n=1, d=1, h=7, w=7, groups=32, per=16, dtype="float32", out="bfloat16", act="relu", affine=True),
        # odd extents and an odd group width
        dict(name="norm 3x13x17x120 fp16", op="norm", n=3, d=1, h=13, w=17, groups=24, per=5, dtype="float16", out="float16", act="silu", affine=True),
        # gradients of the first and of a volume with few channels
        dict(name="norm gradient 32x56x56x256", op="gradient", n=32, d=1, h=56, w=56, groups=32, per=8, dtype="bfloat16", out="bfloat16", act="silu", affine=True),
        dict(name="norm gradient 2x9x33x35x48", op="gradient", n=2, d=9, h=33, w=35, groups=16, per=3, dtype="float32", out="float32", act="silu", affine=True),
    ]


def _log(rng, low, high):
    """a whole number between low and high, spread over its logarithm"""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "step", "norm", "norm", "gradient"])
    if op == "quantize":
        return dict(op=op, rows=_log(rng, 1, 8192), cols=_log(rng, 1, 8192), dtype=rng.choice(sorted(_DTYPE)), axis=rng.choice([0, 1]))
    if op == "product":
        return dict(op=op, m=_log(rng, 1, 8192), n=_log(rng, 8, 8192), k=_log(rng, 16, 8192), a=rng.choice(["mxfp4"] + sorted(_DTYPE)),
                    out=rng.choice(sorted(_DTYPE)), bias=rng.random() < 0.5, add=rng.random() < 0.3)
    if op == "step":
        return dict(op=op, m=_log(rng, 16, 4096), n=_log(rng, 16, 2048), k=_log(rng, 16, 2048))
    groups, per = rng.choice([1, 2, 4, 8, 16, 24, 32]), _log(rng, 1, 40)
    deep = rng.random() < 0.25
    n, d, h, w = _log(rng, 1, 32), _log(rng, 2, 16) if deep else 1, _log(rng, 1, 64), _log(rng, 1, 64)
    most = 32 * 56 * 56 * 256
    n = max(1, min(n, most // (d * h * w * groups * per)))
    d = max(1, min(d, most // (n * h * w * groups * per)))
    if d * h * w * per < 16:   # (of a group of a few elements the gradient is all cancellation)
        per = 16
    dtype = rng.choice(sorted(_DTYPE))
    out = dtype if rng.random() < 0.6 else rng.choice(sorted(_DTYPE))
    # (no gradient of relu: which side of its corner an element is on goes by the last bit of a sum)
    act = rng.choice(["none", "silu"] if op == "gradient" else ["none", "relu", "silu"])
    return dict(op=op, n=n, d=d, h=h, w=w, groups=groups, per=per, dtype=dtype, out=out, act=act, affine=rng.random() < 0.8)


# ---- inputs -----------------------------------------------------------------------------------


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, cols):
    """normal values, some columns far larger than the others"""
    return _normal(g, rows, cols) * torch.exp(0.7 * _normal(g, 1, cols))


def _pack(values, exponent, cols):
    """values of _blocks -> (codes [rows, cols padded to 128, / 2], scales): the lower element of a
    pair in the low half of its byte, the padding as zeros"""
    a = values.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | ((values < 0).to(torch.uint8) << 3)
    rows, blocks = exponent.shape
    padded = -(-cols // _PAD) * _PAD
    codes = torch.zeros(rows, padded, dtype=torch.uint8, device=code.device)
    codes[:, :blocks * _BLOCK] = code.reshape(rows, -1)
    scales = torch.zeros(rows, padded // _BLOCK, dtype=torch.uint8, device=code.device)
    scales[:, :blocks] = (exponent + 127).to(torch.uint8)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    state = {"case": case}
    if op == "quantize":
        state["x"] = _activations(g, case["rows"], case["cols"]).to(_DTYPE[case["dtype"]])
    elif op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = _activations(g, m, k)
        state["a"] = _pack(*_blocks(a), k) if case["a"] == "mxfp4" else a.to(_DTYPE[case["a"]])
        state["b"] = _pack(*_blocks(_normal(g, n, k) / math.sqrt(k)), k)
        state["bias"] = _normal(g, n) if case["bias"] else None
        state["add"] = _normal(g, m, n).to(torch.bfloat16) if case["add"] else None
    elif op == "step":
        m, n, k = case["m"], case["n"], case["k"]
        state["x"] = _activations(g, m, k).to(torch.bfloat16)
        state["w"] = (_normal(g, n, k) / math.sqrt(k)).to(torch.bfloat16)
        state["dy"] = (_normal(g, m, n) * 1e-3).to(torch.bfloat16)
    else:
        c = case["groups"] * case["per"]
        shape = (case["n"], case["h"], case["w"], c) if case["d"] == 1 else (case["n"], case["d"], case["h"], case["w"], c)
        state["layout"] = "nhwc" if case["d"] == 1 else "ndhwc"
        x = _normal(g, *shape) * torch.exp(0.3 * _normal(g, c)) + 0.5 * _normal(g, c)
        state["x"] = x.to(_DTYPE[case["dtype"]])
        state["weight"] = 1 + 0.2 * _normal(g, c) if case["affine"] else None
        state["bias"] = 0.3 * _normal(g, c) if case["affine"] else None
        if op == "gradient":
            state["dy"] = _normal(g, *shape).to(_DTYPE[case["out"]])
            state["mean"], state["rstd"] = _statistics(state["x"], case["groups"])
    return state


# ---- the plain forms --------------------------------------------------------------------------


def _blocks(x):
    """[rows, cols] -> the 4-bit values of its blocks of 32 (rows, blocks, 32) and the blocks'
    exponents: the power of two that brings the largest magnitude into [4, 8), each element rounded
    to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (ties to the even code), at most 6"""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -cols % _BLOCK)).reshape(rows, -1, _BLOCK)
    exponent = torch.frexp(x.abs().amax(-1))[1] - 3
    exponent = torch.where((x == 0).all(-1), -127, exponent).clamp(-127, 127)
    x = x * torch.exp2(-exponent.double())[..., None]
    a = x.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.round(a / step).mul(step).clamp(max=6).mul(torch.sign(x)), exponent


def _rounded(x, cols):
    """x [rows, cols] as its 4-bit blocks stand for it"""
    values, exponent = _blocks(x)
    return (values * torch.exp2(exponent.double())[..., None]).reshape(x.shape[0], -1)[:, :cols].float()


def _unpack(packed, cols):
    codes, scales = packed
    code = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1, _BLOCK)
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    scale = torch.exp2(scales.double() - 127).float()
    return (table[code.int()] * scale[..., None]).reshape(codes.shape[0], -1)[:, :cols]


def _by_group(x, groups):
    """channels-last x -> [images, pixels, groups, channels of a group]"""
    return x.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)


def _statistics(x, groups):
    v = _by_group(x, groups).double()
    mean = v.mean((1, 3))
    var = (v - mean[:, None, :, None]).square().mean((1, 3))
    return mean.float(), torch.rsqrt(var + 1e-5).float()


def _affine(state, groups):
    c = state["x"].shape[-1]
    weight, bias = state["weight"], state["bias"]
    weight = torch.ones(c, device="cuda") if weight is None else weight
    bias = torch.zeros(c, device="cuda") if bias is None else bias
    return weight.reshape(groups, -1), bias.reshape(groups, -1)


def _plain_norm(state):
    case, x = state["case"], state["x"]
    groups = case["groups"]
    mean, rstd = _statistics(x, groups)
    weight, bias = _affine(state, groups)
    y = (_by_group(x, groups).float() - mean[:, None, :, None]) * rstd[:, None, :, None] * weight + bias
    if case["act"] == "relu":
        y = y.clamp(min=0)
    elif case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y.reshape(x.shape).to(_DTYPE[case["out"]]), mean, rstd


def _plain_gradient(state):
    case, x = state["case"], state["x"]
    groups = case["groups"]
    mean, rstd = state["mean"][:, None, :, None], state["rstd"][:, None, :, None]
    weight, bias = _affine(state, groups)
    normal = (_by_group(x, groups).float() - mean) * rstd
    dz = _by_group(state["dy"], groups).float()
    if case["act"] == "relu":
        dz = dz * (normal * weight + bias > 0)
    elif case["act"] == "silu":
        z = normal * weight + bias
        s = 1 / (1 + torch.exp(-z))
        dz = dz * s * (1 + z * (1 - s))
    dweight, dbias = (dz * normal).double().sum((0, 1)).float(), dz.double().sum((0, 1)).float()
    d = dz * weight
    of_d = d.double().mean((1, 3), keepdim=True).float()
    of_dn = (d * normal).double().mean((1, 3), keepdim=True).float()
    dx = (d - of_d - normal * of_dn) * rstd
    out = [dx.reshape(x.shape).to(x.dtype)]
    return out + [dweight.reshape(-1), dbias.reshape(-1)] if case["affine"] else out


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "quantize":
        x = state["x"]
        return _rounded(x, x.shape[1]).to(x.dtype) if case["axis"] == 1 else _rounded(x.t(), x.shape[0]).to(x.dtype)
    if op == "product":
        k = case["k"]
        a = _unpack(state["a"], k) if case["a"] == "mxfp4" else _rounded(state["a"], k)
        c = a @ _unpack(state["b"], k).t()
        if state["bias"] is not None:
            c = c + state["bias"]
        if state["add"] is not None:
            c = c + state["add"].float()
        return c.to(_DTYPE[case["out"]])
    if op == "step":
        x, w, dy = state["x"], state["w"], state["dy"]
        m, n, k = case["m"], case["n"], case["k"]
        y = _rounded(x, k) @ _rounded(w, k).t()
        dx = _rounded(dy, n) @ _rounded(w.t(), n).t()
        dw = _rounded(dy.t(), m) @ _rounded(x.t(), m).t()
        return y.to(torch.bfloat16), dx.to(torch.bfloat16), dw
    return _plain_norm(state) if op == "norm" else _plain_gradient(state)


# ---- the framework's calls ---------------------------------------------------------------------


def _framework(state):
    from amos_amd import ops
    case = state["case"]
    op = case["op"]
    if op == "quantize":
        return ops.mxfp4_dequantize(ops.mxfp4_quantize(state["x"], axis=case["axis"]), state["x"].dtype)
    if op == "product":
        a = ops.Mxfp4(*state["a"], case["k"]) if case["a"] == "mxfp4" else state["a"]
        return ops.mxfp4_gemm(a, ops.Mxfp4(*state["b"], case["k"]), out_dtype=_DTYPE[case["out"]], bias=state["bias"], add=state["add"])
    if op == "step":
        x, w, dy = state["x"], state["w"], state["dy"]
        y = ops.mxfp4_gemm(x, ops.mxfp4_quantize(w), out_dtype=torch.bfloat16)
        dx = ops.mxfp4_gemm(dy, ops.mxfp4_quantize(w, axis=0), out_dtype=torch.bfloat16)
        return y, dx, ops.mxfp4_gemm(ops.mxfp4_quantize(dy, axis=0), ops.mxfp4_quantize(x, axis=0))
    act = None if case["act"] == "none" else case["act"]
    if op == "norm":
        return ops.group_norm(state["x"], case["groups"], state["weight"], state["bias"], eps=1e-5, activation=act, layout=state["layout"],
                              out_dtype=_DTYPE[case["out"]], stats=True)
    dx, dweight, dbias = ops.group_norm_backward(state["dy"], state["x"], state["mean"], state["rstd"], case["groups"], state["weight"], state["bias"],
                                                 activation=act, layout=state["layout"])
    return [dx, dweight, dbias] if case["affine"] else [dx]


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------


def _held(rows, cols):
    """bytes of a matrix in 4 bits with its scales"""
    return rows * (cols / 2 + cols / _BLOCK)


def work(case):
    size = lambda t: 4 if t == "float32" else 2
    op = case["op"]
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": 2 * rows * cols * size(case["dtype"]) + 2 * _held(rows, cols), "flops": 4.0 * rows * cols}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = _held(m, k) if case["a"] == "mxfp4" else m * k * size(case["a"])
        return {"bytes": a + _held(n, k) + m * n * size(case["out"]) + (4 * n if case["bias"] else 0) + (2 * m * n if case["add"] else 0), "flops": 2.0 * m * n * k}
    if op == "step":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * (m * k + n * k + m * n) + 2 * (m * n + m * k) + 4 * n * k, "flops": 6.0 * m * n * k}
    elements = case["n"] * case["d"] * case["h"] * case["w"] * case["groups"] * case["per"]
    small = 4 * case["groups"] * (2 * case["n"] + (2 * case["per"] if case["affine"] else 0))
    if op == "norm":
        return {"bytes": elements * (size(case["dtype"]) + size(case["out"])) + small, "flops": 10.0 * elements}
    return {"bytes": elements * (2 * size(case["dtype"]) + size(case["out"])) + 2 * small, "flops": 20.0 * elements}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def _nearest(x):
    """x [rows, cols] -> the values its 4-bit blocks along a row stand for: codes by comparison with
    the midpoints of neighbouring values, a midpoint itself going to the even code"""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for first in range(0, x.shape[1], _BLOCK):
        v = x[:, first:first + _BLOCK].double()
        top = v.abs().amax(1, keepdim=True)
        scale = torch.exp2((torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2).clamp(-127, 127))
        a, code = v.abs() / scale, torch.zeros_like(v, dtype=torch.int64)
        for i in range(7):
            middle = (grid[i] + grid[i + 1]) / 2
            code += (a > middle) if i % 2 == 0 else (a >= middle)
        out[:, first:first + _BLOCK] = torch.copysign(grid[code] * scale, v)
    return out


def _decoded(packed, cols):
    """the values of codes and scales, from the fields of the 4 bits"""
    codes, scales = packed
    bits = torch.zeros(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes >> (4 * half)).long()
        e, f = (c >> 1) & 3, (c & 1).double()
        magnitude = torch.where(e == 0, f / 2, (1 + f / 2) * torch.exp2((e - 1).double()))
        bits[:, half::2] = torch.where((c & 8) > 0, -magnitude, magnitude)
    bits *= torch.exp2(scales.double() - 127).repeat_interleave(_BLOCK, 1)
    return bits[:, :cols]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _nearest(state["x"] if case["axis"] == 1 else state["x"].t().contiguous())
    if op == "product":
        a = _decoded(state["a"], case["k"]) if case["a"] == "mxfp4" else _nearest(state["a"])
        c = torch.mm(a, _decoded(state["b"], case["k"]).t().contiguous())
        for more in (state["bias"], state["add"]):
            if more is not None:
                c += more.double()
        return c
    if op == "step":
        x, w, dy = state["x"], state["w"], state["dy"]
        turned = lambda t: t.t().contiguous()
        y = torch.mm(_nearest(x), turned(_nearest(w)))
        dx = torch.mm(_nearest(dy), turned(_nearest(turned(w))))
        return y, dx, torch.mm(_nearest(turned(dy)), turned(_nearest(turned(x))))
    x = state["x"].double()
    c, groups = x.shape[-1], case["groups"]
    leaves = [x, torch.ones(c, dtype=torch.float64, device="cuda"), torch.zeros(c, dtype=torch.float64, device="cuda")]
    if case["affine"]:
        leaves[1:] = [state["weight"].double(), state["bias"].double()]
    if op == "gradient":
        for leaf in leaves:
            leaf.requires_grad_(True)
    v = leaves[0].movedim(-1, 1).reshape(x.shape[0], groups, -1)
    mean, var = v.mean(-1), v.var(-1, unbiased=False)
    rstd = (var + 1e-5) ** -0.5
    y = ((v - mean[..., None]) * rstd[..., None]).reshape(x.movedim(-1, 1).shape).movedim(1, -1) * leaves[1] + leaves[2]
    if case["act"] == "relu":
        y = torch.where(y > 0, y, 0.0)
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    if op == "norm":
        return y, mean, rstd
    got = torch.autograd.grad(y, leaves, state["dy"].double())
    return list(got) if case["affine"] else [got[0]]
