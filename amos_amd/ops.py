"""Tensor-level entry points over the C ABI.

PyTorch-ROCm only supplies device memory and the current stream here; every
computation goes through libamos_mi355x.so.  There is no CPU or eager fallback:
tensors that are not on a HIP device are rejected.
"""
import ctypes
import os

import torch

from . import _lib
from ._lib import (AMOS_OP_BGEMM, AMOS_OP_CONV2D, AMOS_OP_CONV3D, AMOS_OP_GEMM, BGemmDesc, ConvDesc,
                   GemmDesc, KernelConfig, check)

_IN_CODE = {torch.float16: _lib.AMOS_F16, torch.bfloat16: _lib.AMOS_BF16, torch.int8: _lib.AMOS_I8}
_OUT_OF = {torch.float16: torch.float32, torch.bfloat16: torch.float32, torch.int8: torch.int32}
_OUT_CODE = {torch.float32: _lib.AMOS_F32, torch.int32: _lib.AMOS_I32}


def _need_device(*tensors):
    for t in tensors:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError("amos_amd runs on the GPU only: got a tensor on %s"
                               % (getattr(t, "device", type(t)),))
        if not t.is_contiguous():
            raise ValueError("operands must be contiguous")


def _stream_ptr(stream):
    if stream is None:
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


_CODE_DTYPE = {_lib.AMOS_F16: torch.float16, _lib.AMOS_BF16: torch.bfloat16, _lib.AMOS_I8: torch.int8,
               _lib.AMOS_F32: torch.float32, _lib.AMOS_I32: torch.int32}


def _gemm_spans(g, batch=1, sa=0, sb=0, sc=0):
    """elements the three operands of a (batched) GEMM descriptor reach"""
    a = (g.K - 1) * g.lda + g.M if g.trans_a else (g.M - 1) * g.lda + g.K
    b = (g.N - 1) * g.ldb + g.K if g.trans_b else (g.K - 1) * g.ldb + g.N
    c = (g.M - 1) * g.ldc + g.N
    return (batch - 1) * sa + a, (batch - 1) * sb + b, (batch - 1) * sc + c


def operand_spans(op, desc):
    """(elements of in0, in1, out the kernels may touch, input dtype, output dtype) of a descriptor"""
    if op == AMOS_OP_GEMM:
        g, spans = desc, _gemm_spans(desc)
    elif op == AMOS_OP_BGEMM:
        g, spans = desc.g, _gemm_spans(desc.g, desc.batch, desc.stride_a, desc.stride_b, desc.stride_c)
    else:
        g = desc
        groups = max(1, desc.groups)
        xs = (desc.N, desc.C, desc.D, desc.H, desc.W)
        ws = (desc.K, desc.C // groups, desc.T, desc.R, desc.S)
        o = conv_out_shape(xs, ws, (desc.stride_d, desc.stride_h, desc.stride_w),
                           (desc.pad_d, desc.pad_h, desc.pad_w), (desc.dil_d, desc.dil_h, desc.dil_w))
        prod = lambda t: int(torch.Size(t).numel())
        spans = (prod(xs), prod(ws), prod(o))
    return spans, _CODE_DTYPE.get(g.in_dtype), _CODE_DTYPE.get(g.out_dtype)


def check_operands(op, desc, in0, in1, out):
    """Refuse, before any launch, arrays that do not hold what the descriptor says: the kernels
    take raw pointers, so a short or wrongly typed array would be read or written out of bounds.
    (The reference's argument binder asserts shape and dtype at call time the same way.)"""
    (n0, n1, nout), in_dt, out_dt = operand_spans(op, desc)
    for what, t, need, dt in (("first input", in0, n0, in_dt), ("second input", in1, n1, in_dt),
                              ("output", out, nout, out_dt)):
        if t.dtype != dt:
            raise ValueError("%s is %s, the descriptor says %s" % (what, t.dtype, dt))
        if t.numel() < need:
            raise ValueError("%s holds %d elements, the descriptor reaches %d" % (what, t.numel(), need))
        if t.device != in0.device:
            raise ValueError("%s is on %s, the first input on %s" % (what, t.device, in0.device))


def _check_out(out, shape, dtype, like):
    """a caller-supplied output: exactly the result's shape and type, on the operands' device"""
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != like.device:
        raise ValueError("out must be a %s tensor of shape %s on %s: got %s %s on %s"
                         % (dtype, tuple(shape), like.device, out.dtype, tuple(out.shape), out.device))


def make_config(config):
    """None | KernelConfig | dict(tile_i=, tile_j=, split_k=) -> KernelConfig or None"""
    if config is None or isinstance(config, KernelConfig):
        return config
    c = KernelConfig()
    c.tile_i = int(config.get("tile_i", 0))
    c.tile_j = int(config.get("tile_j", 0))
    c.split_k = int(config.get("split_k", 0))
    c.pipeline = int(config.get("pipeline", 0))
    c.reserved[0] = int(config.get("flags", 0))
    return c


def _cfg_ref(cfg):
    return ctypes.byref(cfg) if cfg is not None else None


def make_epilogue(add, out_shape, out_dtype):
    """None | tensor of the output's shape -> Epilogue (out = acc + add) or None.  `add` is fp32,
    fp16 or bf16 for fp32 outputs, int32 for int32 outputs."""
    if add is None:
        return None
    _need_device(add)
    if tuple(add.shape) != tuple(out_shape):
        raise ValueError("the added operand has shape %s, the output %s" % (tuple(add.shape), tuple(out_shape)))
    codes = {torch.float32: _lib.AMOS_F32, torch.float16: _lib.AMOS_F16, torch.bfloat16: _lib.AMOS_BF16,
             torch.int32: _lib.AMOS_I32}
    ok = (torch.int32,) if out_dtype == torch.int32 else (torch.float32, torch.float16, torch.bfloat16)
    if add.dtype not in ok:
        raise ValueError("cannot add a %s operand to a %s output" % (add.dtype, out_dtype))
    e = _lib.Epilogue()
    e.kind, e.dtype, e.operand, e.ld, e.stride = _lib.AMOS_EPI_ADD, codes[add.dtype], add.data_ptr(), 0, 0
    return e


def _epi_ref(e):
    return ctypes.byref(e) if e is not None else None


def gemm_desc(M, N, K, in_dtype, trans_a=False, trans_b=False, lda=None, ldb=None, ldc=None):
    d = GemmDesc()
    d.M, d.N, d.K = M, N, K
    d.in_dtype = _IN_CODE[in_dtype]
    d.out_dtype = _OUT_CODE[_OUT_OF[in_dtype]]
    d.trans_a, d.trans_b = int(trans_a), int(trans_b)
    d.lda = lda if lda is not None else (M if trans_a else K)
    d.ldb = ldb if ldb is not None else (K if trans_b else N)
    d.ldc = ldc if ldc is not None else N
    return d


def conv_desc(x_shape, w_shape, in_dtype, stride, pad, dil, groups=1, layout="nchw"):
    """x_shape NCDHW, w_shape K,(C/groups),T,R,S (the logical extents, whatever the layout in
    memory); stride / pad / dil are 3-tuples"""
    d = ConvDesc()
    d.layout = _lib.LAYOUT_CODE[layout] if isinstance(layout, str) else int(layout)
    d.N, d.C, d.D, d.H, d.W = x_shape
    d.K, cg, d.T, d.R, d.S = w_shape
    if cg * groups != d.C:
        raise ValueError("weights have %d channels per group, activations %d channels in %d groups"
                         % (cg, d.C, groups))
    d.groups = groups
    d.stride_d, d.stride_h, d.stride_w = stride
    d.pad_d, d.pad_h, d.pad_w = pad
    d.dil_d, d.dil_h, d.dil_w = dil
    d.in_dtype = _IN_CODE[in_dtype]
    d.out_dtype = _OUT_CODE[_OUT_OF[in_dtype]]
    return d


def _tup(v, n, unit=None):
    if isinstance(v, (tuple, list)):
        assert len(v) == n
        return tuple(int(t) for t in v)
    return (int(v),) * n


def conv_out_shape(x_shape, w_shape, stride, pad, dil):
    out = []
    for ext, k, s, p, d in zip(x_shape[2:], w_shape[2:], stride, pad, dil):
        out.append((ext + 2 * p - ((k - 1) * d + 1)) // s + 1)
    return (x_shape[0], w_shape[0]) + tuple(out)


def gemm(a, b, trans_a=False, trans_b=False, out=None, config=None, stream=None, add=None):
    """C[M,N] = A(m,k) B(k,n) (+ add[M,N]); a is [M,K] ([K,M] if trans_a), b is [K,N] ([N,K] if trans_b)."""
    _need_device(a, b)
    M, K = (a.shape[1], a.shape[0]) if trans_a else a.shape
    N = b.shape[0] if trans_b else b.shape[1]
    if (b.shape[1] if trans_b else b.shape[0]) != K or a.dtype != b.dtype:
        raise ValueError("operand shapes / dtypes do not agree")
    if out is None:
        out = torch.empty((M, N), dtype=_OUT_OF[a.dtype], device=a.device)
    _need_device(out)
    _check_out(out, (M, N), _OUT_OF[a.dtype], a)
    d = gemm_desc(M, N, K, a.dtype, trans_a, trans_b)
    cfg = make_config(config)
    epi = make_epilogue(add, (M, N), out.dtype)
    ws, ws_ptr, ws_bytes = _workspace(AMOS_OP_GEMM, d, cfg, a.device, stream)
    check(_lib.load().amos_run_fused(AMOS_OP_GEMM, ctypes.byref(d), _cfg_ref(cfg), _epi_ref(epi), a.data_ptr(),
                                     b.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes, _stream_ptr(stream)))
    return out


def bgemm_desc(batch, M, N, K, in_dtype, trans_a=False, trans_b=False):
    d = BGemmDesc()
    d.batch = batch
    d.g = gemm_desc(M, N, K, in_dtype, trans_a, trans_b)
    d.stride_a, d.stride_b, d.stride_c = M * K, K * N, M * N
    return d


def bgemm(a, b, trans_a=False, trans_b=False, out=None, config=None, stream=None, add=None):
    """batched GEMM; a is [B,M,K] ([B,K,M] if trans_a), b is [B,K,N] ([B,N,K] if trans_b)."""
    _need_device(a, b)
    B = a.shape[0]
    M, K = (a.shape[2], a.shape[1]) if trans_a else a.shape[1:]
    N = b.shape[1] if trans_b else b.shape[2]
    if b.shape[0] != B or (b.shape[2] if trans_b else b.shape[1]) != K or a.dtype != b.dtype:
        raise ValueError("operand shapes / dtypes do not agree")
    if out is None:
        out = torch.empty((B, M, N), dtype=_OUT_OF[a.dtype], device=a.device)
    _need_device(out)
    _check_out(out, (B, M, N), _OUT_OF[a.dtype], a)
    d = bgemm_desc(B, M, N, K, a.dtype, trans_a, trans_b)
    cfg = make_config(config)
    epi = make_epilogue(add, (B, M, N), out.dtype)
    ws, ws_ptr, ws_bytes = _workspace(AMOS_OP_BGEMM, d, cfg, a.device, stream)
    check(_lib.load().amos_run_fused(AMOS_OP_BGEMM, ctypes.byref(d), _cfg_ref(cfg), _epi_ref(epi), a.data_ptr(),
                                     b.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes, _stream_ptr(stream)))
    return out


def workspace_bytes(op, desc, config=None):
    cfg = make_config(config)
    return int(_lib.load().amos_workspace_bytes(op, ctypes.byref(desc), _cfg_ref(cfg)))


def _workspace(op, desc, cfg, device, stream=None):
    """device scratch of amos_workspace_bytes() (conv: repacked weights); (tensor, ptr, bytes).
    The tensor is dropped as soon as the asynchronous launch returns, so it is allocated on the
    launch stream: the caching allocator then hands the block to later work of that stream only,
    which runs behind the kernel that still reads it."""
    need = _lib.load().amos_workspace_bytes(op, ctypes.byref(desc), _cfg_ref(cfg))
    if need == 0:
        return None, None, 0
    if stream is None:
        ws = torch.empty(need + 256, dtype=torch.uint8, device=device)
    else:
        with torch.cuda.stream(stream):
            ws = torch.empty(need + 256, dtype=torch.uint8, device=device)
    ptr = (ws.data_ptr() + 255) // 256 * 256
    return ws, ptr, need


def logical_conv_shapes(x_shape, w_shape, layout):
    """(N,C,D,H,W), (K,C/groups,T,R,S) of operands stored in `layout` (4-d operands: D = T = 1)"""
    code = _lib.LAYOUT_CODE[layout]
    x_shape, w_shape = tuple(int(e) for e in x_shape), tuple(int(e) for e in w_shape)
    if len(x_shape) == 4:
        x_shape = {0: x_shape[:2] + (1,) + x_shape[2:], 1: x_shape[:1] + (1,) + x_shape[1:],
                   2: (1,) + x_shape}[code]
        w_shape = w_shape[:2] + (1,) + w_shape[2:] if code == 0 else (1,) + w_shape
    if code == 0:
        return x_shape, w_shape
    t, r, s, c, k = w_shape
    if code == 1:
        n, d, h, w_, cx = x_shape
    else:
        d, h, w_, n, cx = x_shape
    return (n, cx, d, h, w_), (k, c, t, r, s)


def stored_conv_out_shape(oshape, layout, ndim):
    """NKDPQ extents -> the output's shape as stored in `layout` (ndim 4: without the depth)"""
    code = _lib.LAYOUT_CODE[layout]
    n, k, od, op, oq = oshape
    sp = (op, oq) if ndim == 4 else (od, op, oq)
    return {0: (n, k) + sp, 1: (n,) + sp + (k,), 2: sp + (n, k)}[code]


def conv2d(x, w, stride=1, pad=0, dil=1, out=None, config=None, stream=None, add=None, groups=1,
           layout="nchw"):
    """layout nchw: x NCHW, w K,(C/groups),R,S -> NKPQ; nhwc: x NHWC, w RSCK -> NPQK; hwnc:
    x HWNC, w RSCK -> PQNK (+ add of the output's shape)"""
    _need_device(x, w)
    st, pd, dl = (1,) + _tup(stride, 2), (0,) + _tup(pad, 2), (1,) + _tup(dil, 2)
    xs, ws = logical_conv_shapes(x.shape, w.shape, layout)
    if xs[1] != ws[1] * groups or x.dtype != w.dtype:
        raise ValueError("operand shapes / dtypes do not agree")
    oshape = conv_out_shape(xs, ws, st, pd, dl)
    if out is None:
        out = torch.empty(stored_conv_out_shape(oshape, layout, 4), dtype=_OUT_OF[x.dtype], device=x.device)
    _need_device(out)
    _check_out(out, stored_conv_out_shape(oshape, layout, 4), _OUT_OF[x.dtype], x)
    d = conv_desc(xs, ws, x.dtype, st, pd, dl, groups, layout)
    cfg = make_config(config)
    ws, ws_ptr, ws_bytes = _workspace(AMOS_OP_CONV2D, d, cfg, x.device, stream)
    epi = make_epilogue(add, tuple(out.shape), out.dtype)
    check(_lib.load().amos_run_fused(AMOS_OP_CONV2D, ctypes.byref(d), _cfg_ref(cfg), _epi_ref(epi), x.data_ptr(),
                                     w.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes, _stream_ptr(stream)))
    return out


def conv3d(x, w, stride=1, pad=0, dil=1, out=None, config=None, stream=None, add=None, groups=1,
           layout="ncdhw"):
    """layout ncdhw: x NCDHW, w K,(C/groups),T,R,S -> NKDPQ; ndhwc: x NDHWC, w TRSCK -> NDPQK;
    dhwnc: x DHWNC, w TRSCK -> DPQNK (+ add of the output's shape)"""
    _need_device(x, w)
    st, pd, dl = _tup(stride, 3), _tup(pad, 3), _tup(dil, 3)
    xs, ws = logical_conv_shapes(x.shape, w.shape, layout)
    if xs[1] != ws[1] * groups or x.dtype != w.dtype:
        raise ValueError("operand shapes / dtypes do not agree")
    oshape = conv_out_shape(xs, ws, st, pd, dl)
    if out is None:
        out = torch.empty(stored_conv_out_shape(oshape, layout, 5), dtype=_OUT_OF[x.dtype], device=x.device)
    _need_device(out)
    _check_out(out, stored_conv_out_shape(oshape, layout, 5), _OUT_OF[x.dtype], x)
    d = conv_desc(xs, ws, x.dtype, st, pd, dl, groups, layout)
    cfg = make_config(config)
    ws, ws_ptr, ws_bytes = _workspace(AMOS_OP_CONV3D, d, cfg, x.device, stream)
    epi = make_epilogue(add, tuple(out.shape), out.dtype)
    check(_lib.load().amos_run_fused(AMOS_OP_CONV3D, ctypes.byref(d), _cfg_ref(cfg), _epi_ref(epi), x.data_ptr(),
                                     w.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes, _stream_ptr(stream)))
    return out


class Gather(object):
    """device side of a dimension-separable gather (amos_gather): `tables[d][o]` = source element
    offset contributed by index o of output dimension d, or -1 where the result is zero"""

    def __init__(self, out_shape, tables, dtype, in_elems, device):
        self.out_shape = [int(e) for e in out_shape]
        self.dtype = dtype
        if not 1 <= len(self.out_shape) <= 5 or [len(t) for t in tables] != self.out_shape:
            raise ValueError("gather needs one table per output dimension, at most five")
        flat, offsets = [], []
        for t in tables:
            offsets.append(len(flat))
            flat.extend(int(e) for e in t)
        self.tables = torch.tensor(flat, dtype=torch.int32, device=device)
        d = _lib.GatherDesc()
        d.ndim, d.elem_bytes, d.in_elems = len(self.out_shape), torch.empty(0, dtype=dtype).element_size(), int(in_elems)
        for k, (ext, off) in enumerate(zip(self.out_shape, offsets)):
            d.out_shape[k], d.table_offset[k] = ext, off
        self.desc = d

    def _check(self, src, out):
        _need_device(src, out)
        if src.numel() != self.desc.in_elems or src.dtype != self.dtype or not src.is_contiguous():
            raise ValueError("gather source must be a dense %s tensor of %d elements" % (self.dtype, self.desc.in_elems))
        if list(out.shape) != self.out_shape or out.dtype != self.dtype or not out.is_contiguous():
            raise ValueError("gather output must be a dense %s tensor of shape %s" % (self.dtype, self.out_shape))

    def __call__(self, src, out=None, stream=None):
        if out is None:
            out = torch.empty(self.out_shape, dtype=self.dtype, device=src.device)
        self._check(src, out)
        check(_lib.load().amos_gather(ctypes.byref(self.desc), src.data_ptr(), self.tables.data_ptr(),
                                      out.data_ptr(), _stream_ptr(stream)))
        return out

    def time(self, src, out, number=100, repeat=1, min_repeat_ms=150, stream=None):
        self._check(src, out)
        res = (ctypes.c_double * repeat)()
        check(_lib.load().amos_time_gather(ctypes.byref(self.desc), src.data_ptr(), self.tables.data_ptr(),
                                           out.data_ptr(), _stream_ptr(stream), number, repeat, min_repeat_ms, res))
        return list(res)


class Eltwise(object):
    """device side of an element-wise stage in front of an operand (amos_eltwise): `program` is a
    list of ("load", k) / ("const", value) / "add" / "sub" / "mul" in postfix order"""

    _DT = {torch.float16: _lib.AMOS_F16, torch.bfloat16: _lib.AMOS_BF16, torch.int8: _lib.AMOS_I8}

    def __init__(self, program, n_inputs, dtype, elems):
        d = _lib.EltwiseDesc()
        d.dtype, d.n_inputs, d.elems = self._DT[dtype], int(n_inputs), int(elems)
        consts = []
        code = {"add": _lib.AMOS_ELT_ADD, "sub": _lib.AMOS_ELT_SUB, "mul": _lib.AMOS_ELT_MUL}
        if len(program) > 16:
            raise ValueError("element-wise stage of %d operations (16 at most)" % len(program))
        for k, step in enumerate(program):
            if isinstance(step, tuple) and step[0] == "load":
                d.program[k] = _lib.AMOS_ELT_LOAD | (int(step[1]) << 8)
            elif isinstance(step, tuple) and step[0] == "const":
                if len(consts) == 4:
                    raise ValueError("element-wise stage with more than four constants")
                d.program[k] = _lib.AMOS_ELT_CONST | (len(consts) << 8)
                consts.append(float(step[1]))
            else:
                d.program[k] = code[step]
        d.n_ops = len(program)
        for k, c in enumerate(consts):
            d.consts[k] = c
        self.desc, self.dtype, self.n_inputs = d, dtype, int(n_inputs)

    def _args(self, inputs, out):
        _need_device(out, *inputs)
        if len(inputs) != self.n_inputs or any(t.numel() != self.desc.elems or t.dtype != self.dtype or
                                               not t.is_contiguous() for t in list(inputs) + [out]):
            raise ValueError("element-wise stage wants %d dense %s tensors of %d elements" %
                             (self.n_inputs, self.dtype, self.desc.elems))
        return (ctypes.c_void_p * self.n_inputs)(*[t.data_ptr() for t in inputs])

    def __call__(self, inputs, out=None, stream=None):
        if out is None:
            out = torch.empty_like(inputs[0])
        ptrs = self._args(inputs, out)
        check(_lib.load().amos_eltwise(ctypes.byref(self.desc), ptrs, out.data_ptr(), _stream_ptr(stream)))
        return out

    def time(self, inputs, out, number=100, repeat=1, min_repeat_ms=150, stream=None):
        ptrs = self._args(inputs, out)
        res = (ctypes.c_double * repeat)()
        check(_lib.load().amos_time_eltwise(ctypes.byref(self.desc), ptrs, out.data_ptr(), _stream_ptr(stream),
                                            number, repeat, min_repeat_ms, res))
        return list(res)


def _epilogue_for(op, desc, add, out):
    """Epilogue for an operand laid out like the output the descriptor describes"""
    if add is None:
        return None
    if add.numel() != out.numel():
        raise ValueError("the added operand has %d elements, the output %d" % (add.numel(), out.numel()))
    epi = make_epilogue(add, tuple(add.shape), out.dtype)
    if op == AMOS_OP_GEMM:
        epi.ld = desc.ldc
    elif op == AMOS_OP_BGEMM:
        epi.ld, epi.stride = desc.g.ldc, desc.stride_c
    return epi


def run_desc(op, desc, in0, in1, out, config=None, stream=None, add=None):
    """launch an op from its C descriptor (leading dimensions and batch strides as the descriptor
    says; the tensors only supply the device memory)"""
    _need_device(in0, in1, out)
    check_operands(op, desc, in0, in1, out)
    cfg = make_config(config)
    ws, ws_ptr, ws_bytes = _workspace(op, desc, cfg, in0.device, stream)
    epi = _epilogue_for(op, desc, add, out)
    check(_lib.load().amos_run_fused(op, ctypes.byref(desc), _cfg_ref(cfg), _epi_ref(epi), in0.data_ptr(),
                                     in1.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes, _stream_ptr(stream)))
    return out


def time_op(op, desc, in0, in1, out, config=None, number=100, repeat=1, min_repeat_ms=150, stream=None,
            add=None):
    """mean seconds per launch, `repeat` values (time_evaluator semantics)"""
    _need_device(in0, in1, out)
    check_operands(op, desc, in0, in1, out)
    cfg = make_config(config)
    res = (ctypes.c_double * repeat)()
    ws, ws_ptr, ws_bytes = _workspace(op, desc, cfg, in0.device, stream)
    epi = _epilogue_for(op, desc, add, out)
    check(_lib.load().amos_time_fused(op, ctypes.byref(desc), _cfg_ref(cfg), _epi_ref(epi), in0.data_ptr(),
                                      in1.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes, _stream_ptr(stream),
                                      number, repeat, min_repeat_ms, res))
    return list(res)


def default_config(op, desc):
    cfg = KernelConfig()
    check(_lib.load().amos_default_config(op, ctypes.byref(desc), ctypes.byref(cfg)))
    return cfg


def kernel_name(op, desc, config=None):
    cfg = make_config(config)
    name = _lib.load().amos_kernel_name(op, ctypes.byref(desc), _cfg_ref(cfg))
    if name is None:
        raise _lib.AmosError(-3, _lib.load().amos_last_error().decode())
    return name.decode()


class Mxfp4(object):
    """A matrix [rows, cols] in microscaled 4 bits: blocks of 32 elements along a row share a
    power-of-two scale.  `codes` uint8 [rows, 64 * ceil(cols / 128)], two e2m1 codes a byte (the element
    of the lower index in the low half, zeros behind `cols`); `scales` uint8 [rows, codes' width / 16],
    2^(byte - 127), 255 = not a number.  Where 128 divides `cols` there is no padding.  The tensors are
    kept as they are, nothing is copied."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes, scales, cols):
        rows = _native.rows(codes, scales, cols)
        if rows is not None:
            self.codes, self.scales, self.shape = codes, scales, (rows, cols)
            return
        _need_device(codes, scales)
        pitch = mxfp4_pitch(cols)
        rows = codes.shape[0] if codes.dim() == 2 else 0
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
            raise ValueError("codes and scales are uint8, got %s and %s" % (codes.dtype, scales.dtype))
        if rows < 1 or codes.shape != (rows, pitch) or scales.shape != (rows, pitch // 16):
            raise ValueError("%d columns want codes [rows, %d] and scales [rows, %d], got %s and %s"
                             % (cols, pitch, pitch // 16, tuple(codes.shape), tuple(scales.shape)))
        if codes.device != scales.device:
            raise ValueError("codes are on %s, scales on %s" % (codes.device, scales.device))
        self.codes, self.scales, self.shape = codes, scales, (rows, int(cols))

    @property
    def device(self):
        return self.codes.device

    def __repr__(self):
        return "Mxfp4(shape=%s, device=%s)" % (self.shape, self.device)


def _mx_check(what, q):
    """an Mxfp4 whose attributes still fit each other (they can be set), contiguous and on one device"""
    if not isinstance(q, Mxfp4):
        raise ValueError("%s must be an Mxfp4, got %s" % (what, type(q)))
    rows, cols = q.shape
    pitch = mxfp4_pitch(cols)
    _need_device(q.codes, q.scales)
    for t, wide in ((q.codes, pitch), (q.scales, pitch // 16)):
        if t.dtype is not torch.uint8 or t.shape != (rows, wide) or t.device != q.codes.device:
            raise ValueError("%s of shape %s wants uint8 codes [%d, %d] and scales [%d, %d] on one device, got %s %s on %s and %s %s on %s"
                             % (what, (rows, cols), rows, pitch, rows, pitch // 16, q.codes.dtype, tuple(q.codes.shape), q.codes.device,
                                q.scales.dtype, tuple(q.scales.shape), q.scales.device))


def mxfp4_pitch(cols):
    """bytes of a row of codes"""
    if cols < 1:
        raise ValueError("a matrix of %d columns" % cols)
    return (int(cols) + 127) // 128 * 64


_FLOAT_CODE = {torch.float32: _lib.AMOS_F32, torch.float16: _lib.AMOS_F16, torch.bfloat16: _lib.AMOS_BF16}


def _float_code(what, dtype):
    code = _FLOAT_CODE.get(dtype)
    if code is None:
        raise ValueError("%s is fp32, fp16 or bf16, got %s" % (what, dtype))
    return code


# (of the module behind torch.cuda; absent from a build without a GPU runtime, where no tensor reaches them)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _on(body, device, stream, *args):
    """body(handle of the stream to launch on, *args) with `device` the current one and `stream` (None: the
    device's current one) current there, so that what the call allocates belongs to that stream's pool"""
    if stream is None:
        with torch.cuda.device(device):
            return body(_raw_stream(device.index), *args)
    if stream.device != device:
        raise ValueError("the stream belongs to %s, the tensors are on %s" % (stream.device, device))
    with torch.cuda.device(device), torch.cuda.stream(stream):
        return body(stream.cuda_stream, *args)


def _scratch(need, like):
    """device scratch from the current stream's pool: (tensor, 256-byte aligned pointer)"""
    ws = like.new_empty(need + 255, dtype=torch.uint8)
    return ws, (ws.data_ptr() + 255) & ~255


def _like_check(what, t, shape, device):
    if isinstance(t, torch.Tensor) and t.shape == shape and t.device == device and t.is_contiguous():
        return
    _need_device(t)
    if t.shape != shape or t.device != device:
        raise ValueError("%s must be of shape %s on %s, got %s on %s" % (what, tuple(shape), device, tuple(t.shape), t.device))


_CALLS_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_calls.so")


class _Native(object):
    """The entry points below in their common form (contiguous tensors on the current device, its current stream) as
    native calls, csrc/python/calls.cc: each returns None for a call that it does not take, and the call is then made,
    or refused, the long way.  Group norm with its statistics, 1 x 7 x 7 x 512: 6.6 us a call; checked and allocated in the interpreter, 11.1."""

    NAMES = ("rows", "quantize", "dequantize", "gemm", "group_norm", "group_norm_backward")

    def __getattr__(self, name):   # (the first call)
        if name not in self.NAMES:
            raise AttributeError(name)
        lib = _lib.load()
        if not os.path.exists(_CALLS_PATH):   # (built without PyTorch's headers: everything goes the long way)
            for f in self.NAMES:
                setattr(self, f, lambda *args: None)
            return object.__getattribute__(self, name)
        try:
            from . import _calls
        except ImportError as e:
            raise RuntimeError("amos_amd/_calls.so does not fit this PyTorch: build it with `python -m amos_amd.build`") from e
        _calls.setup(Mxfp4, _current_device, _raw_stream,
                     *(ctypes.cast(f, ctypes.c_void_p).value for f in (
                         lib.amos_mxfp4_quantize, lib.amos_mxfp4_dequantize, lib.amos_mxfp4_gemm, lib.amos_mxfp4_gemm_workspace_bytes,
                         lib.amos_group_norm, lib.amos_group_norm_backward, lib.amos_group_norm_workspace_bytes)))
        for f in self.NAMES:
            setattr(self, f, getattr(_calls, f))
        return object.__getattribute__(self, name)


_native = _Native()


def mxfp4_quantize(x, axis=1, out=None, stream=None):
    """x [rows, cols] (fp32, fp16, bf16) -> Mxfp4.  axis 1: blocks along the rows, shape (rows, cols);
    axis 0: blocks down the columns, the result is the quantised transpose, shape (cols, rows) -- what a
    product that sums over the rows of x takes.  A block's scale brings its largest magnitude into
    [4, 8); elements are rounded to nearest even and saturate at 6; a block with an infinity or a NaN
    stands for NaN."""
    if stream is None:
        done = _native.quantize(x, axis, out)
        if done is not None:
            return done
    _need_device(x)
    plan = _quantize_plan(x.shape, x.dtype, axis)
    if out is not None:
        _mx_check("out", out)
        if out.shape != plan[1] or out.device != x.device:
            raise ValueError("out must be an Mxfp4 of shape %s on %s, got %r" % (plan[1], x.device, out))
    return _on(_quantize, x.device, stream, plan, x, out)


def _quantize_plan(shape, dtype, axis):
    """(descriptor, shape of the result, of its codes, of its scales)"""
    if len(shape) != 2 or 0 in shape:
        raise ValueError("x must be a matrix with elements, got shape %s" % (tuple(shape),))
    if axis not in (0, 1, -1, -2):
        raise ValueError("axis %s of a matrix" % (axis,))
    d = _lib.Mxfp4Desc(shape[0], shape[1], _float_code("x", dtype), axis % 2)
    rows, cols = tuple(shape) if axis % 2 else (shape[1], shape[0])
    pitch = mxfp4_pitch(cols)
    return ctypes.byref(d), (rows, cols), (rows, pitch), (rows, pitch // 16)


def _quantize(s, plan, x, out):
    d, shape, codes, scales = plan
    if out is None:
        out = Mxfp4.__new__(Mxfp4)
        out.codes, out.scales, out.shape = x.new_empty(codes, dtype=torch.uint8), x.new_empty(scales, dtype=torch.uint8), shape
    check(_lib.load().amos_mxfp4_quantize(d, x.data_ptr(), out.codes.data_ptr(), out.scales.data_ptr(), s))
    return out


def mxfp4_dequantize(q, dtype=torch.float32, out=None, stream=None):
    """the values an Mxfp4 stands for, rounded once to `dtype` (fp32 and bf16 hold them all)"""
    if stream is None:
        done = _native.dequantize(q, dtype, out)
        if done is not None:
            return done
    _mx_check("q", q)
    if out is not None:
        _need_device(out)
        _check_out(out, q.shape, dtype, q.codes)
    d = _lib.Mxfp4Desc(q.shape[0], q.shape[1], _float_code("the result", dtype), 1)
    return _on(_dequantize, q.codes.device, stream, q, d, dtype, out)


def _dequantize(s, q, d, dtype, out):
    if out is None:
        out = q.codes.new_empty(q.shape, dtype=dtype)
    check(_lib.load().amos_mxfp4_dequantize(ctypes.byref(d), q.codes.data_ptr(), q.scales.data_ptr(), out.data_ptr(), s))
    return out


def mxfp4_gemm(a, b, out=None, out_dtype=torch.float32, add=None, bias=None, stream=None):
    """C[M,N] = sum_k A(m,k) B(n,k) (+ bias[N]) (+ add[M,N]); b is an Mxfp4 of shape (N, K), a an
    Mxfp4 of shape (M, K) or a dense matrix [M, K] (fp32, fp16, bf16) that the call quantises the way
    mxfp4_quantize does.  fp32 accumulation, one rounding to the output's type; `add` may be `out`.  No
    gradient is recorded."""
    if stream is None:
        done = _native.gemm(a, b, out, out_dtype, add, bias)
        if done is not None:
            return done
    _mx_check("b", b)
    device = b.codes.device
    dense = not isinstance(a, Mxfp4)
    if dense:
        _need_device(a)
    else:
        _mx_check("a", a)
    if a.device != device:
        raise ValueError("a is on %s, b on %s" % (a.device, device))
    if out is not None:
        out_dtype = out.dtype
    plan = _mxfp4_gemm_plan(a.shape, b.shape, a.dtype if dense else None, out_dtype)
    if out is not None:
        _like_check("out", out, plan[1], device)
    epi = None
    if add is not None or bias is not None:
        epi = _lib.Mxfp4Epilogue()
        if bias is not None:
            _like_check("bias", bias, plan[1][1:], device)
            epi.bias, epi.bias_dtype = bias.data_ptr(), _float_code("bias", bias.dtype)
        if add is not None:
            _like_check("the added operand", add, plan[1], device)
            epi.add, epi.add_dtype = add.data_ptr(), _float_code("the added operand", add.dtype)
        epi = ctypes.byref(epi)
    return _on(_mxfp4_gemm, device, stream, plan, a, b, dense, out, out_dtype, epi)


def _mxfp4_gemm_plan(a_shape, b_shape, a_dtype, out_dtype):
    """(descriptor, shape of the result, workspace bytes)"""
    if len(a_shape) != 2 or a_shape[0] < 1 or a_shape[1] != b_shape[1]:
        raise ValueError("operands do not agree: a %s, b %s" % (tuple(a_shape), b_shape))
    d = _lib.Mxfp4GemmDesc(a_shape[0], b_shape[0], b_shape[1], _lib.AMOS_MXFP4 if a_dtype is None else _float_code("a", a_dtype),
                           _float_code("the output", out_dtype))
    need = _lib.load().amos_mxfp4_gemm_workspace_bytes(ctypes.byref(d))
    return ctypes.byref(d), (a_shape[0], b_shape[0]), need


def _mxfp4_gemm(s, plan, a, b, dense, out, out_dtype, epi):
    d, shape, need = plan
    if out is None:
        out = b.codes.new_empty(shape, dtype=out_dtype)
    ws, ws_ptr = _scratch(need, b.codes) if need else (None, None)
    ac, asc = (a.data_ptr(), None) if dense else (a.codes.data_ptr(), a.scales.data_ptr())
    check(_lib.load().amos_mxfp4_gemm(d, epi, ac, asc, b.codes.data_ptr(), b.scales.data_ptr(), out.data_ptr(), ws_ptr, need, s))
    return out


_ACT_CODE = {None: _lib.AMOS_ACT_NONE, "none": _lib.AMOS_ACT_NONE, "relu": _lib.AMOS_ACT_RELU, "silu": _lib.AMOS_ACT_SILU}


def _group_norm_plan(gradient, x_shape, x_dtype, y_dtype, groups, weight_dtype, bias_dtype, eps, activation, layout):
    """(descriptor, workspace bytes, shape of the coefficients, shape of the statistics)"""
    code = _lib.LAYOUT_CODE.get(layout)
    if code not in (_lib.AMOS_LAYOUT_NHWC, _lib.AMOS_LAYOUT_HWNC):
        raise ValueError("group norm runs on the channels-last layouts (nhwc, ndhwc, hwnc, dhwnc), got %r" % (layout,))
    if len(x_shape) != len(layout) or 0 in x_shape:
        raise ValueError("layout %s wants a tensor of %d dimensions with elements, got shape %s" % (layout, len(layout), tuple(x_shape)))
    if activation not in _ACT_CODE:
        raise ValueError("activation is None, 'relu' or 'silu', got %r" % (activation,))
    ext = dict(zip(layout, x_shape))
    if groups < 1 or ext["c"] % groups:
        raise ValueError("%d channels in %d groups" % (ext["c"], groups))
    if weight_dtype is not None and bias_dtype is not None and weight_dtype != bias_dtype:
        raise ValueError("weight is %s, bias %s" % (weight_dtype, bias_dtype))
    d = _lib.GroupNormDesc()
    d.N, d.C, d.D, d.H, d.W = ext["n"], ext["c"], ext.get("d", 1), ext["h"], ext["w"]
    d.groups, d.activation, d.layout, d.eps = groups, _ACT_CODE[activation], code, eps
    d.x_dtype, d.y_dtype = _float_code("x", x_dtype), _float_code("the output", y_dtype)
    for t in (weight_dtype, bias_dtype):
        if t is not None:
            d.affine_dtype = _float_code("weight and bias", t)
    need = _lib.load().amos_group_norm_workspace_bytes(ctypes.byref(d), int(gradient))
    return ctypes.byref(d), need, (ext["c"],), (ext["n"], groups)


def _group_norm_checked(gradient, x, y_dtype, groups, weight, bias, eps, activation, layout):
    """the plan of a call, its coefficients checked"""
    plan = _group_norm_plan(gradient, x.shape, x.dtype, y_dtype, groups, None if weight is None else weight.dtype,
                            None if bias is None else bias.dtype, eps, activation, layout)
    device = x.device
    if weight is not None:
        _like_check("weight", weight, plan[2], device)
    if bias is not None:
        _like_check("bias", bias, plan[2], device)
    return plan


def _ptr(t):
    return None if t is None else t.data_ptr()


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None, layout="nhwc", out_dtype=None, out=None,
               stats=False, stream=None):
    """act(group norm of x) over a channels-last tensor (layout nhwc, ndhwc, hwnc or dhwnc): per image
    and group of neighbouring channels h = (x - mean) / sqrt(var + eps), then h * weight[C] + bias[C],
    then None / 'relu' / 'silu'.  Statistics and arithmetic are fp32, the result is x's type or
    out_dtype (a convolution's fp32 output can leave at 16 bits for the next one); `out` may be x.  A group
    whose values or squared deviations add up to 2^128 and more (deviations from about 2^64 / sqrt(elements
    of the group) up), or that holds an infinity or a NaN, is NaN.  No gradient is recorded.
    stats=True: (y, mean, rstd), both fp32 [N, groups], for group_norm_backward."""
    if stream is None:
        done = _native.group_norm(x, groups, weight, bias, eps, activation, layout, out_dtype, out, stats)
        if done is not None:
            return done
    _need_device(x)
    if out is not None:
        _like_check("out", out, x.shape, x.device)
        if out_dtype is not None and out_dtype != out.dtype:
            raise ValueError("out is %s, out_dtype %s" % (out.dtype, out_dtype))
        out_dtype = out.dtype
    elif out_dtype is None:
        out_dtype = x.dtype
    plan = _group_norm_checked(False, x, out_dtype, groups, weight, bias, eps, activation, layout)
    return _on(_group_norm, x.device, stream, plan, x, weight, bias, out, out_dtype, stats)


def _group_norm(s, plan, x, weight, bias, out, out_dtype, stats):
    d, need, _, stats_shape = plan
    if out is None:
        out = x.new_empty(x.shape, dtype=out_dtype)
    mean = rstd = None
    if stats:
        mean, rstd = x.new_empty(stats_shape, dtype=torch.float32), x.new_empty(stats_shape, dtype=torch.float32)
    ws, ws_ptr = _scratch(need, x) if need else (None, None)
    check(_lib.load().amos_group_norm(d, x.data_ptr(), _ptr(weight), _ptr(bias), out.data_ptr(), _ptr(mean), _ptr(rstd), ws_ptr, need, s))
    return (out, mean, rstd) if stats else out


def group_norm_backward(dy, x, mean, rstd, groups, weight=None, bias=None, activation=None, layout="nhwc", stream=None):
    """gradients of group_norm: (dx of x's type, dweight, dbias in fp32 -- None where the coefficient
    is), from the statistics that group_norm(..., stats=True) returned for x (rstd below 2^63: its square
    is formed in fp32)"""
    if stream is None:
        done = _native.group_norm_backward(dy, x, mean, rstd, groups, weight, bias, activation, layout)
        if done is not None:
            return done
    _need_device(dy, x, mean, rstd)
    if dy.shape != x.shape or dy.device != x.device:
        raise ValueError("dy is %s on %s, x %s on %s" % (tuple(dy.shape), dy.device, tuple(x.shape), x.device))
    plan = _group_norm_checked(True, x, dy.dtype, groups, weight, bias, 0.0, activation, layout)
    for what, t in (("mean", mean), ("rstd", rstd)):
        if t.shape != plan[3] or t.device != x.device or t.dtype != torch.float32:
            raise ValueError("%s must be fp32 of shape %s on %s, got %s %s on %s" % (what, plan[3], x.device, t.dtype, tuple(t.shape), t.device))
    return _on(_group_norm_backward, x.device, stream, plan, dy, x, mean, rstd, weight, bias)


def _group_norm_backward(s, plan, dy, x, mean, rstd, weight, bias):
    d, need, coefficients, _ = plan
    dx = x.new_empty(x.shape)
    dweight = None if weight is None else x.new_empty(coefficients, dtype=torch.float32)
    dbias = None if bias is None else x.new_empty(coefficients, dtype=torch.float32)
    ws, ws_ptr = _scratch(need, x) if need else (None, None)
    check(_lib.load().amos_group_norm_backward(d, dy.data_ptr(), x.data_ptr(), _ptr(weight), _ptr(bias), mean.data_ptr(),
                                               rstd.data_ptr(), dx.data_ptr(), _ptr(dweight), _ptr(dbias), ws_ptr, need, s))
    return dx, dweight, dbias


def device_info():
    info = _lib.DeviceInfo()
    check(_lib.load().amos_device_info(ctypes.byref(info)))
    return info
