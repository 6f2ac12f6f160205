"""The native calls of the 4-bit operators and group norm: that they take what they are meant to take, leave the rest, and
agree with the way through the interpreter, in results and in refusals."""
import threading

import pytest
import torch

from test_gpu_channels_last_block import every_call

pytestmark = pytest.mark.gpu


class Watched(object):
    """ops._native with a note of every answer: (entry point, whether it took the call)"""

    def __init__(self, native):
        self.native, self.answers = native, []

    def __getattr__(self, name):
        call = getattr(self.native, name)

        def noted(*args):
            done = call(*args)
            self.answers.append((name, done is not None))
            return done
        return noted


@pytest.fixture
def watched(gpu, monkeypatch):
    from amos_amd import ops
    w = Watched(ops._native)
    monkeypatch.setattr(ops, "_native", w)
    return w


def poisoned(q):
    """an Mxfp4 like q with other contents"""
    from amos_amd import ops
    return ops.Mxfp4(torch.full_like(q.codes, 0x5a), torch.full_like(q.scales, 3), q.shape[1])


def test_common_calls_are_taken_and_agree(watched):
    """a named stream goes through the interpreter, the current one is the native call's"""
    calls = list(every_call())
    for name, call, tensors in calls:
        watched.answers.clear()
        one = [t.clone() for t in tensors(call(None))]
        assert watched.answers and all(took for _, took in watched.answers), name
        watched.answers.clear()
        two = tensors(call(torch.cuda.current_stream()))
        assert not [a for a in watched.answers if a[0] != "rows"], name
        assert len(one) == len(two)
        for a, b in zip(one, two):
            assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b), name


@pytest.mark.parametrize("axis", [0, 1])
def test_quantize_into(watched, axis):
    from amos_amd import ops
    x = torch.randn(24, 200, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    want = ops.mxfp4_quantize(x, axis=axis)
    for stream in (None, torch.cuda.current_stream()):
        out = poisoned(want)
        watched.answers.clear()
        assert ops.mxfp4_quantize(x, axis=axis, out=out, stream=stream) is out
        assert watched.answers == ([("quantize", True)] if stream is None else [])
        assert torch.equal(out.codes, want.codes) and torch.equal(out.scales, want.scales)


def refused():
    """(entry point, call with a stream or None) that both ways have to refuse"""
    from amos_amd import ops
    z = lambda *shape: torch.zeros(*shape, device="cuda")
    x, q, wide = z(4, 64), ops.mxfp4_quantize(z(4, 64)), ops.mxfp4_quantize(z(4, 200))
    for name, args, more in [
            ("quantize", (x.long(),), {}), ("quantize", (x.t(),), {}), ("quantize", (x[None],), {}), ("quantize", (x[:0],), {}),
            ("quantize", (x.cpu(),), {}), ("quantize", (x,), dict(axis=2)), ("quantize", (x,), dict(axis=-3)), ("quantize", (x,), dict(out=x)),
            ("quantize", (x,), dict(axis=0, out=q)), ("quantize", (x,), dict(out=wide)), ("quantize", (None,), {}),
            ("dequantize", (x,), {}), ("dequantize", (q, torch.int8), {}), ("dequantize", (q, torch.float16), dict(out=x)),
            ("dequantize", (q,), dict(out=x[:3])), ("dequantize", (q,), dict(out=z(64, 4).t())), ("dequantize", (q,), dict(out=x.cpu())),
            ("gemm", (x, x), {}), ("gemm", (q, wide), {}), ("gemm", (x[0], q), {}), ("gemm", (x.long(), q), {}), ("gemm", (x.t(), q), {}),
            ("gemm", (x[:0], q), {}), ("gemm", (x.cpu(), q), {}), ("gemm", (q, q), dict(out_dtype=torch.int8)), ("gemm", (q, q), dict(bias=x[0])),
            ("gemm", (q, q), dict(bias=z(4).long())), ("gemm", (q, q), dict(add=x)), ("gemm", (q, q), dict(add=z(4, 4).int())),
            ("gemm", (q, q), dict(add=z(4, 8)[:, ::2])), ("gemm", (q, q), dict(out=x)), ("gemm", (q, q), dict(out=z(4, 4).long())),
            ("gemm", (q, q), dict(out=z(4, 8)[:, ::2])), ("gemm", (q, q), dict(bias=z(4).cpu()))]:
        yield name, lambda s, f=getattr(ops, "mxfp4_" + name), a=args, m=more: f(*a, stream=s, **m)
    v, s22, w = z(2, 3, 3, 8), z(2, 2), z(8)
    for args, more in [((v, 3), {}), ((v, 0), {}), ((v, -2), {}), ((v, 16), {}), ((v, 2), dict(layout="nchw")), ((v, 2), dict(layout="ndhwc")), ((v[0], 2), {}),
                       ((v, 2), dict(activation="gelu")), ((v.transpose(1, 3), 2), {}), ((v[:0], 2), {}), ((v.long(), 2), {}), ((v.cpu(), 2), {}),
                       ((v, 2), dict(out_dtype=torch.int8)), ((v, 2, w[:4]), {}), ((v, 2, w, w.half()), {}), ((v, 2, w.long()), {}), ((v, 2, None, w[::2]), {}),
                       ((v, 2, w.cpu()), {}), ((v, 2), dict(out=v[:1])), ((v, 2), dict(out=v, out_dtype=torch.float16)), ((v, 2), dict(out=v.long())),
                       ((v, 2), dict(eps=-1.0)), ((v, 2), dict(eps=float("nan"))), ((v, 2), dict(eps=float("inf")))]:
        yield "group_norm", lambda s, a=args, m=more: ops.group_norm(*a, stream=s, **m)
    for args, more in [((v[:1], v, s22, s22, 2), {}), ((v, v, s22[:1], s22, 2), {}), ((v, v, s22, s22.double(), 2), {}), ((v, v, s22, s22, 4), {}),
                       ((v, v, s22.t(), s22[:, ::2], 2), {}), ((v.long(), v, s22, s22, 2), {}), ((v, v, s22, s22, 2, w[:4]), {}), ((v, v, s22, s22, 2, w, w.half()), {}),
                       ((v, v, s22.cpu(), s22, 2), {}), ((v, v, s22, s22, 2), dict(activation="gelu")), ((v, v, s22, s22, 2), dict(layout="nchw"))]:
        yield "group_norm_backward", lambda s, a=args, m=more: ops.group_norm_backward(*a, stream=s, **m)


def test_refused_calls_are_refused_both_ways(watched):
    """what the native call leaves, the interpreter refuses, in the same words as on a named stream"""
    for i, (name, call) in enumerate(refused()):
        said = []
        for stream in (None, torch.cuda.current_stream()):
            watched.answers.clear()
            with pytest.raises((ValueError, RuntimeError)) as e:
                call(stream)
            said.append((type(e.value), str(e.value)))
            assert watched.answers == ([(name, False)] if stream is None else []), (i, name)
        assert said[0] == said[1], (i, name)


def test_calls_from_threads_all_finish(gpu):
    """several threads at once, each on a stream of its own: every loop runs to its end, none raises, all agree"""
    want = [[t.clone() for t in tensors(call(None))] for _, call, tensors in every_call()]
    torch.cuda.synchronize()
    wrong, done = [], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    calls = list(every_call())
                    torch.cuda.current_stream().synchronize()
                    for ours, (name, call, tensors) in zip(want, calls):
                        if not all(torch.equal(a, b) for a, b in zip(ours, tensors(call(None)))):
                            wrong.append((k, name))
                    done.append((k, len(calls)))
        except BaseException as e:
            wrong.append((k, repr(e)))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(100)
    assert not wrong
    assert sorted(done) == sorted((k, len(want)) for k in range(4) for _ in range(5))


def test_without_the_native_calls(gpu, monkeypatch, tmp_path):
    """a build without them: every call goes through ctypes, with the same results"""
    from amos_amd import ops
    calls = list(every_call())
    want = [[t.clone() for t in tensors(call(None))] for _, call, tensors in calls]
    monkeypatch.setattr(ops, "_CALLS_PATH", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(ops, "_native", ops._Native())
    for ours, (name, call, tensors) in zip(want, every_call()):
        assert all(torch.equal(a, b) for a, b in zip(ours, tensors(call(None)))), name
