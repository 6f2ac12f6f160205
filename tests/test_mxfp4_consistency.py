"""An Mxfp4's attributes can be set: a call with one whose tensors do not fit its shape any more is refused before anything
is launched.  On the host, with the launch and the demand for device memory replaced."""
import pytest
import torch

from amos_amd import ops


def made(rows, cols):
    q = ops.Mxfp4.__new__(ops.Mxfp4)
    q.codes = torch.zeros(rows, ops.mxfp4_pitch(cols), dtype=torch.uint8)
    q.scales = torch.zeros(rows, ops.mxfp4_pitch(cols) // 16, dtype=torch.uint8)
    q.shape = (rows, cols)
    return q


@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(ops, "_on", lambda body, *args: calls.append(body))
    real = ops._need_device

    def contiguous(*tensors):
        for t in tensors:
            if not isinstance(t, torch.Tensor):
                real(t)
            if not t.is_contiguous():
                raise ValueError("operands must be contiguous")
    monkeypatch.setattr(ops, "_need_device", contiguous)
    return calls


SPOIL = {
    "more rows": lambda q: setattr(q, "shape", (q.shape[0] * 2, q.shape[1])),
    "more columns": lambda q: setattr(q, "shape", (q.shape[0], q.shape[1] + 128)),
    "fewer codes": lambda q: setattr(q, "codes", q.codes[:-1]),
    "narrower codes": lambda q: setattr(q, "codes", q.codes[:, :-64].contiguous()),
    "fewer scales": lambda q: setattr(q, "scales", q.scales[:-1]),
    "turned codes": lambda q: setattr(q, "codes", q.codes.t()),
    "strided scales": lambda q: setattr(q, "scales", q.scales.repeat(1, 2)[:, ::2]),
    "flat codes": lambda q: setattr(q, "codes", q.codes.reshape(-1)),
    "wide codes": lambda q: setattr(q, "codes", q.codes.int()),
    "no tensor": lambda q: setattr(q, "scales", None),
}


@pytest.mark.parametrize("spoil", sorted(SPOIL))
def test_spoilt_matrices_are_refused(launched, spoil):
    uses = {
        "quantize": lambda q: ops.mxfp4_quantize(torch.zeros(*q.shape), out=q),
        "dequantize": lambda q: ops.mxfp4_dequantize(q),
        "b": lambda q: ops.mxfp4_gemm(torch.zeros(3, q.shape[1]), q),
        "a": lambda q: ops.mxfp4_gemm(q, made(5, q.shape[1])),
    }
    for name, use in uses.items():
        use(made(6, 200))
        assert len(launched) == 1, name      # as it was made: taken
        launched.clear()
        q = made(6, 200)
        SPOIL[spoil](q)
        with pytest.raises((ValueError, RuntimeError)):
            use(q)
        assert not launched, name
