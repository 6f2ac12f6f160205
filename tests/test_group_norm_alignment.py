"""Pointers of the group norm calls that are off their elements' size are refused, each by its own type, on the host: no
call here reaches a launch."""
import ctypes

import pytest

from amos_amd import _lib
from test_mxfp4_refusals import AT, norm_desc

TYPES = {_lib.AMOS_F32: 4, _lib.AMOS_F16: 2, _lib.AMOS_BF16: 2}
FORWARD = ["x", "weight", "bias", "y", "mean", "rstd"]
GRADIENT = ["dy", "x", "weight", "bias", "mean", "rstd", "dx", "dweight", "dbias"]


@pytest.mark.parametrize("affine", sorted(TYPES))
@pytest.mark.parametrize("y", sorted(TYPES))
@pytest.mark.parametrize("x", sorted(TYPES))
def test_misaligned_pointers(x, y, affine):
    lib = _lib.load()
    d = norm_desc(x_dtype=x, y_dtype=y, affine_dtype=affine)
    size = dict(x=TYPES[x], dx=TYPES[x], y=TYPES[y], dy=TYPES[y], weight=TYPES[affine], bias=TYPES[affine])
    for names, call in ((FORWARD, lib.amos_group_norm), (GRADIENT, lib.amos_group_norm_backward)):
        for name in names:
            for off in range(1, size.get(name, 4)):
                at = [AT + off if n == name else AT for n in names]
                assert call(ctypes.byref(d), *at, AT, 1 << 30, None) == _lib.AMOS_ERR_BAD_ARG, (name, off)
                assert b"misaligned" in lib.amos_last_error()
