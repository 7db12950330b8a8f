"""Irrep blocks that do not fit into shared memory are refused by the pass that a user calls first, whatever their length (no GPU: made
before a launch)."""
import ctypes as C

import pytest

from cuequivariance_b200 import _lib


def _args(mode, blocks, dtype, gate=0, **kw):
    a = _lib.NormArgs()
    a.struct_bytes, a.mode, a.mul_ir, a.num_blocks, a.rows, a.eps, a.dtype, a.gate = C.sizeof(a), mode, 1, len(blocks), 3, 1e-5, dtype, gate
    a.param_dtype = dtype if dtype == 1 else 0
    a.blocks = (_lib.NormBlock * len(blocks))(*blocks)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("mode", [_lib.NORM_BRANCH, _lib.NORM_ALONE, _lib.NORM_BOTH])
@pytest.mark.parametrize("count", [1, 31, 63, 64])
@pytest.mark.parametrize("mul", [1 << 20, (1 << 20) - 1, 600001])
def test_no_length_wraps_around(mul, count, mode, dtype):
    """63 blocks of a million values in float64: a stage of all of them would have 2.1 GB."""
    a = _args(mode, ((mul, 1),) * count, dtype)
    assert _lib.lib().cueq_b200_norm_parts(C.byref(a)) == -1
    assert "shared memory" in _lib.lib().cueq_b200_last_error().decode()


@pytest.mark.parametrize("mode,blocks,dtype", [
    (_lib.NORM_BOTH, ((1024, 7),), 1), (_lib.NORM_ALONE, ((20000, 1),), 0), (_lib.NORM_BRANCH, ((12000, 1),), 0), (_lib.NORM_BOTH, ((8, 3), (4000, 5)), 2),
])
def test_a_forward_pass_whose_gradient_would_not_fit(mode, blocks, dtype):
    """Refused where statistics are kept for a backward pass, run where none are.  No rows: nothing is launched."""
    L = _lib.lib()
    width = sum(m * d for m, d in blocks)
    a = _args(mode, blocks, dtype, x=16, ldx=width, y=16, ldy=width, scale=16, weight=16, out=16, norm=16)
    a.rows = 0
    assert L.cueq_b200_norm_parts(C.byref(a)) == -1
    assert L.cueq_b200_norm_forward(C.byref(a), None) == 0
    a.stats = 16
    assert L.cueq_b200_norm_forward(C.byref(a), None) != 0
    assert "shared memory" in L.cueq_b200_last_error().decode()
