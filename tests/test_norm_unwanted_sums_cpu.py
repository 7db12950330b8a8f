"""The C entry of the norms' backward pass without gradients of the parameters: refusals (no GPU: made before a launch)."""
import ctypes as C

from cuequivariance_b200 import _lib


def _args(**kw):
    a = _lib.NormArgs()
    a.struct_bytes, a.mode, a.mul_ir, a.num_blocks, a.rows, a.eps = C.sizeof(a), _lib.NORM_ALONE, 1, 2, 0, 1e-5
    a.blocks = (_lib.NormBlock * 2)((4, 1), (4, 3))
    for k, v in dict(weight=16, stats=16, h=16, ldh=16, gn=16, ldgn=16, dx=16, parts_values=-1, **kw).items():
        setattr(a, k, v)
    return a


def test_no_room_but_a_gradient():
    L = _lib.lib()
    a = _args(dweight=16)
    assert L.cueq_b200_norm_backward(C.byref(a), None) != 0
    assert "partial sums" in L.cueq_b200_last_error().decode()


def test_no_room_and_no_gradient():
    """No rows: nothing is launched."""
    a = _args()
    assert _lib.lib().cueq_b200_norm_backward(C.byref(a), None) == 0
