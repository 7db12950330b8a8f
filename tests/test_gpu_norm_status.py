"""Sums of parameters' gradients after a wait that ran out: the status word is set, as a warp that gives up sets it, and the sums, of which that
warp has left none, are not handed to the caller."""
import ctypes as C

import pytest
import torch

from cuequivariance_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_no_sums_after_a_wait_that_ran_out(dtype):
    rows, width, channels = 50, 8, 8
    gen = torch.Generator().manual_seed(0)
    x, gn = (torch.randn(rows, width, generator=gen).to(DEV, dtype) for _ in range(2))
    w, norm, dx, dw = torch.ones(channels, device=DEV, dtype=dtype), torch.empty_like(x), torch.empty_like(x), torch.full((channels,), 7.0, device=DEV, dtype=dtype)
    status = torch.zeros(1, device=DEV, dtype=torch.int32)
    stats = torch.zeros(rows, 1, 4, device=DEV, dtype=dtype)
    a = _lib.NormArgs()
    a.struct_bytes, a.mode, a.mul_ir, a.num_blocks, a.rows, a.eps = C.sizeof(a), _lib.NORM_ALONE, 1, 1, rows, 1e-5
    a.dtype = a.param_dtype = int(dtype == torch.float64)
    a.blocks = (_lib.NormBlock * 1)((8, 1))
    a.x, a.ldx, a.weight, a.norm, a.stats, a.status = x.data_ptr(), width, w.data_ptr(), norm.data_ptr(), stats.data_ptr(), status.data_ptr()
    L, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    _lib.check(L.cueq_b200_norm_forward(C.byref(a), stream))
    n = L.cueq_b200_norm_parts(C.byref(a))
    parts = torch.empty(n, device=DEV, dtype=dtype)
    a.h, a.ldh, a.gn, a.ldgn, a.dx, a.dweight, a.parts, a.parts_values = (x.data_ptr(), width, gn.data_ptr(), width, dx.data_ptr(), dw.data_ptr(),
                                                                          parts.data_ptr(), n)
    status.fill_(2)
    _lib.check(L.cueq_b200_norm_backward(C.byref(a), stream))
    assert bool((dw == 7.0).all())
    status.zero_()
    _lib.check(L.cueq_b200_norm_backward(C.byref(a), stream))
    r = (x.double().pow(2).mean(1, keepdim=True) + 1e-5).rsqrt()
    want = (gn.double() * x.double() * r).sum(0)
    assert bool(((dw.double() - want).abs() <= 200 * torch.finfo(dtype).eps * (gn * x).abs().double().mul(r).sum(0)).all())
