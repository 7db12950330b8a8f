"""Refusals of the norm modules and of their C entries (no GPU: every one is made before a launch)."""
import copy
import ctypes as C
import pickle

import pytest
import torch

import cuequivariance_b200 as cb
from cuequivariance_b200 import _lib


def test_constructor_refusals():
    for bad in (dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(saved_activations="int4")):
        with pytest.raises(ValueError):
            cb.IrrepsNorm("4x0e", **bad)
    with pytest.raises(ValueError, match="gate"):
        cb.GatedResidual("4x0e", gate="tanh")
    with pytest.raises(ValueError, match="blocks"):
        cb.IrrepsNorm("+".join(["1x0e", "1x1o"] * 33))
    with pytest.raises(ValueError, match="blocks"):
        cb.IrrepsNorm("0x0e")


def test_parameters():
    m = cb.GatedResidual("4x0e+3x1o", norm_output=True, initial_scale=0.25)
    assert m.scale.shape == m.weight.shape == (7,) and float(m.scale[0]) == 0.25 and float(m.weight[0]) == 1.0
    assert cb.GatedResidual("4x0e+3x1o").weight is None
    assert dict(cb.GatedResidual("4x0e", internal_weights=False).named_parameters()) == {}
    for copied in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert [(b.mul, b.dim) for b in copied._block.blocks] == [(4, 1), (3, 3)]


def test_call_refusals():
    n, r = cb.IrrepsNorm("4x0e+4x1o"), cb.GatedResidual("4x0e+4x1o")
    x = torch.zeros(3, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        n(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        r(x, x, torch.zeros(3, 8))
    with pytest.raises(ValueError, match="shape"):
        n(x[:, :15])
    with pytest.raises(ValueError, match="shape"):
        n(x[0])
    with pytest.raises(ValueError, match="Internal weights"):
        n(x, torch.ones(8))


def _args(mode, blocks=((4, 1), (4, 3)), rows=3, **kw):
    a = _lib.NormArgs()
    a.struct_bytes, a.mode, a.mul_ir, a.num_blocks, a.rows, a.eps = C.sizeof(a), mode, 1, len(blocks), rows, 1e-5
    a.blocks = (_lib.NormBlock * len(blocks))(*blocks)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(struct_bytes=8), "another argument block"), (dict(mode=4), "mode"), (dict(gate=3), "gate"), (dict(dtype=7), "element type"),
    (dict(num_blocks=0), "irrep blocks"), (dict(num_blocks=65), "irrep blocks"), (dict(rows=-1), "rows"), (dict(eps=0.0), "eps"), (dict(eps=float("inf")), "eps"), (dict(eps=1e-39), "eps"), (dict(eps=1e-39, dtype=1), "null weight"),
    (dict(codes=16, dtype=1), "8 bits"), (dict(stats_stride=5), "stride"), (dict(), "null weight"), (dict(weight=16), "operand"),
    (dict(weight=16, x=16, ldx=8), "operand"), (dict(weight=16, x=16, ldx=16), "null result"),
    (dict(weight=16, x=16, ldx=16, norm=16, codes=16, ld_codes=16), "codes need"),
    (dict(weight=16, x=16, ldx=16, norm=16, codes=16, ld_codes=32), "null statistics"),
    (dict(weight=16, x=16, ldx=16, norm=16, stats=8), "statistics must be"),
])
def test_forward_refusals(change, text):
    a = _args(_lib.NORM_ALONE)
    for k, v in change.items():
        setattr(a, k, v)
    assert _lib.lib().cueq_b200_norm_forward(C.byref(a), None) != 0
    assert text in _lib.lib().cueq_b200_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(), "null scale"), (dict(scale=16), "gates"), (dict(scale=16, g=16, ldg=8), "null statistics"),
    (dict(scale=16, g=16, ldg=8, stats=16), "kept operand"), (dict(scale=16, g=16, ldg=8, stats=16, y=16, ldy=16), "cotangent"),
    (dict(scale=16, g=16, ldg=8, stats=16, y=16, ldy=16, go=16, ldgo=15), "cotangent"),
    (dict(scale=16, g=16, ldg=8, stats=16, y=16, ldy=16, go=16, ldgo=16, dy=16), "null result"),
    (dict(scale=16, g=16, ldg=8, stats=16, y=16, ldy=16, go=16, ldgo=16, dy=16, dg=16), "partial sums"),
    (dict(scale=16, g=16, ldg=8, stats=16, y=16, ldy=16, go=16, ldgo=16, dy=16, dg=16, parts=16, parts_values=3), "partial sums"),
])
def test_backward_refusals(change, text):
    a = _args(_lib.NORM_BRANCH, gate=1)
    for k, v in change.items():
        setattr(a, k, v)
    assert _lib.lib().cueq_b200_norm_backward(C.byref(a), None) != 0
    assert text in _lib.lib().cueq_b200_last_error().decode()


def test_sizes_that_a_caller_allocates():
    L = _lib.lib()
    a = _args(_lib.NORM_BOTH, gate=1, codes=16)
    assert L.cueq_b200_norm_code_bytes(C.byref(a)) == 2 * (16 + 16) + 2 * 16 and L.cueq_b200_norm_stats(C.byref(a)) == 2 * 8
    m = cb.GatedResidual("4x0e+4x1o", norm_output=True, saved_activations="int8")
    assert m._block.code_bytes == L.cueq_b200_norm_code_bytes(C.byref(a)) and m._block.stats_stride == 8
    a = _args(_lib.NORM_ALONE)
    assert L.cueq_b200_norm_stats(C.byref(a)) == 2 * 4
    # a thread block per three rows at most; every thread block of an irrep block leaves one sum per channel and parameter
    assert L.cueq_b200_norm_parts(C.byref(a)) % (2 * 4) == 0 and L.cueq_b200_norm_parts(C.byref(a)) <= 2 * 8 * 3
    a = _args(_lib.NORM_BRANCH, blocks=((100000, 1),))
    assert L.cueq_b200_norm_parts(C.byref(a)) == -1 and "shared memory" in L.cueq_b200_last_error().decode()


def test_linear_refusals():
    kw = dict(layout=cb.mul_ir, saved_activations="int8")
    for bad in (("48x0e", "32x0e"), ("160x0e", "32x0e"), ("32x4e", "32x4e"), ("32x0e+32x0e", "32x0e")):
        with pytest.raises(ValueError, match="int8"):
            cb.Linear(*bad, **kw)
    with pytest.raises(ValueError, match="saved_activations"):
        cb.Linear("32x0e", "32x0e", saved_activations="fp8")
    m = cb.Linear("32x0e", "32x0e", **kw)
    with pytest.raises(ValueError, match="CUDA"):
        m(torch.zeros(4, 32))


@pytest.mark.parametrize("change,text", [
    (dict(struct_bytes=4), "another block"), (dict(codes=None), "null codes"), (dict(ld_codes=112), "rows of codes"), (dict(ld_codes=136), "rows of codes"),
    (dict(ld_steps=8), "rows of codes"), (dict(ld_steps=11), "rows of codes"), (dict(rows=8), "class bounds"), (dict(steps=8), "rows of codes"),
])
def test_refusals_of_the_linear_codes(change, text):
    m = cb.Linear("32x0e+32x1o", "32x0e+32x1o", layout=cb.mul_ir, internal_weights=False, shared_weights=True)
    a, c = _lib.LinearArgs(), _lib.LinearCodes()
    a.x = a.w = a.out = a.parts = 16
    a.bounds, a.parts_floats = _lib.int32_array([0, 9]), 1 << 20
    a.num_paths, a.num_classes, a.struct_bytes = 2, 1, C.sizeof(a)
    a.ldx = a.ldo = 128
    for q, (wo, u, v, xo, oo, d, k) in zip(a.paths, m._fused_plan["paths"]):
        q.u, q.v, q.d, q.x_off, q.out_off, q.w_off, q.c = u, v, d, xo, oo, wo, k
    c.struct_bytes, c.rows, c.codes, c.ld_codes, c.steps, c.ld_steps = C.sizeof(c), 9, 16, 128, 16, 12
    for k, v in change.items():
        setattr(c, k, v)
    L = _lib.lib()
    for fn in (L.cueq_b200_linear_pack, L.cueq_b200_linear_gw_codes):
        assert fn(C.byref(a), C.byref(c), None) != 0 and text in L.cueq_b200_last_error().decode()
        assert fn(C.byref(a), None, None) != 0
