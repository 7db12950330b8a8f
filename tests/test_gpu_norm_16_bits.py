"""The norm, gate and residual with the next block's norm on 16-bit features: the gradients of float32 scales and weights are good to
float32, and those of the features are rounded once (against float64 sums over the same 16-bit inputs)."""
import pytest
import torch

import cuequivariance_b200 as cb
from _norm_reference import blocks_of, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16
U = 2.0**-24


def bounds(blocks, rows, gate):
    """Roundings of 2^-24 that a term of dw, of the sum that reaches h, and of ds meets, and of their sums over rows.

    chain: a sum over a block, a lane's share and five steps over the warp.  r: half of that, product, reciprocal (4) and sum halved, and 4 of rsqrtf.
    act: 2 + 1.173 |g| units in the last place, 2 roundings each, of the fast exponential (|g| < 8: 23), sum, reciprocal (4), product, 2 to spare.
    h = x + s act r y: act, r and 3.  dw = r(h) sum_i gn h: h, its own r, dim, 3; the reference's magnitude holds what h does to r(h).
    What reaches h: go + w r gn - r (r (dot / n)) h, dot a sum over dw's terms: at most dw, one more chain, twice r(h) with its h, 10.
    ds = act r sum_i o y: that, act, r, dim, 3.  Over rows: a warp's rows of the 148 warps at least that share them, up to 32 rows side by side, at
    most 148 * 16 warps in chains of 19, and 9 steps."""
    chain = max(m * d for m, d in blocks) / 32 + 10
    dim = max(d for _, d in blocks)
    r = chain / 2 + 8
    act = 32 if gate else 0
    h = act + r + 3
    over_rows = rows / 148 + 8 + 32 + 19 + 9
    dw = h + r + dim + 3
    o = dw + chain + 2 * (h + r) + 10
    return {"dw": dw + over_rows, "dx": o, "ds": o + act + r + dim + 3 + over_rows, "dg": o + 2 * act + r + dim + 6, "dy": 2 * (o + act + 2 * r + chain + dim) + 10}


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("layout", [cb.mul_ir, cb.ir_mul], ids=["mul_ir", "ir_mul"])
@pytest.mark.parametrize("gate", [None, "sigmoid", "silu"])
@pytest.mark.parametrize("irreps,rows", [
    ("64x0e+64x1o", 1), ("64x0e+64x1o", 21), ("64x0e+64x1o", 1999), ("128x0e+128x1o+128x2e+128x3o", 37), ("5x0e+3x1o+2x2e", 77),
    ("33x0e+7x1o", 5), ("192x0e+130x1o+40x4e", 19), ("48x0e+36x2e", 260),
])
def test_gradients_behind_a_rounded_sum(irreps, rows, gate, layout, dtype):
    m = cb.GatedResidual(irreps, layout=layout, gate=gate, norm_output=True, internal_weights=False)
    blocks = blocks_of(m.irreps)
    gen = torch.Generator().manual_seed(rows)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    v = {"x": randn(rows, m.irreps.dim).to(dtype), "y": randn(rows, m.irreps.dim).to(dtype)}
    if gate:
        v["g"] = (1.5 * randn(rows, m.irreps.num_irreps)).clamp(-7, 7).to(dtype)
    v["s"], v["w"] = 0.5 + 0.1 * randn(m.irreps.num_irreps), 1 + 0.2 * randn(m.irreps.num_irreps)
    go, gn = randn(rows, m.irreps.dim).to(dtype), randn(rows, m.irreps.dim).to(dtype)
    d = {k: t.to(DEV).requires_grad_(True) for k, t in v.items()}
    outs = m(d["x"], d["y"], d.get("g"), d["s"], d["w"])
    for cots, first in (((go, gn), go), ((None, gn), None)):
        if first is None:
            grads = torch.autograd.grad(outs[1], tuple(d.values()), gn.to(DEV), retain_graph=True)
        else:
            grads = torch.autograd.grad(outs, tuple(d.values()), [c.to(DEV) for c in cots], retain_graph=True)
        ref = reference(blocks, layout is cb.mul_ir, m.eps, gate, False, v["x"], v["y"], v.get("g"), v["s"], v["w"], first, gn)
        units = bounds(blocks, rows, gate)
        for name, t in zip(["d" + k for k in d], grads):
            value, mag = ref[name]
            tol = units[name] * U * mag + 1e-37
            if name not in ("ds", "dw"):
                tol = tol + torch.finfo(dtype).eps / 2 * value.abs() * (1 + 2.0**-7) + (2.0**-25 if dtype == F16 else 0)
            else:
                assert t.dtype == torch.float32
            err = (t.cpu().double() - value).abs()
            assert bool((err <= tol).all()), (name, err.max().item(), (err / tol).max().item())
