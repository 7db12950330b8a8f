"""Norms of blocks so long that a warp has one stage, of which rows or their ends move element by element, with several refills per warp."""
import pytest
import torch

import cuequivariance_b200 as cb
from _norm_reference import blocks_of, bound, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("irreps,rows,dtype", [
    ("2045x0e+3x1o", 3001, torch.float32),             # odd rows: element by element
    ("3001x0e", 2203, torch.float32),
    ("2046x0e", 2999, torch.float32),                  # dense, in stages of two rows: the ends of an odd number of rows
    ("4097x0e+5x1o", 1601, torch.bfloat16),
    ("1023x1o+1x0e", 1801, torch.float64),
])
def test_stages_that_are_refilled(irreps, rows, dtype):
    m = cb.GatedResidual(irreps, norm_output=True, internal_weights=False)
    n = cb.IrrepsNorm(irreps, internal_weights=False)
    blocks, channels = blocks_of(m.irreps), m.irreps.num_irreps
    gen = torch.Generator().manual_seed(rows)
    randn = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    pd = torch.float64 if dtype == torch.float64 else torch.float32
    v = {"x": randn(rows, m.irreps.dim), "y": randn(rows, m.irreps.dim), "g": randn(rows, channels), "s": (0.5 + 0.1 * randn(channels)).to(pd),
         "w": (1 + 0.1 * randn(channels)).to(pd)}
    go, gn = randn(rows, m.irreps.dim), randn(rows, m.irreps.dim)
    d = {k: t.to(DEV).requires_grad_(True) for k, t in v.items()}
    outs = m(*d.values())
    grads = torch.autograd.grad(outs, tuple(d.values()), (go.to(DEV), gn.to(DEV)))
    ref = reference(blocks, True, m.eps, "sigmoid", False, v["x"], v["y"], v["g"], v["s"], v["w"], go, gn)
    alone = n(d["x"], d["w"])
    dx, dw = torch.autograd.grad(alone, (d["x"], d["w"]), gn.to(DEV))
    ref1 = reference(blocks, True, n.eps, None, False, v["x"], w=v["w"], gn=gn)
    for got, want, both in ((dict(zip(("out", "norm", *["d" + k for k in d]), (*outs, *grads))), ref, True), ({"norm": alone, "dx": dx, "dw": dw}, ref1, False)):
        for name, t in got.items():
            value, mag = want[name]
            err = (t.detach().cpu().double() - value).abs()
            tol = bound(name, mag, value, blocks, rows, dtype, both)
            assert bool((err <= tol).all()), (name, err.max().item(), (err / tol).max().item())
