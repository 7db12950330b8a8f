"""Gradients of parameters where only a few rows have a cotangent: the last ones, in incomplete stages, and the first.  The others add exact
zeros, so that a row left out, or counted twice, is much of the gradient whatever the number of rows."""
import pytest
import torch

import cuequivariance_b200 as cb
from _norm_reference import blocks_of, reference
from test_gpu_norm_16_bits import U, bounds

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("irreps,rows", [("5x0e+3x1o+2x2e", 70001), ("48x0e+32x1o", 30011), ("64x0e+7x1o", 45003), ("16x0e+1x1o", 20007), ("1x0e", 100003),
                                         ("128x0e+128x1o+128x2e+128x3o", 4099), ("200x0e+65x1o", 9001)])
@pytest.mark.parametrize("dtype,saved", [(F32, "full"), (F32, "int8"), (BF16, "full"), (F16, "int8")])
def test_few_rows_of_many(irreps, rows, dtype, saved):
    blocks = blocks_of(cb.Irreps(irreps))
    dim, channels = sum(m * d for m, d in blocks), sum(m for m, _ in blocks)
    gen = torch.Generator().manual_seed(rows)
    randn = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    x, y, g = randn(rows, dim), randn(rows, dim), randn(rows, channels).clamp(-7, 7)
    s, w = 0.5 + 0.1 * torch.randn(channels, generator=gen), 1 + 0.2 * torch.randn(channels, generator=gen)
    modules = {"norm": cb.IrrepsNorm(irreps, internal_weights=False, saved_activations=saved),
               "residual": cb.GatedResidual(irreps, internal_weights=False, saved_activations=saved)}
    if saved == "full":       # the code of a computed sum may be either neighbour
        modules["both"] = cb.GatedResidual(irreps, norm_output=True, internal_weights=False)
    on = {k: t.to(DEV) for k, t in {"x": x, "y": y, "g": g, "s": s, "w": w}.items()}
    for k in ("s", "w"):
        on[k].requires_grad_(True)
    for name, m in modules.items():
        outs = {"norm": lambda: (m(on["x"], on["w"]),), "residual": lambda: (m(on["x"], on["y"], on["g"], on["s"]),),  # noqa: B023
                "both": lambda: m(on["x"], on["y"], on["g"], on["s"], on["w"])}[name]()
        leaves = {"norm": ["w"], "residual": ["s"], "both": ["s", "w"]}[name]
        for few in (slice(rows - 1, rows), slice(rows - 7, rows), slice(rows - 40, rows), slice(0, 3)):
            go, gn = torch.zeros(rows, dim, dtype=dtype), torch.zeros(rows, dim, dtype=dtype)
            go[few], gn[few] = randn(go[few].shape[0], dim), randn(go[few].shape[0], dim)
            cots = {"norm": [gn], "residual": [go], "both": [go, gn]}[name]
            got = torch.autograd.grad(outs, [on[k] for k in leaves], [c.to(DEV) for c in cots], retain_graph=True)
            c = lambda t: None if t is None else t[few]  # noqa: B023, E731
            branch = name != "norm"
            ref = reference(blocks, True, m.eps, "sigmoid" if branch else None, saved == "int8", x[few], c(y if branch else None), c(g if branch else None),
                            s if branch else None, w if name != "residual" else None, c(go if branch else None), c(gn if name != "residual" else None))
            units = bounds(blocks, go[few].shape[0], True)
            for k, t in zip(leaves, got):
                value, mag = ref["d" + k]
                err = (t.cpu().double() - value).abs()
                assert bool((err <= units["d" + k] * U * mag + 1e-37).all()), (name, few, k, (err / (units["d" + k] * U * mag + 1e-37)).max().item())
