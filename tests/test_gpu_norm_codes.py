"""The gated residual with the next norm, activations in 8 bits: the codes that the forward pass keeps - those of update and gates exactly, those
of the computed sum to half a step and what it is off - and the gradients, which are those of the kept values, in every type."""
import pytest
import torch

import cuequivariance_b200 as cb
from _norm_reference import act, blocks_of, join, kept, split, step_of
from test_gpu_norm_16_bits import U, bounds

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
pad16 = lambda n: (n + 15) // 16 * 16  # noqa: E731


def _decode(codes, stats, blocks, mul_ir, gated):
    """[(y, gates, h)] per block, from rows of codes and the steps in the statistics."""
    codes, stats, at, res = codes.cpu().double(), stats.cpu().double(), 0, [[None, None, None] for _ in blocks]
    parts = [(0, 2, lambda m, d: m * d)] + ([(1, 3, lambda m, d: m)] if gated else []) + [(2, 4, lambda m, d: m * d)]
    for which, step, width in parts:
        for k, (m, d) in enumerate(blocks):
            n = width(m, d)
            v = codes[:, at : at + n] * stats[:, k, step : step + 1]
            res[k][which] = v if which == 1 else split(v, [(m, d)], mul_ir)[0]
            at += pad16(n)
    assert at == codes.shape[1]
    return res


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", [cb.mul_ir, cb.ir_mul], ids=["mul_ir", "ir_mul"])
@pytest.mark.parametrize("irreps,rows,gate", [
    ("128x0e+128x1o+128x2e+128x3o", 37, "sigmoid"), ("64x0e+64x1o", 1025, "silu"), ("5x0e+3x1o+2x2e", 77, "silu"), ("16x0e+16x1o", 1, "sigmoid"),
    ("33x0e+7x1o", 64, None), ("200x0e+130x1o+9x4e", 19, "sigmoid"),
])
def test_kept_values_and_their_gradients(irreps, rows, gate, layout, dtype):
    m = cb.GatedResidual(irreps, layout=layout, gate=gate, norm_output=True, internal_weights=False, saved_activations="int8")
    blocks, mul_ir, channels = blocks_of(m.irreps), layout is cb.mul_ir, m.irreps.num_irreps
    gen = torch.Generator().manual_seed(rows)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    v = {"x": randn(rows, m.irreps.dim).to(dtype), "y": randn(rows, m.irreps.dim).to(dtype)}
    if gate:
        v["g"] = randn(rows, channels).clamp(-7, 7).to(dtype)
    v["s"], v["w"] = 0.5 + 0.1 * randn(channels), 1 + 0.2 * randn(channels)
    go, gn = randn(rows, m.irreps.dim).to(dtype), randn(rows, m.irreps.dim).to(dtype)
    d = {k: t.to(DEV).requires_grad_(True) for k, t in v.items()}
    outs = m(d["x"], d["y"], d.get("g"), d["s"], d["w"])
    codes, stats = outs[0].grad_fn.saved_tensors[3:5]
    grads = torch.autograd.grad(outs, tuple(d.values()), (go.to(DEV), gn.to(DEV)))
    units, res = bounds(blocks, rows, gate), {}
    decoded = _decode(codes, stats, blocks, mul_ir, gate is not None)
    sp = lambda t: split(t.double(), blocks, mul_ir)  # noqa: E731
    ch = lambda t: t.double().split([q for q, _ in blocks], dim=-1)  # noqa: E731
    gates = ch(v["g"]) if gate else [torch.zeros(rows, q, dtype=torch.float64) for q, _ in blocks]
    for (mul, dim), xb, yb, gb, sb, wb, ob, nb, (yk, gk, hk) in zip(blocks, sp(v["x"]), sp(v["y"]), gates, ch(v["s"]), ch(v["w"]), sp(go), sp(gn), decoded):
        n, sc, wc = mul * dim, sb[None, :, None], wb[None, :, None]
        rms = lambda t: ((t * t).flatten(1).mean(1) + m.eps).rsqrt().reshape(-1, 1, 1)  # noqa: B023, E731
        r = rms(yb)
        branch = sc * act(gb, gate)[0][:, :, None] * yb * r
        h, hmag = xb + branch, xb.abs() + branch.abs()
        rh = rms(h)
        assert torch.equal(yk, kept(yb, True))
        if gate:
            assert torch.equal(gk, kept(gb, True))
        # h: half a step; the step may be the next one where the largest magnitude lies at 127 steps
        off = units["dw"] * U * hmag
        assert bool(((hk - h).abs() <= step_of(h.abs() + off) / 2 + off).all())
        # as in the reference, of the kept values; h itself enters r(h) only
        rhe = rh**2 * (hmag * h.abs()).flatten(1).mean(1)[:, None, None]
        p, pm = (nb * hk).sum(2, keepdim=True), (nb * hk).abs().sum(2, keepdim=True) * (1 + rhe)
        mean, mm = (wc * p).sum(1, keepdim=True) / n, (wc * pm).abs().sum(1, keepdim=True) / n
        o = ob + rh * (wc * nb - hk * rh**2 * mean)
        om = ob.abs() + rh * ((wc * nb).abs() * (1 + rhe) + hk.abs() * rh**2 * mm * (1 + rhe))
        av, dv, dvm = (t[:, :, None] for t in act(gk if gate else gb, gate))
        q, qm = (o * yk).sum(2, keepdim=True), (om * yk.abs()).sum(2, keepdim=True)
        a = sc * av
        mean, mm = (a * q).sum(1, keepdim=True) / n, (a.abs() * qm).sum(1, keepdim=True) / n
        got = {"dw": ((rh * p).sum((0, 2)), (rh * pm).sum((0, 2))), "dx": (o, om), "ds": ((av * r * q).sum((0, 2)), (av.abs() * r * qm).sum((0, 2))),
               "dy": (r * (a * o - yk * r**2 * mean), r * (a.abs() * om + yk.abs() * r**2 * mm))}
        if gate:
            got["dg"] = ((sc * dv * r * q)[:, :, 0], (sc.abs() * dvm * r * qm)[:, :, 0])
        for k, pair in got.items():
            res.setdefault(k, []).append(pair)
    for name, t in zip(["d" + k for k in d], grads):
        whole = (lambda ts: join(ts, mul_ir)) if name in ("dx", "dy") else (lambda ts: torch.cat(ts, dim=-1))
        value, mag = whole([a for a, _ in res[name]]), whole([b for _, b in res[name]])
        tol = units[name] * U * mag + 1e-37
        if t.dtype != F32:
            tol = tol + torch.finfo(dtype).eps / 2 * value.abs() * (1 + 2.0**-7) + (2.0**-25 if dtype == F16 else 0)
        err = (t.cpu().double() - value).abs()
        assert bool((err <= tol).all()), (name, err.max().item(), (err / tol).max().item())
