"""Linear with its input kept in 8 bits (csrc/linear_fused.cu: linear_pack, linear_gw_codes) against float64 sums over the kept values, and a
whole block - norm, linear, channelwise product, linear, gate and residual - as a model runs it."""
import pytest
import torch

import cuequivariance_b200 as cb
from _norm_reference import blocks_of, join, kept, split

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _kept_rows(x, irreps, mul_ir):
    blocks = blocks_of(irreps)
    return join([kept(b, True) for b in split(x.double(), blocks, mul_ir)], mul_ir)


def _weight_gradient(m, x, cot, bounds, lin, lout):
    """(value, sum of magnitudes), paths between irreps that occur once on each side."""
    vals = torch.zeros(m.weight_classes, m.weight_numel, dtype=torch.float64)
    mags = vals.clone()
    ins = {str(ir): b for (_, ir), b in zip(m.irreps_in, split(x, blocks_of(m.irreps_in), lin is cb.mul_ir))}
    outs = {str(ir): b for (_, ir), b in zip(m.irreps_out, split(cot, blocks_of(m.irreps_out), lout is cb.mul_ir))}
    at = 0
    for mul, ir in m.irreps_in:
        if str(ir) not in outs:
            continue
        a, b = ins[str(ir)], outs[str(ir)]
        n = mul * b.shape[1]
        for k in range(m.weight_classes):
            s = slice(bounds[k], bounds[k + 1])
            vals[k, at : at + n] = (torch.einsum("zui,zvi->uv", a[s], b[s]) / mul**0.5).reshape(-1)
            mags[k, at : at + n] = (torch.einsum("zui,zvi->uv", a[s].abs(), b[s].abs()) / mul**0.5).reshape(-1)
        at += n
    return vals, mags


@pytest.mark.parametrize("s_in,s_out,rows,classes,lin,lout", [
    ("128x0e+128x1o+128x2e+128x3o", "128x0e+128x1o+128x2e+128x3o", 1, 1, "mul_ir", "mul_ir"),
    ("128x0e+128x1o+128x2e+128x3o", "128x0e+128x1o+128x2e+128x3o", 8021, 1, "mul_ir", "mul_ir"),
    ("32x0e+96x1o+64x2e+32x3o", "96x0e+32x1o+64x2e+128x3o", 421, 1, "ir_mul", "mul_ir"),
    ("96x0e+64x1o", "32x0e+96x1o", 37, 1, "mul_ir", "ir_mul"),
    ("64x0e+64x1o+64x2e+64x3o", "64x0e+64x1o+64x2e+64x3o", 911, 10, "ir_mul", "ir_mul"),
    ("4x0o+128x1o+64x3o", "64x0e+32x1o+32x3o", 3001, 3, "mul_ir", "mul_ir"),
    ("32x0e", "32x0e", 131, 64, "mul_ir", "mul_ir"),
])
def test_against_float64_sums(s_in, s_out, rows, classes, lin, lout):
    lin, lout = getattr(cb, lin), getattr(cb, lout)
    kw = dict(layout_in=lin, layout_out=lout, internal_weights=False, shared_weights=True, weight_classes=classes)
    m, full = cb.Linear(s_in, s_out, saved_activations="int8", **kw), cb.Linear(s_in, s_out, **kw)
    gen = torch.Generator().manual_seed(rows)
    x, w = torch.randn(rows, m.irreps_in.dim, generator=gen), torch.randn(classes, m.weight_numel, generator=gen)
    x *= torch.exp(torch.randn(rows, 1, generator=gen))
    if rows > 2:
        x[rows // 2] = 0.0
    cot = torch.randn(rows, m.irreps_out.dim, generator=gen)
    idx, bounds = None, (0, rows)
    if classes > 1:   # class 1 owns no row
        idx = torch.sort(torch.randint(0, classes, (rows,), generator=gen)).values
        idx[idx == 1] = 0
        bounds = torch.searchsorted(idx, torch.arange(classes + 1)).tolist()
        idx = idx.to(DEV)
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    out = m(xd, wd, idx)
    assert "FusedLinear8" in type(out.grad_fn).__name__
    gw, gx = torch.autograd.grad(out, (wd, xd), cot.to(DEV))
    if rows >= 256:   # the output and the input gradient do not know of it
        want = full(xd, wd, idx)
        assert torch.equal(out, want) and torch.equal(gx, torch.autograd.grad(want, xd, cot.to(DEV))[0])
    ref, mag = _weight_gradient(m, _kept_rows(x, m.irreps_in, lin is cb.mul_ir), cot.double(), bounds, lin, lout)
    # a product: 2^-21 (rounding of g's lower half; the codes are exact); sums that need not round to nearest: 2^-23 of the magnitude per
    # addition - 4 * 128 / 3 per accumulator, four accumulators and one addition per thread block
    err = (gw.cpu().double() - ref).abs()
    assert bool((err <= (2.0**-21 + (200 + rows // 64) * 2.0**-23) * mag + 1e-30).all()), err.max().item()
    assert torch.equal(torch.autograd.grad(m(xd, wd, idx), wd, cot.to(DEV))[0], gw)


def test_values_that_are_not_finite():
    """The gradient of the weights that met an infinity is not finite; other irreps' are."""
    m = cb.Linear("32x0e+32x1o", "32x0e+32x1o", layout=cb.mul_ir, saved_activations="int8").to(DEV)
    x = torch.randn(70, 128, device=DEV)
    x[69, 40] = float("inf")
    m(x).nan_to_num().sum().backward()
    gw = m.weight.grad[0]
    assert torch.isnan(gw[1024:]).all() and torch.isfinite(gw[:1024]).all()


def test_no_rows_and_no_gradient():
    m = cb.Linear("32x0e+32x1o", "32x0e+32x1o", layout=cb.mul_ir, saved_activations="int8").to(DEV)
    x = torch.zeros(0, 128, device=DEV, requires_grad=True)
    out = m(x)
    out.sum().backward()
    assert out.shape == x.grad.shape == (0, 128) and torch.equal(m.weight.grad, torch.zeros_like(m.weight))
    with torch.no_grad():
        assert m(torch.ones(3, 128, device=DEV)).grad_fn is None
    m.weight.requires_grad_(False)          # nothing is kept where no weight gradient is wanted
    out = m(torch.ones(3, 128, device=DEV, requires_grad=True))
    assert all(t is None or t.dtype == torch.float32 for t in out.grad_fn.saved_tensors)


def test_refusals():
    kw = dict(layout=cb.mul_ir, internal_weights=False, shared_weights=True, saved_activations="int8")
    m, c = cb.Linear("32x0e", "32x0e", **kw), cb.Linear("32x0e", "32x0e", weight_classes=3, **kw)
    x, w = torch.randn(9, 32, device=DEV), torch.randn(1, 1024, device=DEV)
    for bad in ((x.double(), w.double()), (x.bfloat16(), w), (x[0], w), (x, w.expand(9, -1)), (x[:, :31], w)):
        with pytest.raises(ValueError, match="int8"):
            m(*bad)
    with pytest.raises(ValueError, match="non-sorted"):
        c(x, w.repeat(3, 1), torch.tensor([0, 2, 1, 0, 0, 0, 0, 0, 0], device=DEV))
    with pytest.raises(ValueError, match="weight_indices"):
        c(x, w.repeat(3, 1), torch.zeros(8, dtype=torch.int64, device=DEV))


def _model(saved, dtype):
    s = "32x0e+32x1o+32x2e"
    kw = dict(layout=cb.mul_ir, internal_weights=False)
    lin = dict(shared_weights=True, **kw)
    eight = dict(saved_activations=saved)
    tp = cb.ChannelWiseTensorProduct(s, "0e+1o+2e", ["0e", "1o", "2e"], shared_weights=False, **kw)
    return {"norm": cb.IrrepsNorm(s, **eight, **kw), "up": cb.Linear(s, s, **lin, **(eight if dtype == torch.float32 else {})), "tp": tp,
            "down": cb.Linear(tp.irreps_out.simplify(), s, **lin), "gates": cb.Linear("32x0e", "96x0e", **lin, **(eight if dtype == torch.float32 else {})),
            "residual": cb.GatedResidual(s, norm_output=True, **eight, **kw)}


def _block(m, v, edges):
    snd, rcv, n = edges
    h = m["up"](m["norm"](v["x"], v["nw"]), v["uw"])
    msg = m["tp"](h, v["sh"], v["tw"], indices_1=snd, indices_out=rcv, size_out=n)
    y = m["down"](msg, v["dw"])
    return m["residual"](v["x"], y, m["gates"](y[:, :32], v["gw"]), v["s"], v["w"])


def test_a_block_as_a_model_runs_it():
    """float32 in full against the same block in float64; kept in 8 bits: the same outputs bit for bit, and gradients off by what the kept values
    are.  Those are off by at most 1/127 of a block's largest magnitude, which is at most 5.5 times its root mean square here (160 values;
    asserted), i.e. by 4.4 % of it, uniformly: 2.5 % in the mean square.  A gradient meets up to five of them in a row: 13 %."""
    nodes, per = 300, 8
    gen = torch.Generator().manual_seed(0)
    m = _model("full", torch.float64)
    rcv = torch.arange(nodes).repeat_interleave(per)
    snd = torch.randint(0, nodes, (nodes * per,), generator=gen)
    randn = lambda *s, scale=1.0: torch.randn(*s, generator=gen, dtype=torch.float64) * scale  # noqa: E731
    v = {"x": randn(nodes, 288), "nw": 1 + randn(96, scale=0.2), "uw": randn(1, m["up"].weight_numel), "sh": randn(nodes * per, 9),
         "tw": randn(nodes * per, m["tp"].weight_numel), "dw": randn(1, m["down"].weight_numel), "gw": randn(1, m["gates"].weight_numel),
         "s": 0.5 + randn(96, scale=0.1), "w": 1 + randn(96, scale=0.2)}
    cots = [randn(nodes, 288) for _ in range(2)]
    results = {}
    for name, saved, dtype in (("f64", "full", torch.float64), ("f32", "full", torch.float32), ("int8", "int8", torch.float32)):
        d = {k: t.to(DEV, dtype).requires_grad_(True) for k, t in v.items()}
        outs = _block(_model(saved, dtype), d, (snd.to(DEV).int(), rcv.to(DEV).int(), nodes))
        grads = torch.autograd.grad(outs, tuple(d.values()), [c.to(DEV, dtype) for c in cots])
        results[name] = ([o.detach().double() for o in outs], dict(zip(d, (g.double() for g in grads))))
    for b in split(results["f64"][0][0].cpu(), blocks_of(m["norm"].irreps), True):
        assert (b.abs().amax((1, 2)) <= 5.5 * b.pow(2).mean((1, 2)).sqrt()).all()
    for a, b in zip(results["f32"][0], results["f64"][0]):
        assert ((a - b).norm() <= 1e-5 * b.norm())
    for a, b in zip(results["int8"][0], results["f32"][0]):
        assert torch.equal(a, b)
    for k, want in results["f64"][1].items():
        assert (results["f32"][1][k] - want).norm() <= 2e-5 * want.norm(), k
        assert (results["int8"][1][k] - want).norm() <= 0.13 * want.norm(), k
