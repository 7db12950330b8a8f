"""The norm in front of a block and the norm, gate and residual behind it (csrc/norm_kernels.cuh) against float64 sums: every type,
layout and gate, blocks that do not start on 16-byte boundaries, one channel, hundreds, more values than a thread block holds
channels for, rows from one to many per thread block, empty rows, rows that lie apart or are all the same one, infinities and NaN."""
import pytest
import torch

import cuequivariance_b200 as cb
from _norm_reference import blocks_of, bound, kept, reference, split, step_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
L3 = "128x0e+128x1o+128x2e+128x3o"


def _features(rows, dim, dtype, gen):
    t = torch.randn(rows, dim, generator=gen, dtype=torch.float64) * torch.exp(0.5 * torch.randn(rows, 1, generator=gen, dtype=torch.float64))
    if rows > 2:
        t[rows // 2] = 0.0                                # a row whose mask left nothing
    return t.to(dtype)


def _inputs(irreps, rows, dtype, gate, norm_output, seed, param_dtype=None):
    gen = torch.Generator().manual_seed(seed)
    blocks = blocks_of(irreps)
    dim, channels = sum(m * d for m, d in blocks), sum(m for m, _ in blocks)
    pd = param_dtype or (F64 if dtype == F64 else F32)
    v = {"x": _features(rows, dim, dtype, gen), "y": _features(rows, dim, dtype, gen)}
    if gate:
        v["g"] = (1.5 * torch.randn(rows, channels, generator=gen, dtype=torch.float64)).to(dtype)
    v["s"] = (0.5 + 0.1 * torch.randn(channels, generator=gen, dtype=torch.float64)).to(pd)
    if norm_output:
        v["w"] = (1 + 0.2 * torch.randn(channels, generator=gen, dtype=torch.float64)).to(pd)
    cots = [torch.randn(rows, dim, generator=gen, dtype=torch.float64).to(dtype) for _ in range(1 + norm_output)]
    return v, cots


def _compare(got, ref, blocks, rows, dtype, both, param_dtype=None):
    for name, t in got.items():
        value, mag = ref[name]
        tol = bound(name, mag, value, blocks, rows, dtype, both)
        if name in ("ds", "dw") and param_dtype in (BF16, F16):
            tol = tol + torch.finfo(param_dtype).eps / 2 * value.abs()
        assert t.shape == value.shape, name
        t = t.detach().cpu().double()
        # Rounding to fp16 takes everything from 65504 + 16 = 65520 on (the middle between the largest number, 2047 * 2^5, and the
        # next at that spacing, 2048 * 2^5 = 65536) to infinity.  The empty row reaches that: with eps = 1e-5 both of its r are 316.2, and
        # dy = s act(g) w gn r^2 = 0.5 * 0.9 * 1.2 * 1.3 * 1e5 = 70200 for factors as drawn here.
        over = torch.isinf(t) & (dtype == F16) & (value.abs() + tol >= 65520.0) & (torch.sign(t) == torch.sign(value))
        err = torch.where(over, 0.0, (t - value).abs())
        assert bool((err <= tol).all()), (name, err.max().item(), (err / tol).max().item())


def _norm(irreps, rows, dtype, layout, saved="full", seed=0, param_dtype=None):
    m = cb.IrrepsNorm(irreps, layout=layout, internal_weights=False, saved_activations=saved)
    v, cots = _inputs(m.irreps, rows, dtype, None, True, seed, param_dtype)
    x, w = v["x"].to(DEV).requires_grad_(True), v["w"].to(DEV).requires_grad_(True)
    out = m(x, w)
    dx, dw = torch.autograd.grad(out, (x, w), cots[1].to(DEV))
    blocks = blocks_of(m.irreps)
    ref = reference(blocks, layout is cb.mul_ir, m.eps, None, saved == "int8", v["x"], w=v["w"], gn=cots[1])
    with torch.no_grad():
        assert torch.equal(m(x, w), out)
    _compare({"norm": out, "dx": dx, "dw": dw}, ref, blocks, rows, dtype, False, param_dtype)


def _residual(irreps, rows, dtype, layout, gate, norm_output, saved="full", seed=0, param_dtype=None):
    m = cb.GatedResidual(irreps, layout=layout, gate=gate, norm_output=norm_output, internal_weights=False, saved_activations=saved)
    v, cots = _inputs(m.irreps, rows, dtype, gate, norm_output, seed, param_dtype)
    d = {k: t.to(DEV).requires_grad_(True) for k, t in v.items()}
    call = lambda: m(d["x"], d["y"], d.get("g"), d["s"], d.get("w"))  # noqa: E731
    out = call()
    outs = out if norm_output else (out,)
    grads = dict(zip(["d" + k for k in d], torch.autograd.grad(outs, tuple(d.values()), [c.to(DEV) for c in cots])))
    blocks = blocks_of(m.irreps)
    ref = reference(blocks, layout is cb.mul_ir, m.eps, gate, saved == "int8", v["x"], v["y"], v.get("g"), v["s"], v.get("w"), cots[0],
                    cots[1] if norm_output else None)
    with torch.no_grad():
        again = call()
        assert all(torch.equal(a, b) for a, b in zip(again if norm_output else (again,), outs))
    _compare({**dict(zip(("out", "norm"), outs)), **grads}, ref, blocks, rows, dtype, norm_output, param_dtype)


SHAPES = [
    (L3, 1), (L3, 37), (L3, 2003),
    ("1x0e", 5), ("1x0e+1x1o+1x2e", 9), ("5x0e+3x1o+2x2e", 301), ("33x0e+7x1o", 64),
    ("32x0e+32x1o+32x2e+32x3o", 1511), ("64x0e+64x1o", 4099), ("64x0e+32x0o+32x1o", 6), ("96x0e+64x2e+32x3o", 131), ("129x0e+97x1o", 47),
    ("2x0e+8x1o+16x2e+12x3o", 203), ("48x0e+36x1o+68x2e+100x3o", 77), ("3x0e+64x1o+128x2e", 41), ("20x0e+24x1o", 2), ("66x0e+34x1o", 35), ("96x0o+48x1e+16x2e+4x4e", 333),
    ("300x0e+260x3o", 55), ("2048x0e", 70), ("16x0e+16x0o+16x1e+16x1o+8x5o", 129),
]


@pytest.mark.parametrize("layout", [cb.mul_ir, cb.ir_mul], ids=["mul_ir", "ir_mul"])
@pytest.mark.parametrize("irreps,rows", SHAPES)
def test_norm_float32(irreps, rows, layout):
    _norm(irreps, rows, F32, layout)


@pytest.mark.parametrize("dtype", [F64, BF16, F16], ids=["f64", "bf16", "f16"])
@pytest.mark.parametrize("irreps,rows", [(L3, 200), ("5x0e+3x1o+2x2e", 77), ("64x0e+64x1o", 1025), ("1x0e+9x1o", 3)])
def test_norm_types(irreps, rows, dtype):
    _norm(irreps, rows, dtype, cb.mul_ir)
    _norm(irreps, rows, dtype, cb.ir_mul, seed=1)


@pytest.mark.parametrize("norm_output", [False, True], ids=["residual", "residual_norm"])
@pytest.mark.parametrize("gate", [None, "sigmoid", "silu"])
@pytest.mark.parametrize("irreps,rows", SHAPES)
def test_residual_float32(irreps, rows, gate, norm_output):
    _residual(irreps, rows, F32, cb.mul_ir if rows % 2 else cb.ir_mul, gate, norm_output)


@pytest.mark.parametrize("norm_output", [False, True], ids=["residual", "residual_norm"])
@pytest.mark.parametrize("dtype", [F64, BF16, F16], ids=["f64", "bf16", "f16"])
@pytest.mark.parametrize("irreps,rows,gate", [(L3, 200, "sigmoid"), ("5x0e+3x1o+2x2e", 77, "silu"), ("64x0e+64x1o", 1025, None), ("1x0e+9x1o", 3, "silu")])
def test_residual_types(irreps, rows, gate, dtype, norm_output):
    _residual(irreps, rows, dtype, cb.ir_mul if rows % 2 else cb.mul_ir, gate, norm_output)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("irreps,rows", [(L3, 150), ("5x0e+3x1o+2x2e", 77), ("64x0e+64x1o", 1025), ("1x0e+9x1o", 3)])
def test_kept_in_8_bits(irreps, rows, dtype):
    _norm(irreps, rows, dtype, cb.mul_ir, "int8")
    _residual(irreps, rows, dtype, cb.mul_ir, "sigmoid", False, "int8")
    _residual(irreps, rows, dtype, cb.ir_mul, None, False, "int8")
    _norm(irreps, rows, dtype, cb.ir_mul, "int8")


@pytest.mark.parametrize("irreps,rows,seed", [("16x0e+16x1o", 5, 0), ("5x0e+3x1o+2x2e", 7, 1)])
def test_residual_norm_in_8_bits(irreps, rows, seed):
    """The kept h is computed; where it lies well away from the middle between two codes, the code is that of float64."""
    m = cb.GatedResidual(irreps, norm_output=True)
    v, _ = _inputs(m.irreps, rows, F32, "silu", True, seed)
    h = reference(blocks_of(m.irreps), True, m.eps, "silu", False, v["x"], v["y"], v["g"], v["s"], v["w"])["out"][0]
    for b in split(h, blocks_of(m.irreps), True):
        part = (b / step_of(b)) % 1.0
        assert ((part - 0.5).abs() > 127 * 60 * 2.0**-24).all()
    _residual(irreps, rows, F32, cb.mul_ir, "silu", True, "int8", seed)


@pytest.mark.parametrize("irreps,rows", [("5x0e+3x1o+2x2e", 70001), ("48x0e+32x1o", 30011), ("64x0e+7x1o", 45003)])
def test_many_stages_per_warp(irreps, rows):
    """More rows than all warps of a GPU take at a time, the last stages incomplete; dense rows of even and odd length."""
    _norm(irreps, rows, F32, cb.mul_ir)
    _norm(irreps, rows, BF16, cb.ir_mul, "int8")
    _residual(irreps, rows, F32, cb.ir_mul, "silu", True)
    _residual(irreps, rows, F16, cb.mul_ir, "sigmoid", False)
    _residual(irreps, rows, F32, cb.mul_ir, None, False, "int8")


@pytest.mark.parametrize("param_dtype", [BF16, F16])
def test_parameters_of_16_bits(param_dtype):
    _norm("64x0e+32x1o", 300, F32, cb.mul_ir, param_dtype=param_dtype)
    _residual("64x0e+32x1o", 300, BF16 if param_dtype == BF16 else F16, cb.mul_ir, "sigmoid", True, param_dtype=param_dtype)


def test_rows_apart_and_shared():
    """Column slices of wider tensors, on and off 16-byte boundaries; one row for all; a transposed tensor."""
    m = cb.GatedResidual("32x0e+32x1o", norm_output=True, internal_weights=False)
    v, cots = _inputs(m.irreps, 61, F32, "sigmoid", True, 3)
    d = {k: t.to(DEV) for k, t in v.items()}
    cots = [c.to(DEV) for c in cots]

    def run(x, y, g):
        leaves = [t.requires_grad_(True) for t in (x, y, g)]
        outs = m(*leaves, d["s"], d["w"])
        return [*outs, *torch.autograd.grad(outs, leaves, cots)]

    want = run(d["x"].clone(), d["y"].clone(), d["g"].clone())
    for pad in (1, 4, 64):
        def wide(t):
            u = torch.full((t.shape[0], t.shape[1] + 2 * pad), float("nan"), device=DEV)  # noqa: B023
            u[:, pad:-pad] = t  # noqa: B023
            return u[:, pad:-pad].detach()  # noqa: B023

        for a, b in zip(run(wide(d["x"]), wide(d["y"]), wide(d["g"])), want):
            assert torch.equal(a, b)
    for a, b in zip(run(d["x"].t().contiguous().t().detach(), d["y"].clone(), d["g"].clone()), want):
        assert torch.equal(a, b)
    one = d["x"][:1].clone()
    a = run(one.expand(61, -1).detach(), d["y"].clone(), d["g"].clone())
    b = run(one.repeat(61, 1), d["y"].clone(), d["g"].clone())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_cotangents_that_are_missing_shared_or_apart():
    m = cb.GatedResidual("32x0e+32x1o", norm_output=True, internal_weights=False)
    for saved in ("full", "int8"):
        m = cb.GatedResidual("32x0e+32x1o", norm_output=True, internal_weights=False, saved_activations=saved)
        v, cots = _inputs(m.irreps, 40, F32, "silu", True, 4)
        d = {k: t.to(DEV).requires_grad_(True) for k, t in v.items()}
        leaves = tuple(d.values())
        go, gn = (c.to(DEV) for c in cots)
        call = lambda: m(*leaves)  # noqa: B023, E731
        zero = torch.zeros_like(go)
        only_norm = torch.autograd.grad(call()[1], leaves, gn)
        for a, b in zip(only_norm, torch.autograd.grad(call(), leaves, (zero, gn))):
            assert torch.allclose(a, b, rtol=1e-6, atol=1e-7)
        out, _ = call()
        only_out = torch.autograd.grad(out, leaves[:4], go)
        for a, b in zip(only_out, torch.autograd.grad(call(), leaves[:4], (go, zero))):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
        assert torch.autograd.grad(call()[0], leaves[4], go, allow_unused=True)[0] is None
        out, n = call()
        summed = torch.autograd.grad(out.sum() + n.sum(), leaves)       # cotangents are one number, expanded: the same calls
        for a, b in zip(summed, torch.autograd.grad(call(), leaves, (torch.ones_like(go), torch.ones_like(gn)))):
            assert torch.equal(a, b)


def test_gradients_against_differences():
    """Central differences in float64: step 1e-6, third derivatives of order one."""
    for norm_output, gate in ((False, "sigmoid"), (True, "silu"), (True, None)):
        m = cb.GatedResidual("3x0e+2x1o", gate=gate, norm_output=norm_output, internal_weights=False)
        v, cots = _inputs(m.irreps, 4, F64, gate, norm_output, 5)
        d = [t.to(DEV).requires_grad_(True) for t in v.values()]
        cots = [c.to(DEV) for c in cots]
        names = list(v)

        def value(ts):
            kw = dict(zip(names, ts))  # noqa: B023
            out = m(kw["x"], kw["y"], kw.get("g"), kw["s"], kw.get("w"))  # noqa: B023
            return sum((o * c).sum() for o, c in zip(out if norm_output else (out,), cots))  # noqa: B023

        grads = torch.autograd.grad(value(d), d)
        gen = torch.Generator().manual_seed(6)
        for k in range(len(d)):
            direction = torch.randn(d[k].shape, generator=gen, dtype=F64).to(DEV)
            if names[k] in ("x", "y"):
                direction[2] = 0          # the empty row: r(0) = eps^-1/2 makes its higher derivatives large
            with torch.no_grad():
                up = value([t + 1e-6 * direction if q == k else t for q, t in enumerate(d)])
                down = value([t - 1e-6 * direction if q == k else t for q, t in enumerate(d)])
            got = (grads[k] * direction).sum()
            assert abs((up - down) / 2e-6 - got) <= 1e-6 * (1 + abs(got)), names[k]


@pytest.mark.parametrize("irreps", ["7000x0e", "1200x0e+3000x1o+33x0o"])
def test_blocks_that_leave_room_for_one_stage(irreps):
    for layout in (cb.mul_ir, cb.ir_mul):
        _norm(irreps, 5, F32, layout)
        _residual(irreps, 5, BF16, layout, "sigmoid", True)
        _residual(irreps, 3, F32, layout, None, False, "int8")


def test_blocks_that_do_not_fit_are_refused():
    m = cb.GatedResidual("30000x0e", gate=None)
    with pytest.raises(RuntimeError, match="shared memory"):
        m.to(DEV)(torch.zeros(2, 30000, device=DEV), torch.zeros(2, 30000, device=DEV))


def test_second_derivatives_are_refused():
    m = cb.GatedResidual("32x0e+3x1o", norm_output=True).to(DEV)
    x, g = torch.randn(5, 41, device=DEV, requires_grad=True), torch.randn(5, 35, device=DEV)
    out, n = m(x, x, g)
    (gx,) = torch.autograd.grad(out.sum() + n.pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()


def test_no_rows():
    m = cb.GatedResidual("32x0e+32x1o", norm_output=True).to(DEV)
    x = torch.zeros(0, 128, device=DEV, requires_grad=True)
    out, n = m(x, x, torch.zeros(0, 64, device=DEV))
    (out.sum() + n.sum()).backward()
    assert out.shape == n.shape == x.grad.shape == (0, 128)
    assert torch.equal(m.scale.grad, torch.zeros(64, device=DEV)) and torch.equal(m.weight.grad, torch.zeros(64, device=DEV))


@pytest.mark.parametrize("saved", ["full", "int8"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_values_that_are_not_finite_stay_in_their_block(bad, saved):
    m = cb.IrrepsNorm("32x0e+32x1o", internal_weights=False, saved_activations=saved)
    gen = torch.Generator().manual_seed(7)
    x, w, go = torch.randn(50, 128, generator=gen), torch.ones(64), torch.randn(50, 128, generator=gen)
    x[11, 70] = bad
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    out = m(xd, wd)
    dx, dw = torch.autograd.grad(out, (xd, wd), go.to(DEV))
    hurt = torch.zeros(50, 128, dtype=torch.bool)
    hurt[11, 32:] = True
    assert not torch.isfinite(dx.cpu()[11, 32:]).any() and torch.isfinite(dx.cpu()[~hurt]).all() and torch.isfinite(out.cpu()[~hurt]).all()
    assert torch.isnan(out.cpu()[11, 70])                      # inf * 0 and NaN alike
    assert torch.isfinite(dw.cpu()[:32]).all()


def test_large_and_small_values_in_8_bits():
    """Magnitudes at the ends of float32 that the statistic still holds, and a block of subnormal numbers."""
    m = cb.IrrepsNorm("32x0e+32x1o+32x2e", internal_weights=False, saved_activations="int8", eps=1e-30)
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(6, 288, generator=gen)
    x[1] *= 1e17
    x[2] *= 1e-13
    x[3, 32:128] = torch.randn(96, generator=gen) * 1e-40
    x[4, :32] = 127.0 * torch.sign(x[4, :32])                  # the largest code, exactly
    x[5, :32] = 127.5
    w, go = torch.ones(96), torch.randn(6, 288, generator=gen)
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    out = m(xd, wd)
    dx, dw = torch.autograd.grad(out, (xd, wd), go.to(DEV))
    blocks = blocks_of(m.irreps)
    ref = reference(blocks, True, 1e-30, None, True, x, w=w, gn=go)
    _compare({"norm": out, "dx": dx, "dw": dw}, ref, blocks, 6, F32, False)
    for b, top in zip(split(kept(x.double(), False)[4:], blocks, True)[:1], (None,)):
        assert torch.equal(kept(b, True)[0], b[0]) and float(step_of(b)[1]) == 2.0


def test_repeatable_on_streams_and_in_graphs():
    """The same bits on every call, from another stream, and from a captured forward and backward pass that is replayed on new
    values; two graphs on one memory pool do not disturb one another."""
    m = cb.GatedResidual(L3, norm_output=True, internal_weights=False, saved_activations="int8")
    v, cots = _inputs(m.irreps, 500, F32, "sigmoid", True, 9)
    d = {k: t.to(DEV).requires_grad_(True) for k, t in v.items()}
    cots = [c.to(DEV) for c in cots]

    def step():
        outs = m(*d.values())
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, tuple(d.values()), cots)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        a = step()
    with torch.cuda.graph(second, pool=first.pool()):
        b = step()
    values = {k: t.detach().clone() for k, t in d.items()}
    with torch.no_grad():
        for k in d:
            d[k].mul_(0.5)
    half = [t.clone() for t in step()]
    for g, res in ((first, a), (second, b), (first, a)):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(res, half))
    with torch.no_grad():
        for k in d:
            d[k].copy_(values[k])
    second.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(b, want))


def test_bytes_kept_for_the_backward_pass():
    """float32 features in 8 bits: a quarter, statistics of 32 bytes per row and block on top."""
    x, y = (torch.randn(4096, 2048, device=DEV, requires_grad=True) for _ in range(2))
    g = torch.randn(4096, 512, device=DEV, requires_grad=True)
    m = cb.GatedResidual(L3, saved_activations="int8").to(DEV)
    out = m(x, y, g)
    held = sum(t.numel() * t.element_size() for t in out.grad_fn.saved_tensors if t is not None and t.dim() > 1)
    assert held <= 4096 * (2048 + 512 + 4 * 16)


def test_more_elements_than_32_bits_count():
    """1.1 million rows of 2,048 16-bit values: the last rows and the parameter's gradient of two rows far apart."""
    rows = 1_100_000
    m = cb.IrrepsNorm(L3, internal_weights=False)
    x = torch.zeros(rows, 2048, device=DEV, dtype=BF16)
    gen = torch.Generator().manual_seed(10)
    some = torch.randn(2, 2048, generator=gen).to(BF16)
    x[0], x[-1] = some[0].to(DEV), some[1].to(DEV)
    x.requires_grad_(True)
    w = torch.ones(512, device=DEV, requires_grad=True)
    out = m(x, w)
    dx, dw = torch.autograd.grad(out, (x, w), out.detach())
    few = some.to(DEV).requires_grad_(True)
    out2 = m(few, w)
    dx2, dw2 = torch.autograd.grad(out2, (few, w), out2.detach())
    assert torch.equal(out[0], out2[0]) and torch.equal(out[-1], out2[1])
    assert torch.equal(dx[0], dx2[0]) and torch.equal(dx[-1], dx2[1]) and not dx[1:-1].any() and not out[1:-1].any()
    assert torch.allclose(dw, dw2, rtol=1e-6)
