"""Layers whose parameters are frozen (forces of a trained model): nothing is kept and nothing is launched for gradients that nobody
asked for."""
import pytest
import torch

import cuequivariance_b200 as cb

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("saved", ["full", "int8"])
@pytest.mark.parametrize("classes", [1, 3])
def test_linear_with_frozen_weights_keeps_no_rows(saved, classes):
    rows = 300
    m = cb.Linear("32x0e+64x1o", "64x0e+32x1o", layout=cb.mul_ir, weight_classes=classes, saved_activations=saved).to(DEV)
    idx = torch.arange(rows, device=DEV) * classes // rows if classes > 1 else None
    gen = torch.Generator().manual_seed(classes)
    x = torch.randn(rows, m.irreps_in.dim, generator=gen).to(DEV).requires_grad_(True)
    cot = torch.randn(rows, m.irreps_out.dim, generator=gen).to(DEV)
    out = m(x, weight_indices=idx)
    assert "FusedLinear" in type(out.grad_fn).__name__
    (want,) = torch.autograd.grad(out, x, cot)
    m.weight.requires_grad_(False)
    frozen = m(x, weight_indices=idx)
    held = [t for t in frozen.grad_fn.saved_tensors if t is not None]
    assert [t.shape for t in held] == [m.weight.shape]
    assert torch.equal(frozen, out) and torch.equal(torch.autograd.grad(frozen, x, cot)[0], want)


def test_linear_of_no_rows_with_frozen_weights():
    m = cb.Linear("32x0e+64x1o", "64x0e+32x1o", layout=cb.mul_ir, saved_activations="int8").to(DEV).requires_grad_(False)
    x = torch.zeros(0, m.irreps_in.dim, device=DEV, requires_grad=True)
    m(x).sum().backward()
    assert x.grad.shape == x.shape


@pytest.mark.parametrize("saved", ["full", "int8"])
@pytest.mark.parametrize("norm_output", [False, True])
@pytest.mark.parametrize("rows", [3, 5003])
@pytest.mark.parametrize("frozen", [("scale", "weight"), ("scale",), ("weight",)])
def test_norms_with_frozen_parameters(frozen, rows, norm_output, saved):
    """The same gradients, and memory for the wanted ones (with partial sums where a parameter's is among them) only."""
    m = cb.GatedResidual("32x0e+5x1o", norm_output=norm_output, saved_activations=saved).to(DEV)
    names = [n for n in ("scale", "weight") if getattr(m, n) is not None]
    gen = torch.Generator().manual_seed(rows)
    leaves = [torch.randn(rows, n, generator=gen).to(DEV).requires_grad_(True) for n in (47, 47, 37)]
    cots = [torch.randn(rows, 47, generator=gen).to(DEV) for _ in range(1 + norm_output)]

    def gradients():
        wanted = leaves + [getattr(m, n) for n in names if getattr(m, n).requires_grad]
        outs = m(*leaves)
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        grads = torch.autograd.grad(outs if norm_output else (outs,), wanted, cots)
        return grads, torch.cuda.memory_stats()["allocation.all.allocated"] - before

    want, _ = gradients()
    want = dict(zip(["x", "y", "g", *names], want))
    for n in frozen:
        if n in names:
            getattr(m, n).requires_grad_(False)
    got, allocations = gradients()
    left = ["x", "y", "g", *[n for n in names if n not in frozen]]
    for n, t in zip(left, got):
        assert torch.equal(t, want[n]), n
    # dx of the plain residual is the cotangent itself
    assert allocations == len(left) - (not norm_output) + (len(left) > 3)


def test_norm_with_a_frozen_weight():
    m = cb.IrrepsNorm("32x0e+5x1o").to(DEV)
    x, cot = torch.randn(41, 47, device=DEV, requires_grad=True), torch.randn(41, 47, device=DEV)
    (want,) = torch.autograd.grad(m(x), x, cot)
    m.requires_grad_(False)
    out = m(x)
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    (got,) = torch.autograd.grad(out, x, cot)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] - before == 1
    assert torch.equal(got, want)
    m.requires_grad_(True)                     # and the weight alone
    out = m(x.detach())
    (dw,) = torch.autograd.grad(out, m.weight, cot)
    assert torch.equal(dw, torch.autograd.grad(m(x), m.weight, cot)[0])
