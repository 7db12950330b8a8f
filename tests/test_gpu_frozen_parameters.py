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
