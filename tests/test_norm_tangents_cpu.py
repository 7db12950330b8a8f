"""Forward-mode derivatives of the norm modules raise; they do not read as zero (no GPU: the launches are stood in for)."""
import pytest
import torch
from torch.autograd import forward_ad

from cuequivariance_b200.operations import norm


class _Block:
    mode, int8 = norm._lib.NORM_ALONE, False

    def forward(self, keep, x, y, g, s, w):
        return None, torch.empty_like(x), None, x.new_empty(1) if keep else None

    def kept(self, x, y, g, out, codes):
        return y, g, x


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("of", ["x", "weight"])
def test_a_tangent_is_not_lost(of, grad_mode):
    x, w = torch.randn(3, 16), torch.ones(8)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        norm._run(_Block(), x, None, None, None, w)                # none: as ever
        if of == "x":
            x = forward_ad.make_dual(x, torch.randn(3, 16))
        else:
            w = forward_ad.make_dual(w, torch.randn(8))
        with pytest.raises(RuntimeError, match="forward mode|jvp"):
            norm._run(_Block(), x, None, None, None, w)
    assert norm._run(_Block(), torch.randn(3, 16), None, None, None, torch.ones(8))[0].grad_fn is None
