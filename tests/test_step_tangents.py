"""What the optimizer steps ask about forward mode (CPU only)."""
import torch

from conftest import sub

ops = sub("enhancers.operands")
forward_ad = torch.autograd.forward_ad


def test_which_tensors_carry_a_tangent():
    x, y = torch.randn(3, 4), torch.randn(5)
    assert not ops.duals([x, y]) and not ops.duals([])
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert ops.duals([y, dual]) and ops.duals(iter([dual])) and ops.duals([dual * 2])
        assert not ops.duals([x, y, forward_ad.unpack_dual(dual).primal])
    assert not ops.duals([x])
