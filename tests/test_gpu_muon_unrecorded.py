"""What orthogonalize returns carries no gradient, and it says so where one would have been recorded."""
import warnings

import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu
fm = sub("enhancers.fused_muon")


def test_a_gradient_that_is_not_recorded_is_said(native):
    leaf = torch.randn(8, 8, device="cuda", requires_grad=True)
    for x in (leaf, leaf * 2):
        with pytest.warns(UserWarning, match="gradient"):
            out = fm.orthogonalize(x)
        assert not out.requires_grad and torch.equal(out, fm.orthogonalize(x.detach()))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        fm.orthogonalize(leaf.detach())
        with torch.no_grad():
            fm.orthogonalize(leaf)
        assert fm.orthogonalize(leaf.cpu()) is None               # (not the kernel's case: nothing was lost)
