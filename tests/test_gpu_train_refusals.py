"""Arguments of the training-step operators that fit together but are no kernel's case, or whose result is empty."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

fn, fd = sub("enhancers.fused_norm"), sub("enhancers.fused_dense")


def test_layer_norm_parameters_of_two_types(native):
    x = torch.randn(6, 32, device="cuda").to(torch.bfloat16)
    w, b = torch.randn(32, device="cuda"), torch.randn(32, device="cuda")
    assert fn.layer_norm(x, w.to(torch.bfloat16), b) is None and fn.layer_norm(x, w, b.to(torch.bfloat16)) is None
    assert fn.layer_norm(x, w, b) is not None
    with pytest.raises(ValueError, match="differ"):
        fn.layer_norm(x, w, b[None].expand(2, 32))


@pytest.mark.parametrize("grad", [False, True])
def test_dense_without_outputs(native, grad):
    x = torch.randn(2, 5, 64, device="cuda").to(torch.bfloat16).requires_grad_(grad)
    w = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    r = torch.empty(2, 5, 0, device="cuda", dtype=torch.bfloat16)
    y = fd.dense(x, w, residual=r)
    assert y.shape == (2, 5, 0) and y.dtype == torch.bfloat16
    if grad:
        (gx,) = torch.autograd.grad(y.sum(), x)
        assert gx.shape == x.shape and float(gx.abs().sum()) == 0.0
