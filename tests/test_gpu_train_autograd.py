"""The training-step operators under more of autograd than a plain backward pass: incoming gradients that are more than
memory, and tracing. Whatever the kernels cannot read is refused; nothing is answered wrongly in silence."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

fn, fd = sub("enhancers.fused_norm"), sub("enhancers.fused_dense")
forward_ad = torch.autograd.forward_ad


def norm():
    x = torch.randn(12, 64, device="cuda").requires_grad_()
    w = torch.randn(64, device="cuda").requires_grad_()
    return fn.layer_norm(x, w), (x, w)


def linear():
    x = torch.randn(12, 64, device="cuda").to(torch.bfloat16).requires_grad_()
    w = torch.randn(48, 64, device="cuda").to(torch.bfloat16).requires_grad_()
    return fd.dense(x, w, act="silu"), (x, w)


@pytest.mark.parametrize("make", [norm, linear])
def test_negative_views_as_gradients(native, make):
    # a view whose values are its memory's negated: the same gradients as its copy's
    y, leaves = make()
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, -dy, retain_graph=True)
    got = torch.autograd.grad(y, leaves, torch._neg_view(dy))
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("make", [norm, linear])
def test_gradients_with_a_tangent_are_refused(native, make):
    # forward over reverse: the tangent of dy belongs into the result, and the kernels read the values alone
    y, leaves = make()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.randn_like(y), torch.randn_like(y))
        with pytest.raises(RuntimeError, match="gradient"):
            torch.autograd.grad(y, leaves, dual, retain_graph=True)
        got = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)       # a plain one beside it
    assert all(torch.equal(g, w) for g, w in zip(got, torch.autograd.grad(y, leaves, torch.ones_like(y))))


@pytest.mark.parametrize("make", [norm, linear])
def test_batches_of_gradients_are_refused(native, make):
    y, leaves = make()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, torch.randn(3, *y.shape, device="cuda").to(y.dtype), is_grads_batched=True)


def falling_back(x, w):
    """What a caller does with None."""
    y = fn.layer_norm(x, w)
    return torch.nn.functional.layer_norm(x, (64,), w) if y is None else y


@pytest.mark.parametrize("grad", [False, True])
def test_traces_record_the_fallback(native, grad):
    # a kernel launched through ctypes is no operation of the trace: it would hold the empty outputs alone
    x = torch.randn(12, 64, device="cuda")
    w = torch.randn(64, device="cuda").requires_grad_(grad)
    traced = torch.jit.trace(falling_back, (x, w), check_trace=False)
    z = torch.randn(12, 64, device="cuda")
    # (12 rows of 64 float32 values in either order of summation: 2^-18 of values below 100)
    assert float((traced(z, w) - falling_back(z, w)).abs().max()) < 1e-3
    linear = lambda x: fd.dense(x, x)                                                          # noqa: E731
    seen = []
    torch.jit.trace(lambda x: seen.append(linear(x)) or x * 1, (torch.randn(8, 64, device="cuda").bfloat16(),),
                    check_trace=False)
    assert seen == [None]


def test_a_trace_takes_no_optimizer_step(native):
    fa = sub("enhancers.fused_adamw")
    p, g = torch.zeros(300, device="cuda"), torch.ones(300, device="cuda")
    state = fa.adamw_state([p])

    def step(x):
        with pytest.raises(ValueError, match="trace"):
            fa.adamw_step([p], [g], state, 1)
        return x * 2
    torch.jit.trace(step, (g,), check_trace=False)
    assert float(p.abs().sum()) == 0.0
