"""residual_norm, rms_norm and gated_dense in a captured graph, forward and backward, two graphs side by side, and under more of
autograd than a plain backward pass."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

fn, fd = sub("enhancers.fused_norm"), sub("enhancers.fused_dense")
forward_ad = torch.autograd.forward_ad


class Block:
    """A gated sub-layer's training pass on tensors of its own."""

    def __init__(self, rows, k, n, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.x, self.dr, self.dy = (self.rnd(rows, k) for _ in range(3))
        self.params = [t.requires_grad_() for t in (self.rnd(k), self.rnd(2 * n, k) / 16, self.rnd(2 * n), self.rnd(k, n) / 16, self.rnd(k),
                                                    self.rnd(k), self.rnd(k), self.rnd(k))]
        self.leaves = [self.x.requires_grad_(), *self.params]

    def rnd(self, *s):
        return torch.randn(*s, generator=self.g, device="cuda").to(torch.bfloat16)

    def renew(self):
        with torch.no_grad():
            for t in (self.x, self.dr, self.dy):
                t.copy_(self.rnd(*t.shape))

    def step(self):
        p = self.params
        h = fd.dense(fd.gated_dense(fn.rms_norm(self.x, p[0]), p[1], p[2]), p[3])
        out = fn.residual_norm(self.x, h, gate=p[4], post_weight=p[5], weight=p[6], bias=p[7], post="layer")
        return (*out, *torch.autograd.grad(out, self.leaves, (self.dr, self.dy)))


@pytest.mark.parametrize("rows,k,n", [(64, 2048, 512), (515, 333, 129)])
def test_training_passes_in_two_graphs(native, rows, k, n):
    blocks = [Block(rows, k, n, rows + i) for i in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for b in blocks:
            for _ in range(2):
                b.step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for b in blocks:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(b.step())
    sides = [torch.cuda.Stream() for _ in blocks]
    for i in range(5):
        for b in blocks:
            b.renew()
        torch.cuda.synchronize()
        for side, graph in zip(sides, graphs):                     # at the same time
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for b, out in zip(blocks, outs):
            got = [t.detach().clone() for t in out]
            assert all(torch.equal(p, q) for p, q in zip(got, b.step())), i


def norm():
    x, h = (torch.randn(12, 64, device="cuda").requires_grad_() for _ in range(2))
    return fn.residual_norm(x, h, post="rms")[1], (x, h)


def linear():
    x = torch.randn(12, 64, device="cuda").to(torch.bfloat16).requires_grad_()
    w = torch.randn(96, 64, device="cuda").to(torch.bfloat16).requires_grad_()
    return fd.gated_dense(x, w), (x, w)


@pytest.mark.parametrize("make", [norm, linear])
def test_gradients_that_are_more_than_memory(native, make):
    y, leaves = make()
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, -dy, retain_graph=True)
    got = torch.autograd.grad(y, leaves, torch._neg_view(dy), retain_graph=True)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.randn_like(y), torch.randn_like(y))
        with pytest.raises(RuntimeError, match="gradient"):
            torch.autograd.grad(y, leaves, dual, retain_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, torch.randn(3, *y.shape, device="cuda").to(y.dtype), is_grads_batched=True)


def test_inputs_that_are_more_than_memory(native):
    x = torch.randn(8, 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(32, 64, device="cuda").to(torch.bfloat16)
    seen = []
    torch.jit.trace(lambda t: seen.append((fn.residual_norm(t, t), fn.rms_norm(t), fd.gated_dense(t, w))) or t * 1, (x,),
                    check_trace=False)
    assert seen == [(None, None, None)]
    assert fn.rms_norm(torch._neg_view(x)) is None and fn.residual_norm(x, torch._neg_view(x)) is None
    with forward_ad.dual_level():
        assert fd.gated_dense(forward_ad.make_dual(x, x), w) is None and fn.rms_norm(forward_ad.make_dual(x, x)) is None
    torch.func.vmap(lambda t: seen.append(fn.rms_norm(t)) or t)(x[None])
    assert seen[-1] is None
