"""The gated sub-layer's operators together -- norms, gated linear, linear, gated residual, both optimizers: the example runs, and one
of its passes agrees with the same sub-layer in float64 torch autograd on the CPU."""
import math

import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

ex = sub("examples.finetune_mlp")


@pytest.mark.parametrize("bits", [8, 32])
def test_example_runs(native, bits):
    r = ex.run(width=256, hidden=512, tokens=128, steps=6, bits=bits, gated=True)
    assert all(math.isfinite(v) for v in r.values()), r


def test_sub_layer_against_float64(native):
    # each bfloat16 rounding on the way is off by 2^-8 at most, and the longest chain has eight of them (normed input, gated
    # product, down's output; backward, the gradient behind the norm, between the products, [dg du], the one in front of the first
    # norm, the result): 8 * 2^-8 = 3.2 % of a gradient's norm if all were at their worst and in one direction
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g)                                              # noqa: E731
    up, down = (rnd(1024, 256) / 16).bfloat16(), (rnd(256, 512) / 22).bfloat16()
    x, gate = rnd(2, 96, 256).bfloat16(), rnd(2, 256).bfloat16()
    dr, dy = rnd(2, 96, 256).bfloat16(), rnd(2, 96, 256).bfloat16()
    mlp = ex.GatedMLP(up.cuda(), down.cuda())
    with torch.no_grad():
        for p in (mlp.before, mlp.post, mlp.after):
            p.copy_(1 + 0.3 * rnd(256))
    leaves = [x.cuda().requires_grad_(), gate.cuda().requires_grad_(), mlp.up, mlp.down, mlp.before, mlp.post, mlp.after]
    out = mlp(leaves[0], leaves[1])
    got = torch.autograd.grad(out, leaves, (dr.cuda(), dy.cuda()))

    d = [t.detach().cpu().double().requires_grad_() for t in leaves]
    xd, gd, w1, w2, before, post, after = d
    rms = lambda t: t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)                   # noqa: E731
    a, u = (rms(xd) * before @ w1.T).chunk(2, -1)
    r = xd + gd[:, None] * rms((a * torch.sigmoid(a) * u) @ w2.T) * post
    want = (r, rms(r) * after)
    off = lambda p, q: float((p.detach().cpu().double() - q.detach()).norm() / q.detach().norm())   # noqa: E731
    assert off(out[0], want[0]) < 0.032 and off(out[1], want[1]) < 0.032
    for name, p, q in zip(("x", "gate", "up", "down", "before", "post", "after"), got,
                          torch.autograd.grad(want, d, (dr.double(), dy.double()))):
        assert off(p, q) < 0.032, name
