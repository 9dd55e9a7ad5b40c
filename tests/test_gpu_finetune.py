"""The training-step operators together: the MLP sub-layer's example lowers its loss, and one of its steps agrees with the
same sub-layer in float64 torch autograd on the CPU."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

ex = sub("examples.finetune_mlp")


@pytest.mark.parametrize("bits", [8, 32])
def test_example_learns(native, bits):
    r = ex.run(width=256, hidden=1024, tokens=256, steps=80, lr=1e-4, bits=bits)
    assert r["after"] < 0.7 * r["before"], r


def test_sub_layer_against_float64(native):
    # gradients through norm, two products, GELU and the gated residual: each bfloat16 rounding on the way is 2^-9 on
    # average, and the chain has six of them (normalised input, h, dh twice, the gradient between the products, the result):
    # 2 % of a gradient's norm is several times their sum
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g)                                              # noqa: E731
    up, down = (rnd(512, 256) / 16).bfloat16(), (rnd(256, 512) / 22).bfloat16()
    x, mod = rnd(2, 96, 256).bfloat16(), [(0.3 * rnd(2, 256)).bfloat16() for _ in range(3)]
    dy = rnd(2, 96, 256).bfloat16()
    mlp = ex.ModulatedMLP(up.cuda(), down.cuda())
    inputs = [x.cuda().requires_grad_()] + [m.cuda().requires_grad_() for m in mod]
    y = mlp(inputs[0], inputs[1:])
    leaves = inputs + [mlp.up, mlp.up_bias, mlp.down, mlp.down_bias]
    got = torch.autograd.grad(y, leaves, dy.cuda())

    d = [t.detach().cpu().double().requires_grad_() for t in leaves]
    xd, shift, scale, gate, w1, b1, w2, b2 = d
    h = torch.nn.functional.layer_norm(xd, (256,), eps=1e-6) * (1 + scale[:, None]) + shift[:, None]
    h = torch.nn.functional.gelu(h @ w1.T + b1, approximate="tanh")
    want = xd + gate[:, None] * (h @ w2.T + b2)
    assert float((y.detach().cpu().double() - want.detach()).norm() / want.detach().norm()) < 0.02
    for name, a, b in zip(("x", "shift", "scale", "gate", "up", "up_bias", "down", "down_bias"), got,
                          torch.autograd.grad(want, d, dy.double())):
        assert float((a.cpu().double() - b).norm() / b.norm()) < 0.02, name
