"""The formula that the GPU tests of the norms around a gated residual hold the kernels to, itself held to differences and to torch's
own norms (CPU, float64)."""
import pytest
import torch

from block_norm_formula import formula

NAMES = ("x", "h", "pw", "gate", "w", "b")


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("post", [None, "rms", "layer"])
@pytest.mark.parametrize("groups,modulation,scale", [(1, False, 1.0), (3, True, 0.5)])
def test_gradients_against_differences(norm, post, groups, modulation, scale):
    g = torch.Generator().manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)                            # noqa: E731
    rows, k = 6, 5
    x, h, gate, w, b = rnd(rows, k), rnd(rows, k), rnd(groups, k), rnd(groups, k), rnd(groups, k)
    pw = rnd(k) if post else None
    dr, dy = rnd(rows, k), rnd(rows, k)
    args = dict(groups=groups, norm=norm, post=post, scale=scale, modulation=modulation)
    value = dict(zip(NAMES, (x, h, pw, gate, w, b)))

    def loss(**changed):
        o = formula(*({**value, **changed}[n] for n in NAMES), None, None, **args)
        return float((o["r"][0] * dr).sum() + (o["y"][0] * dy).sum())
    grads = formula(x, h, pw, gate, w, b, dr, dy, **args)
    for n in NAMES:
        if value[n] is None:
            continue
        got, step = grads["d" + n][0], 1e-5
        want = torch.empty_like(value[n])
        for i in range(value[n].numel()):
            d = torch.zeros(value[n].numel(), dtype=torch.float64)
            d[i] = step
            d = d.view_as(value[n])
            want.view(-1)[i] = (loss(**{n: value[n] + d}) - loss(**{n: value[n] - d})) / (2 * step)
        # (a central difference is off by step^2 times a third derivative, and by 1e-15 / step of the loss's rounding)
        assert torch.allclose(got, want, rtol=1e-6, atol=1e-6), n


def test_outputs_against_torch():
    g = torch.Generator().manual_seed(6)
    x, h, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((4, 9), (4, 9), (9,), (9,)))
    o = formula(x, h, None, None, w, b, None, None, 1, "layer", None)
    assert torch.allclose(o["y"][0], torch.nn.functional.layer_norm(x + h, (9,), w, b, 1e-6))
    o = formula(x, h, w, None, None, None, None, None, 1, "rms", "rms")
    r = x + h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * w
    assert torch.allclose(o["r"][0], r) and torch.allclose(o["y"][0], r / torch.sqrt((r * r).mean(1, keepdim=True) + 1e-6))
