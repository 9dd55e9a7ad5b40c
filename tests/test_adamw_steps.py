"""The optimizer's bookkeeping when a step is refused, and moments that lie on the host (CPU only: no kernel runs)."""
import pytest
import torch

from conftest import sub

fa = sub("enhancers.fused_adamw")


def parameter(*shape):
    p = torch.nn.Parameter(torch.randn(*shape))
    p.grad = torch.randn(*shape)
    return p


def test_a_refused_step_is_not_counted():
    # (parameters on the host are refused by adamw_step itself, after the optimizer's own checks)
    p = parameter(300)
    opt = fa.AdamW([p])
    for _ in range(3):
        with pytest.raises(ValueError, match="GPU"):
            opt.step()
    assert opt.state[p].get("step", 0) == 0


def test_every_group_is_looked_at_before_the_first_step():
    # (a first group that stepped would be refused for lying on the host)
    p, q, r = parameter(300), parameter(20), parameter(5)
    opt = fa.AdamW([{"params": [p]}, {"params": [q, r]}])
    r.grad = None
    with pytest.raises(ValueError, match="GPU"):
        opt.step()
    p.grad = None
    with pytest.raises(ValueError, match="no gradient"):
        opt.step()
    q.grad = None
    opt.step()                                                  # no gradients at all: nothing to do
    assert not any(opt.state.values())


def test_values_of_moments_on_the_host():
    p = torch.randn(300)
    with pytest.raises(ValueError, match="GPU"):
        fa.adamw_state([p], 8).values()
    assert all(t.numel() == 512 for t in fa.adamw_state([p], 32).values())     # float32: the state's own tensors
