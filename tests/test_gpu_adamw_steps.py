"""AdamW steps that are refused leave everything as it was: parameters, moments and the count of steps.
A step is not captured into a graph."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

fa = sub("enhancers.fused_adamw")


@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_step_changes_nothing(native, bits):
    g = torch.Generator(device="cuda").manual_seed(1)
    start = torch.randn(40, 60, generator=g, device="cuda")
    grads = [torch.randn(40, 60, generator=g, device="cuda") for _ in range(3)]
    p, q = (torch.nn.Parameter(start.clone()) for _ in range(2))
    opt, ref = fa.AdamW([p], bits=bits), fa.AdamW([q], bits=bits)
    for d in grads:
        p.grad = d.T.contiguous().T                                 # not contiguous: refused, then mended
        with pytest.raises(ValueError, match="contiguous"):
            opt.step()
        p.grad, q.grad = d.clone(), d.clone()
        opt.step()
        ref.step()
        assert torch.equal(p, q)
    assert opt.state[p]["step"] == ref.state[q]["step"] == 3


def test_no_group_steps_when_another_is_refused(native):
    p, q, r = (torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(3))
    opt = fa.AdamW([{"params": [p]}, {"params": [q, r]}])
    for t in (p, q, r):
        t.grad = torch.ones(300, device="cuda")
    for wrong in (None, torch.ones(600, device="cuda")[::2]):
        r.grad = wrong
        with pytest.raises(ValueError):
            opt.step()
        assert all(torch.equal(t.detach(), torch.ones_like(t)) for t in (p, q, r)) and not any(opt.state.values())
    r.grad = torch.ones(300, device="cuda")
    opt.step()
    assert torch.equal(p, q) and torch.equal(q, r) and float(p.detach().max()) < 1.0
    assert opt.state[p]["step"] == opt.state[q]["step"] == 1


def test_a_step_is_not_captured(native):
    # its step count, rates and addresses are the call's: a replay would repeat them
    p = torch.nn.Parameter(torch.zeros(300, device="cuda"))
    p.grad = torch.ones(300, device="cuda")
    opt = fa.AdamW([p])
    opt.step()
    torch.cuda.synchronize()
    before = p.detach().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = p.detach() * 2
        with pytest.raises(RuntimeError, match="graph"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), before) and torch.equal(y, before * 2) and opt.state[p]["step"] == 1
