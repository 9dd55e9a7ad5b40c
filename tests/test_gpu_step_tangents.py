"""Optimizer steps under forward mode: a tangent of a stepped tensor would be left behind, so the step is refused."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu
fa, fm = sub("enhancers.fused_adamw"), sub("enhancers.fused_muon")
forward_ad = torch.autograd.forward_ad


def test_tangents_are_refused(native):
    p, g = ([torch.randn(s, device="cuda") for s in ((40, 90), (8, 9))] for _ in range(2))
    m, state = fm.muon_momenta(p), fa.adamw_state(p, 32)
    kept = [t.clone() for t in (*p, *m, state.exp_avg, state.exp_avg_sq)]
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))                                # noqa: E731
    with forward_ad.dual_level():
        for args in (([dual(p[0]), p[1]], g, m), (p, [g[0], dual(g[1])], m), (p, g, [m[0], dual(m[1])])):
            with pytest.raises(ValueError, match="tangent"):
                fm.muon_step(*args)
        for args in (([dual(p[0]), p[1]], g, state), (p, [g[0], dual(g[1])], state), (p, g, state._replace(exp_avg=dual(state.exp_avg)))):
            with pytest.raises(ValueError, match="tangent"):
                fa.adamw_step(*args, 1)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, (*p, *m, state.exp_avg, state.exp_avg_sq)))
        fm.muon_step(p, g, m)                                     # forward mode at work elsewhere is no reason
        fa.adamw_step(p, g, state, 1)
    assert not torch.equal(p[0], kept[0]) and not torch.equal(state.exp_avg, kept[4])
