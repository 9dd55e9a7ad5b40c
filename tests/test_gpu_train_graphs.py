"""layer_norm and dense in a captured graph, forward and backward: every replay, on new inputs and with the program's own work
between, gives what the eager calls give."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

fn, fd = sub("enhancers.fused_norm"), sub("enhancers.fused_dense")


@pytest.mark.parametrize("rows,k,n", [(64, 2048, 512), (515, 333, 129)])
def test_training_passes_in_a_graph(native, rows, k, n):
    g = torch.Generator(device="cuda").manual_seed(rows)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)            # noqa: E731
    x, dy, res = rnd(rows, k), rnd(rows, n), rnd(rows, n)
    params = [t.requires_grad_() for t in (rnd(k), rnd(k), rnd(n, k) / 16, rnd(n), rnd(n))]
    leaves = [x.requires_grad_(), *params]

    def step():
        h = fn.layer_norm(x, params[0], params[1])
        y = fd.dense(h, params[2], params[3], "gelu_tanh", res, params[4])
        return (y, *torch.autograd.grad(y, leaves, dy))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(5):
        with torch.no_grad():
            x.copy_(rnd(rows, k))
            dy.copy_(rnd(rows, n))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i
