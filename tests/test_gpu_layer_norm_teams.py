"""LayerNorm at row counts that fill a workgroup with teams of waves (the backward pass then meets in up to 120 KB of LDS) and
walk several rows a team; tolerances are test_gpu_layer_norm.py's."""
import pytest
import torch

from conftest import sub
from test_gpu_layer_norm import check, formula, inputs

pytestmark = pytest.mark.gpu

fn = sub("enhancers.fused_norm")


@pytest.mark.parametrize("rows,k,dtype,pdtype,groups", [
    (4097, 1024, "bfloat16", "bfloat16", 1), (5000, 2048, "float16", "float32", 2), (4500, 770, "float32", "float32", 1),
    (9000, 509, "bfloat16", "float32", 3), (20000, 33, "float32", "float32", 1), (4100, 4100, "bfloat16", "bfloat16", 1),
    (2600, 1900, "float32", "float32", 4), (4098, 1023, "float16", "float16", 2049)])
def test_teams_of_waves(native, rows, k, dtype, pdtype, groups):
    print(f"case layer_norm rows={rows} k={k} {dtype} groups={groups}", flush=True)
    x, w, b, dy = inputs(rows, k, getattr(torch, dtype), getattr(torch, pdtype), groups, "wb", rows + k)
    want = formula(x, w, b, dy, groups, 1.0, 1e-6)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = fn.layer_norm(*leaves, eps=1e-6, modulation=True)
    check(y.detach(), want["y"], "y")
    grads = torch.autograd.grad(y, leaves, dy.cuda(), retain_graph=True)
    for name, got in zip(("dx", "dw", "db"), grads):
        check(got, want[name], name)
    for i, leaf in enumerate(leaves):                              # one gradient at a time is the same gradient
        assert torch.equal(torch.autograd.grad(y, leaf, dy.cuda(), retain_graph=True)[0], grads[i]), i
