"""A matrix that holds an infinity or a NaN: divided by its norm it holds a NaN, which the first product of a row with a row carries into
every place. The other matrices of the same launches are what they are without it."""
import pytest
import torch

from conftest import sub
from test_gpu_muon import matrix

pytestmark = pytest.mark.gpu
fm = sub("enhancers.fused_muon")
SHAPES = [(1, 1), (1, 40), (16, 16), (40, 90), (90, 40), (64, 300), (65, 70), (200, 90), (90, 200), (129, 300), (600, 600), (130, 4000)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
def test_every_place_of_its_matrix_alone(native, bad, dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    for rows, cols in SHAPES:
        print(f"case {rows} x {cols} {bad} {dtype}", flush=True)
        x = torch.stack([matrix(rows, cols, "flat", g) for _ in range(4)]).to(getattr(torch, dtype))
        x[2] = 0                                                  # (alone among zeros, where a norm of infinity leaves nothing else)
        want = fm.orthogonalize(x)
        y = x.clone()
        y[1, rows // 2, cols // 3] = y[2, rows - 1, 0] = float(bad)
        for steps in (1, 2, 5):
            got = fm.orthogonalize(y, steps=steps)
            assert got[1].isnan().all() and got[2].isnan().all(), (rows, cols, steps)
            assert got[0].isfinite().all() and got[3].isfinite().all()
        assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])
        p, m = [torch.ones_like(t) for t in y], fm.muon_momenta(y)
        fm.muon_step(p, list(y), m)
        for i, (q, v) in enumerate(zip(p, m)):
            assert q.isnan().all() if i in (1, 2) else q.isfinite().all() and v.isfinite().all(), (rows, cols, i)
        at = torch.zeros(rows, cols, dtype=torch.bool, device="cuda")
        at[rows // 2, cols // 3] = True
        assert torch.equal(~m[1].isfinite(), at)                  # a momentum stays what it is, place by place
