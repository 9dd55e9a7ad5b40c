"""The forms of the orthogonalised updates that test_gpu_muon.py's shapes do not reach (tests/test_muon_forms.py holds both files to the
plan): sums in slices with their second launch, the large tiles in both orders, and calls of more matrices than a launch takes,
whose last launch may run in another form than the ones before. Bounds as there."""
import ctypes
import math

import pytest
import torch

from conftest import sub
from test_gpu_muon import UNIT, definition, hold, matrix, rounded

pytestmark = pytest.mark.gpu
fm = sub("enhancers.fused_muon")

SHAPES = [(3, 2288, 2394), (1, 1428, 2925), (1, 1021, 13824), (5, 1194, 10176), (1, 65, 2127), (1, 200, 5000), (8, 76, 5732),
          (2, 182, 8000), (4, 2097, 1936), (1, 7360, 4480), (19, 544, 409), (1, 8448, 2706), (1, 2944, 1443), (1, 6542, 3080),
          (1, 2292, 68), (1, 3000, 130), (8, 3866, 66), (1, 12352, 657), (16, 392, 1088), (1, 1532, 7552), (3, 11968, 261),
          (100, 418, 147), (3, 262, 11720), (2, 66, 13312), (3, 8512, 65)]
# more matrices than a launch takes: narrow ones both ways; tiles; a last launch in slices where the ones before are not; ones
# before in slices of their own
BATCHES = [(131, 16, 40), (257, 40, 16), (129, 50, 300), (129, 65, 68), (20, 2048, 2048), (129, 65, 2113), (129, 2113, 65),
           (59, 129, 4353), (8, 1025, 7169), (22, 5133, 513)]


def batch(count, rows, cols):
    plan = (ctypes.c_int * 7)()
    assert sub("_native").lib().wf_muon_plan(count, rows, cols, plan) == 0
    return plan[0]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("i", range(len(SHAPES)), ids=["x".join(map(str, s)) for s in SHAPES])
def test_orthogonalize(native, i, dtype):
    count, rows, cols = SHAPES[i]
    g = torch.Generator(device="cuda").manual_seed(300 + i)
    print(f"case orthogonalize {count} x {rows} x {cols} {dtype}", flush=True)
    x = torch.stack([matrix(rows, cols, ("falling", "flat")[(k + i) % 2], g) for k in range(count)]).to(getattr(torch, dtype))
    got = fm.orthogonalize(x)
    for k in {0, count - 1}:
        hold(got[k], x[k], (i, k))
    assert torch.equal(got, fm.orthogonalize(x))


@pytest.mark.parametrize("count,rows,cols", BATCHES)
def test_more_matrices_than_a_launch_takes(native, count, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(count + rows)
    print(f"case batches {count} x {rows} x {cols}", flush=True)
    x = torch.stack([matrix(rows, cols, "falling", g) for _ in range(count)]).bfloat16()
    got, n = fm.orthogonalize(x), batch(count, rows, cols)
    assert n < count
    ends = sorted({k for first in range(0, count, n) for k in (first, min(first + n, count) - 1)})
    for k in ends:
        hold(got[k], x[k], k)
    # every matrix of a whole launch as in a launch of its own, and what is left as a call of that many
    for first in range(0, count, n):
        assert torch.equal(got[first:first + n], fm.orthogonalize(x[first:first + n])), first


@pytest.mark.parametrize("count,rows,cols", [s for s in BATCHES if s[0] * s[1] * s[2] < 40e6] + [(18, 2048, 2048)])
def test_a_step_of_more_matrices_than_a_launch_takes(native, count, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(count + cols)
    print(f"case a step of batches {count} x {rows} x {cols}", flush=True)
    lr, mu, decay = 0.05, 0.9, 0.2
    p = [(0.02 * torch.randn(rows, cols, generator=g, device="cuda")).bfloat16() for _ in range(count)]
    grads = [matrix(rows, cols, "falling", g).bfloat16() for _ in range(count)]
    m = [matrix(rows, cols, "flat", g) for _ in range(count)]
    old_p, old_m = [t.double() for t in p], [t.double() for t in m]
    fm.muon_step(p, grads, m, lr=lr, momentum=mu, weight_decay=decay, adjust="rms")
    n = batch(count, rows, cols)
    assert n < count
    ends = {k for first in range(0, count, n) for k in (first, min(first + n, count) - 1)}
    rate = lr * 0.2 * math.sqrt(max(rows, cols))
    for k in range(count):                                        # the tolerances of test_gpu_muon.test_steps
        d = grads[k].double()
        want_m = mu * old_m[k] + (1 - mu) * d
        assert bool(((m[k].double() - want_m).abs() <= 2.0 ** -22 * (mu * old_m[k].abs() + d.abs())).all()), k
        # a singular value is 1.21 at most: no parameter moves further than that times the rate from its decayed self
        moved = (p[k].double() - (1 - lr * decay) * old_p[k]).abs()
        assert float(moved.max()) <= 1.25 * rate + 2.0 ** -8 * float(old_p[k].abs().max()) and float(moved.max()) > 0, k
        if k not in ends:
            continue
        u = mu * want_m + (1 - mu) * d
        o = definition(u)
        want = (1 - lr * decay) * old_p[k] - rate * o
        off = 485 * 3 * 2.0 ** -24 + (3 * float((rounded(u) - o).abs().max()) if min(rows, cols) > 64 else 0)
        tol = UNIT[torch.bfloat16] * want.abs() + rate * off + 2.0 ** -22 * (old_p[k].abs() + rate * o.abs())
        err = (p[k].double() - want).abs()
        assert bool((err <= tol).all()), (k, float((err - tol).max()))
