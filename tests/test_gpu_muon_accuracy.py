"""How far orthogonalised updates above a shorter side of 64 are from the definition, by the kind of matrix: the figures that the operator
states. What matters is the conditioning of the five steps: a singular value's relative error grows by up to 10 on the polynomial's steep
parts, each step adds roundings of 2^-11, and many singular values average them.

Tolerances (set before the first run). The float64 model of the kernels' roundings (test_gpu_muon.rounded) is off by at most 1.6e-3 of the
norm for flat spectra, 1.0e-3 for falling ones, 3.6e-3 for one to 64 random directions of equal or falling sizes with noise up to
1e-2, 1.15e-2 for two or three entries, over 6000 matrices from 65 x 65 to 1531 x 1021; the stated figures are those, rounded up.
Beside them each result stays within half as much again as its own model's distance, and its type's rounding."""
import pytest
import torch

from conftest import sub
from test_gpu_muon import UNIT, definition, matrix, rounded

pytestmark = pytest.mark.gpu
fm = sub("enhancers.fused_muon")
STATED = {"flat": 2e-3, "falling": 2e-3, "directions": 4e-3, "entries": 1.5e-2}


def matrices(rows, cols, g):
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")                                # noqa: E731
    for kind in ("flat", "falling"):
        yield kind, matrix(rows, cols, kind, g)
    for rank in (1, 2, 8, 32, 64):
        for fall, noise in ((0, 0.0), (0, 1e-3), (1, 1e-2), (4, 0.0)):
            sizes = torch.arange(1, rank + 1, device="cuda") ** -float(fall)
            yield "directions", (rnd(rows, rank) * sizes) @ rnd(rank, cols) + noise * rnd(rows, cols)
    for entries in (1, 2, 3):
        for fall in (0, 1):
            x = torch.zeros(rows, cols, device="cuda")
            x.diagonal()[:entries] = rnd(entries) * torch.arange(1, entries + 1, device="cuda") ** -float(fall)
            yield "entries", x


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(65, 65), (200, 90), (96, 512), (257, 333), (1021, 1531), (4000, 65)])
def test_stated_accuracy(native, rows, cols, dtype):
    dt, g = getattr(torch, dtype), torch.Generator(device="cuda").manual_seed(rows + cols)
    print(f"case accuracy {rows} x {cols} {dtype}", flush=True)
    for i, (kind, x) in enumerate(matrices(rows, cols, g)):
        x = x.to(dt)
        got, want = fm.orthogonalize(x).double(), definition(x)
        off, model = (float((v - want).norm() / want.norm()) for v in (got, rounded(x)))
        assert off <= STATED[kind] + UNIT[dt], (i, kind, off)
        assert off <= 1.5 * model + UNIT[dt] + 1e-6, (i, kind, off, model)
