"""Gradients of the gated linear in float16 where [dg du], the operand between the pass's two kinds of kernels, leaves float16's range:
dg = dy u act'(g) is a product of two float16-sized values and passes 65504 long before a gradient does, or lies below 2^-24.

Tolerances (set before the first run): test_gpu_gated.py's, and where the operand is stored times a power of two that brings its largest
magnitude m to 2^14 or above, a rounding of 2^-25 there, which is 2^-39 m at most."""
import pytest
import torch

from conftest import sub
from test_gpu_dense import check
from test_gpu_gated import act64, formula, run_both

pytestmark = pytest.mark.gpu
fd = sub("enhancers.fused_dense")


def case(rows, n, k, x, w, g, u, dy, seed, positive=False):
    """Standard deviations of everything; g and u come from a float32 bias. `positive`: no signs, and dy the same everywhere."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")                              # noqa: E731
    t = {"x": rnd(rows, k) * x, "w": rnd(2 * n, k) * w, "b": torch.cat((rnd(n) * g, rnd(n) * u)), "dy": rnd(rows, n) * dy}
    if positive:
        t = {name: v.abs() for name, v in t.items()}
        t["dy"].fill_(dy)
    return {name: v if name == "b" else v.half() for name, v in t.items()}


def largest(t, act):
    d = {name: v.double() for name, v in t.items()}
    g, u = (d["x"] @ d["w"].T + d["b"]).chunk(2, 1)
    a, slope = act64(g, act)
    return float(torch.maximum((d["dy"] * u * slope).abs().max(), (d["dy"] * a).abs().max()))


def hold(t, act, names, what):
    m, want = largest(t, act), formula(t, act)
    want["dx"] = want["dx"][0], want["dx"][1] + 2.0 ** -39 * m * t["w"].double().abs().sum(0)
    want["dw"] = want["dw"][0], want["dw"][1] + 2.0 ** -39 * m * t["x"].double().abs().sum(0)
    y, grads = run_both(t, act)
    check(y, want["y"], (what, "y"))
    for name in names:
        assert grads[name].isfinite().all(), (what, name)
        check(grads[name], want[name], (what, name))
    again = run_both(t, act)[1]
    assert all(torch.equal(again[name], grads[name]) for name in grads)
    return m, grads


# the backward products as few rows, in tiles, in slices, of odd lengths
SHAPES = [(1, 64, 72), (5, 640, 4160), (33, 320, 64), (300, 1000, 264), (301, 77, 129), (2049, 130, 200), (16, 2048, 1024)]


@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_products_past_the_largest(native, rows, n, k):
    print(f"case gated range, large: {rows} x {n} x {k}", flush=True)
    # dg is about 1e5 and reaches 1e6; x and w are so small that dx and dw are not
    t = case(rows, n, k, 1e-3, 0.03 / n ** 0.5, 1.0, 1000.0, 100.0, rows + n)
    m, _ = hold(t, "silu", ("dx", "dw", "db"), (rows, n, k))
    assert m > 2 * 65504


@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_products_below_the_smallest(native, rows, n, k):
    print(f"case gated range, small: {rows} x {n} x {k}", flush=True)
    # dg and du are about 2^-26 and would be zeros; dw is a sum of 50 times as much, or dx is
    for x, w, name in ((64.0, 1.0 / (64 * k), "dw"), (1.0 / (64 * k), 64.0, "dx")):
        t = case(rows, n, k, x, w, 0.2, 0.2, 2.0 ** -24, rows + n, positive=True)
        m, grads = hold(t, None, ("dx", "dw", "db"), (rows, n, k, name))
        assert m < 2.0 ** -20 and (grads[name] != 0).all()


def test_one_gradient_alone_and_float32_range(native):
    t = case(64, 96, 80, 1e-3, 0.003, 1.0, 1000.0, 100.0, 5)
    want = run_both(t, "silu")[1]
    for name, key in (("dx", "x"), ("dw", "w"), ("db", "b")):
        leaf = {k: v.clone().requires_grad_(k == key) for k, v in t.items() if k != "dy"}
        got, = torch.autograd.grad(fd.gated_dense(leaf["x"], leaf["w"], leaf["b"]), leaf[key], t["dy"])
        assert torch.equal(got, want[name]), name
    # an infinite or missing gradient stays in its row; the others are finite though the finite ones would not fit
    t["dy"][3, 7], t["dy"][9, 1] = float("inf"), float("nan")
    grads = run_both(t, "silu")[1]
    clean = torch.ones(64, dtype=torch.bool, device="cuda")
    clean[3] = clean[9] = False
    assert torch.equal(grads["dx"][clean], want["dx"][clean])
    assert not grads["dx"][3].isfinite().any() and grads["dx"][9].isnan().all()
    # no gradient at all
    t["dy"].zero_()
    assert all((g == 0).all() for g in run_both(t, "silu")[1].values())


def test_replayed_with_other_ranges(native):
    t = case(130, 200, 160, 1e-3, 0.02, 1.0, 1000.0, 1.0, 7)
    leaf = {k: v.clone().requires_grad_() for k, v in t.items() if k != "dy"}
    step = lambda: torch.autograd.grad(fd.gated_dense(leaf["x"], leaf["w"], leaf["b"]), list(leaf.values()), t["dy"])   # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for size in (1.0, 1e3, 1e-6, 1.0, 0.0, 1e2):                  # as it is, past the largest, below the smallest, and back
        t["dy"].copy_(torch.randn(130, 200, device="cuda") * size)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), size
