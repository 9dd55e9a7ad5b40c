"""GPU parity of the gated linear, forward and backward, against the formula in float64, and of its refusals.

Tolerances (set before the first run), elementwise. Both pre-activations are float32 sums, off by at most 2^-16 of the sum of their
terms' magnitudes (K up to 2^13 terms in any order stay far below that); activations by 2^-20 (1 + |g|), and none is steeper
than 1.13. y is their product, rounded once (u = 2^-8 bfloat16, 2^-11 float16). For the backward pass g and u are kept in 24 bits,
off by 2^-17 more; the slope's own slope is at most 1.3. dg and du are rounded to the operands' type before the two products, whose
float32 sums add 2^-16 of the terms' magnitudes, and whose outputs are rounded once."""
import math

import pytest
import torch

from conftest import sub
from test_gpu_dense import UNIT, act64, check

pytestmark = pytest.mark.gpu
fd = sub("enhancers.fused_dense")


def make(rows, n, k, dtype, bias, seed, bdtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")                               # noqa: E731
    return {"x": rnd(rows, k).to(dtype), "w": (rnd(2 * n, k) * 1.5 / math.sqrt(k)).to(dtype),
            "b": rnd(2 * n).to(bdtype or dtype) if bias else None, "dy": rnd(rows, n).to(dtype)}


def formula(t, act):
    """{name: (value, tolerance before the output's rounding)} in float64."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    n, unit = d["w"].shape[0] // 2, UNIT[t["x"].dtype]
    h, eh = d["x"] @ d["w"].T, 2.0 ** -16 * (d["x"].abs() @ d["w"].abs().T)
    if d["b"] is not None:
        h, eh = h + d["b"], eh + 2.0 ** -23 * d["b"].abs()
    g, u, eg, eu = h[:, :n], h[:, n:], eh[:, :n], eh[:, n:]
    a, slope = act64(g, act)
    soft = act in ("gelu", "gelu_tanh", "silu")
    own = 2.0 ** -20 * (1 + g.abs()) if soft else 0.0
    ea = 1.13 * eg + own
    out = {"y": (a * u, u.abs() * ea + (a.abs() + ea) * eu + 2.0 ** -23 * (a * u).abs())}
    eg, eu = eg + 2.0 ** -17 * g.abs(), eu + 2.0 ** -17 * u.abs()
    es = 1.3 * eg + 2.0 ** -19 if soft else 0.0 * g
    if act == "relu":
        es = es + (g.abs() <= eg)                               # on either side of the corner
    dy = d["dy"]
    dh = torch.cat((dy * u * slope, dy * a), 1)
    e = torch.cat((dy.abs() * (eu * slope.abs() + (u.abs() + eu) * es), dy.abs() * (1.13 * eg + own)), 1) + 2.0 ** -22 * dh.abs()
    out["db"] = (dh.sum(0), e.sum(0) + 2.0 ** -16 * (dh.abs() + e).sum(0))
    e = e + unit * (dh.abs() + e) + (2.0 ** -25 if t["x"].dtype == torch.float16 else 0.0)
    mag = dh.abs() + e
    out["dx"] = (dh @ d["w"], e @ d["w"].abs() + 2.0 ** -16 * (mag @ d["w"].abs()))
    out["dw"] = (dh.T @ d["x"], e.T @ d["x"].abs() + 2.0 ** -16 * (mag.T @ d["x"].abs()))
    return out


def run_both(t, act):
    names = [n for n in ("x", "w", "b") if t[n] is not None]
    leaf = {n: t[n].detach().clone().requires_grad_() for n in names}
    y = fd.gated_dense(leaf["x"], leaf["w"], leaf.get("b"), act)
    grads = torch.autograd.grad(y, [leaf[n] for n in names], t["dy"])
    return y, dict(zip(["d" + n for n in names], grads))


def hold(t, act):
    want = formula(t, act)
    y, grads = run_both(t, act)
    check(y, want["y"], "y")
    for name, got in grads.items():
        check(got, want[name], name)
    with torch.no_grad():                                       # without a gradient the plan may be another: the same bounds
        check(fd.gated_dense(t["x"], t["w"], t["b"], act), want["y"], "y alone")
    return y, grads


# every kernel, tiling and whether in slices (tests/test_gated_forms.py holds the plan to that), sizes below / past a run, a
# fragment, a stage and a tile, odd everything
SHAPES = [
    (1, 1, 1), (1, 8, 8), (2, 2, 4448), (1, 1000, 5120), (2, 515, 1531), (3, 64, 72), (16, 2048, 4096), (17, 2607, 333),
    (33, 320, 64), (64, 640, 1088), (77, 2607, 1531), (130, 129, 127), (300, 1000, 264), (325, 2, 1), (290, 2, 312),
    (280, 5, 5760), (512, 1280, 1280), (1023, 1537, 513), (1560, 1024, 1024), (2049, 2056, 200), (4096, 2560, 320),
    (5000, 333, 96), (536, 524, 4736), (803, 3008, 455), (3880, 1560, 576), (1096, 1903, 6264), (6080, 4, 400), (8224, 165, 2),
    (256, 2560, 5120), (1881, 3424, 736), (1419, 1655, 896), (1392, 1536, 5376), (904, 1135, 7552), (262, 6, 1152), (512, 16, 928),
    (2112, 1824, 648), (104, 1265, 3264), (3640, 1, 2934), (2225, 1295, 1744), (104, 1791, 2448), (8640, 1, 1152), (2113, 1824, 648),
    (1984, 3200, 1302), (2048, 1040, 1814), (1420, 1656, 900), (1900, 3420, 737), (905, 1136, 7553), (1393, 1537, 5376), (263, 7, 1153), (513, 17, 928),
    (7144, 1, 1992), (10104, 2, 1536), (4584, 5, 365), (1292, 528, 20), (622, 5320, 626), (3640, 2, 2935), (300, 200, 9), (301, 201, 65),
    (330, 130, 8), (300, 200, 7), (260, 300, 127), (257, 65, 10), (1, 600, 4001), (8, 1000, 2047), (100, 700, 1025), (1, 9001, 2047)]


@pytest.mark.parametrize("i", range(len(SHAPES)), ids=["x".join(map(str, s)) for s in SHAPES])
def test_gated_and_gradients(native, i):
    rows, n, k = SHAPES[i]
    dtype = (torch.bfloat16, torch.float16)[i % 2]
    act = ("silu", "gelu", "gelu_tanh", None, "relu")[i % 5]
    print(f"case gated rows={rows} n={n} k={k} {dtype} {act}", flush=True)
    t = make(rows, n, k, dtype, i % 3 != 0, rows + 3 * n + 7 * k)
    y, grads = hold(t, act)
    y2, grads2 = run_both(t, act)
    assert torch.equal(y, y2) and all(torch.equal(grads[k_], grads2[k_]) for k_ in grads)


@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh", "silu", "relu"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_gated_activations_with_float32_bias(native, act, dtype):
    t = make(96, 200, 160, getattr(torch, dtype), True, 11, torch.float32)
    _, grads = hold(t, act)
    assert grads["db"].dtype == torch.float32


def test_gated_rows_that_start_anywhere(native):
    # views at every place of a 16-byte run, row lengths of their own, the last row ending with its memory
    for k in (8, 9, 15, 57, 64, 71, 128, 200, 449):
        for place in range(0, 8, 1 if k < 64 else 3):
            rows, n, x_row, w_row = 300 + place, 66 + k % 5, k + 3 * place + 1, k + place
            t = make(rows, n, k, torch.float16, False, k)

            def at(v, row, off):
                whole = torch.full((off + (v.shape[0] - 1) * row + k,), float("nan"), dtype=v.dtype, device="cuda")
                return torch.as_strided(whole, v.shape, (row, 1), off).copy_(v)
            got = fd.gated_dense(at(t["x"], x_row, place), at(t["w"], w_row, 7 - place), None, "silu")
            check(got, formula(t, "silu")["y"], f"k={k} place={place}")


def test_gated_gradient_against_differences(native):
    # along the gradient's own direction the loss, a float64 sum of float32-accurate outputs rounded once, changes by |gradient|
    # times the step. A step moves it by 2^-3 of the gradient's length; second differences cancel in the middle, the outputs'
    # rounding (2^-11 each, 6000 of them at random) stays below a per cent of the change
    t = make(64, 96, 80, torch.float16, True, 3, torch.float32)
    loss = lambda v: (fd.gated_dense(v["x"], v["w"], v["b"], "silu").double() * t["dy"].double()).sum()  # noqa: E731
    leaf = {n: t[n].clone().requires_grad_() for n in ("x", "w", "b")}
    grads = dict(zip(leaf, torch.autograd.grad(loss(leaf), list(leaf.values()))))
    for n in ("x", "w", "b"):
        g = grads[n].double()
        step = 0.05 * t[n].double().norm() / g.norm()
        with torch.no_grad():
            up, down = ({**t, n: (t[n].double() + s * step * g).to(t[n].dtype)} for s in (1, -1))
            moved = ((up[n].double() - down[n].double()) * g).sum()          # what rounding left of the two steps
            assert abs(float((loss(up) - loss(down)) / moved) - 1) < 0.03, n


def test_gated_strides_batches_streams_and_empty(native):
    t = make(48, 264, 200, torch.bfloat16, True, 5)
    y, grads = run_both(t, "silu")
    # rows apart, a weight that lies across, a misaligned start, a batch
    wide = torch.zeros(48, 300, dtype=torch.bfloat16, device="cuda")
    wide[:, 37:237] = t["x"]
    across = t["w"].t().contiguous().t()
    odd = torch.empty(528 * 200 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(528, 200).copy_(t["w"])
    for x, w in ((wide[:, 37:237], t["w"]), (t["x"], across), (t["x"].t().contiguous().t(), odd), (t["x"].view(4, 12, 200), t["w"])):
        leaf = x.detach().requires_grad_(), w.detach().requires_grad_(), t["b"].clone().requires_grad_()
        got = fd.gated_dense(*leaf)
        g = torch.autograd.grad(got, leaf, t["dy"].view(got.shape))
        want = formula(t, "silu")
        for v, name in ((got, "y"), (g[0], "dx"), (g[1], "dw"), (g[2], "db")):
            check(v, want[name], name)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other, _ = run_both(t, "silu")
    side.synchronize()
    assert torch.equal(other, y)
    # rows expanded from one; a gradient expanded from one
    one = t["x"][:1]
    assert torch.equal(fd.gated_dense(one.expand(48, 200), t["w"], t["b"]), fd.gated_dense(one.repeat(48, 1), t["w"], t["b"]))
    leaf = t["x"].clone().requires_grad_()
    a, = torch.autograd.grad(fd.gated_dense(leaf, t["w"]), leaf, t["dy"][:1].expand(48, 264))
    b, = torch.autograd.grad(fd.gated_dense(leaf, t["w"]), leaf, t["dy"][:1].repeat(48, 1))
    assert torch.equal(a, b)
    for rows, n in ((0, 264), (48, 0)):
        x = torch.zeros(rows, 200, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        w = torch.zeros(2 * n, 200, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        got = fd.gated_dense(x, w)
        assert got.shape == (rows, n)
        got.sum().backward()
        assert (x.grad == 0).all() and (w.grad == 0).all() and w.grad.shape == w.shape


def test_gated_infinities_stay_in_place(native):
    t = make(40, 64, 64, torch.bfloat16, False, 7)
    t["x"][3, 5], t["x"][9, 1] = float("inf"), float("nan")
    t["dy"][11] = 0
    y, grads = run_both(t, "silu")
    rows = torch.arange(40, device="cuda")
    clean = (rows != 3) & (rows != 9)
    assert y[clean].isfinite().all() and y[9].isnan().all() and not y[3].isfinite().all()
    assert grads["dx"][clean].isfinite().all() and (grads["dx"][11] == 0).all() and grads["dx"][9].isnan().all()


def test_gated_refusals(native):
    t = make(8, 16, 32, torch.bfloat16, True, 1)
    x, w, b = t["x"], t["w"], t["b"]
    call = fd.gated_dense
    assert call(x.cpu(), w.cpu()) is None and call(x.float(), w.float()) is None and call(x, w.half()) is None
    assert call(x, w, b.half()) is None and call(x.detach()._neg_view(), w) is None
    for bad in (lambda: call(x, w[:31]), lambda: call(x, w[:, :31]), lambda: call(x, w, b[:16]), lambda: call(x, w, act="tanh")):
        with pytest.raises(ValueError):
            bad()
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(call(leaf, w).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
