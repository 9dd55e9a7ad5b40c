"""GPU parity of the 16-bit linear with its epilogue, forward and backward, against the formula in float64, and of its
refusals.

Tolerances (set before the first run), elementwise. The pre-activation is a float32 sum: off by at most 2^-16 of the sum of
its terms' magnitudes (K up to 2^13 terms in any order stay far below that), and activations by 2^-20 (1 + |h|); no
activation is steeper than 1.13. The output is rounded once (u = 2^-8 bfloat16, 2^-11 float16). In the backward pass h and
dh are rounded to the operands' type: dh is off by u |dh| and, through h, by 1.3 u |h dy gate| (|act''| <= 1.13), and dx, dw
by those errors multiplied through the product, their own float32 sums and one rounding."""
import math

import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
fd = sub("enhancers.fused_dense")


def act64(h, act):
    """The activation and its slope in float64."""
    if act == "gelu":
        phi = 0.5 * torch.special.erfc(-h / math.sqrt(2))
        return h * phi, phi + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)
    if act in ("gelu_tanh", "silu"):
        c = 2 * math.sqrt(2 / math.pi) if act == "gelu_tanh" else 1.0
        b = 0.044715 * c if act == "gelu_tanh" else 0.0
        s = torch.sigmoid(c * h + b * h ** 3)
        return h * s, s + h * s * (1 - s) * (c + 3 * b * h * h)
    if act == "relu":
        return h.clamp(min=0), (h > 0).double()
    return h, torch.ones_like(h)


def make(rows, n, k, dtype, bias, res, groups, seed, vdtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")                               # noqa: E731
    v = vdtype or dtype
    return {"x": rnd(rows, k).to(dtype), "w": (rnd(n, k) * 1.5 / math.sqrt(k)).to(dtype),
            "b": rnd(n).to(v) if bias else None, "r": rnd(rows, n).to(dtype) if res else None,
            "g": rnd(groups, n).to(v) if groups else None, "dy": rnd(rows, n).to(dtype)}


def formula(t, act):
    """{name: (value, tolerance before the output's rounding)} in float64."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    rows, n = d["x"].shape[0], d["w"].shape[0]
    u = UNIT[t["x"].dtype]
    h = d["x"] @ d["w"].T
    eh = 2.0 ** -16 * (d["x"].abs() @ d["w"].abs().T)
    if d["b"] is not None:
        h, eh = h + d["b"], eh + 2.0 ** -23 * d["b"].abs()
    a, slope = act64(h, act)
    ea = 1.13 * eh + (2.0 ** -20 * (1 + h.abs()) if act else 0)
    gate = torch.ones_like(h)
    groups = 1
    if d["g"] is not None:
        groups = d["g"].shape[0]
        gate = d["g"].repeat_interleave(rows // groups, 0)
    out = {"y": (gate * a + (0 if d["r"] is None else d["r"]), gate.abs() * ea + 2.0 ** -22 * (gate * a).abs())}
    da = d["dy"] * gate
    dh = da * slope
    soft = act in ("gelu", "gelu_tanh", "silu")
    es = da.abs() * (1.3 * (u * h.abs() + eh) + 2.0 ** -19 if soft else 0.0)
    if act == "relu":
        es = es + da.abs() * (h.abs() <= eh)                    # on either side of the corner
    ed = es + (u * (dh.abs() + es) if act or d["g"] is not None else 0)
    mag = dh.abs() + ed
    out["dx"] = (dh @ d["w"], ed @ d["w"].abs() + 2.0 ** -16 * (mag @ d["w"].abs()))
    out["dw"] = (dh.T @ d["x"], ed.T @ d["x"].abs() + 2.0 ** -16 * (mag.T @ d["x"].abs()))
    out["db"] = (dh.sum(0), es.sum(0) + 2.0 ** -16 * mag.sum(0))
    out["dr"] = (d["dy"], torch.zeros_like(h))
    fold = lambda v: v.reshape(groups, rows // groups, n).sum(1)                               # noqa: E731
    out["dg"] = (fold(d["dy"] * a), fold(d["dy"].abs() * (ea + 1.13 * u * h.abs() + 2.0 ** -16 * a.abs())))
    return out


def check(got, want, what):
    ref, tol = want
    err = (got.double().reshape(ref.shape) - ref).abs()
    most = tol + (ref.abs() + tol) * UNIT[got.dtype] + (2.0 ** -24 if got.dtype == torch.float16 else 0)
    assert bool((err <= most).all()), (what, float((err - most).max()), float((err / most.clamp(min=1e-30)).max()))


def run_both(t, act):
    names = [n for n in ("x", "w", "b", "r", "g") if t[n] is not None]
    leaf = {n: t[n].detach().clone().requires_grad_() for n in names}
    y = fd.dense(leaf["x"], leaf["w"], leaf.get("b"), act, leaf.get("r"), leaf.get("g"))
    grads = torch.autograd.grad(y, [leaf[n] for n in names], t["dy"])
    with torch.no_grad():
        assert torch.equal(fd.dense(t["x"], t["w"], t["b"], act, t["r"], t["g"]), y)
    return y, dict(zip(["d" + n for n in names], grads))


# one row to several tiles of every tiling, sizes below / past a pack, a stage and a tile, K slices, odd everything
@pytest.mark.parametrize("rows,n,k,dtype,act,bias,res,groups", [
    (1, 1, 1, "bfloat16", None, False, False, 0), (1, 8, 8, "float16", "relu", True, True, 1),
    (1, 1000, 5120, "bfloat16", "gelu_tanh", True, False, 0), (2, 515, 1531, "float16", "silu", True, True, 2),
    (3, 64, 72, "bfloat16", "gelu", True, False, 0), (16, 2048, 8192, "bfloat16", None, False, True, 1),
    (17, 2607, 333, "float16", "gelu", True, True, 0), (33, 320, 64, "bfloat16", "silu", True, False, 0),
    (64, 640, 1088, "bfloat16", "relu", False, False, 0), (77, 2607, 1531, "float16", "gelu", True, True, 0),
    (130, 129, 127, "bfloat16", "gelu_tanh", True, True, 2), (300, 1000, 264, "bfloat16", "gelu", True, False, 0),
    (512, 5120, 1280, "bfloat16", None, True, True, 4), (1023, 1537, 513, "float16", "gelu_tanh", True, True, 3),
    (1560, 2048, 1024, "bfloat16", "gelu_tanh", True, False, 0), (2049, 4104, 200, "bfloat16", "silu", False, True, 1),
    (4096, 5120, 320, "bfloat16", "gelu_tanh", True, True, 2), (5000, 333, 96, "float16", "relu", True, False, 0)])
def test_dense_and_gradients(native, rows, n, k, dtype, act, bias, res, groups):
    print(f"case dense rows={rows} n={n} k={k} {dtype} {act}", flush=True)
    rows = rows // max(1, groups) * max(1, groups)
    t = make(rows, n, k, getattr(torch, dtype), bias, res, groups, rows + 3 * n + 7 * k)
    want = formula(t, act)
    y, grads = run_both(t, act)
    check(y, want["y"], "y")
    for name, got in grads.items():
        check(got, want[name], name)
    y2, grads2 = run_both(t, act)
    assert torch.equal(y, y2) and all(torch.equal(grads[k_], grads2[k_]) for k_ in grads)


@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh", "silu", "relu"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_dense_activations_with_float32_vectors(native, act, dtype):
    t = make(96, 200, 160, getattr(torch, dtype), True, True, 3, 11, torch.float32)
    want = formula(t, act)
    y, grads = run_both(t, act)
    assert grads["db"].dtype == torch.float32 and grads["dg"].dtype == torch.float32
    check(y, want["y"], "y")
    for name, got in grads.items():
        check(got, want[name], name)


def test_dense_gradient_against_differences(native):
    # along the gradient's direction, in float16 with steps of many of its roundings: the loss (from float32 sums of the
    # outputs) changes by |gradient| times the step, to a few per cent
    t = make(64, 96, 80, torch.float16, True, True, 2, 3, torch.float32)
    names = ("x", "w", "b", "r", "g")
    loss = lambda v: (fd.dense(v["x"], v["w"], v["b"], "gelu", v["r"], v["g"]).double() * t["dy"].double()).sum()  # noqa: E731
    leaf = {n: t[n].clone().requires_grad_() for n in names}
    grads = torch.autograd.grad(loss(leaf), [leaf[n] for n in names])
    for name, g in zip(names, grads):
        step = g.double() / g.double().abs().max() * 0.05
        hi, lo = dict(t), dict(t)
        hi[name] = (t[name].double() + step).to(t[name].dtype)
        lo[name] = (t[name].double() - step).to(t[name].dtype)
        with torch.no_grad():
            diff = float(loss(hi) - loss(lo))
        along = float(((hi[name].double() - lo[name].double()) * g.double()).sum())
        assert abs(diff / along - 1) < 0.03, (name, diff, along)


def test_dense_views(native):
    # transposed, sliced and expanded operands give what their copies give
    big = torch.randn(400, 700, device="cuda").to(torch.bfloat16)
    x, w = big[:, 100:356], torch.randn(256, 192, device="cuda").to(torch.bfloat16).T
    r = torch.randn(192, 400, device="cuda").to(torch.bfloat16).T
    want = fd.dense(x.contiguous(), w.contiguous(), residual=r.contiguous())
    assert torch.equal(fd.dense(x, w, residual=r), want)
    assert torch.equal(fd.dense(big[:, 101:357].contiguous(), w), fd.dense(big[:, 101:357], w.contiguous()))
    x3 = x.reshape(4, 100, 256).transpose(0, 1)
    y3 = fd.dense(x3, w.contiguous(), residual=r.contiguous().view(4, 100, 192).transpose(0, 1))
    assert y3.shape == (100, 4, 192) and torch.equal(y3.transpose(0, 1).reshape(400, 192), want)
    one = w[:1].expand(64, 256)
    assert torch.equal(fd.dense(x, one), fd.dense(x, one.contiguous()))
    vec = fd.dense(x[0], w)
    assert vec.shape == (192,) and torch.equal(vec, fd.dense(x[:1], w)[0])
    # gradients through the views, dy a broadcast scalar
    xl, wl = big.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(fd.dense(xl[:, 100:356], wl, act="silu").float().sum(), (xl, wl))
    xc, wc = x.contiguous().requires_grad_(), w.contiguous().requires_grad_()
    hx, hw = torch.autograd.grad(fd.dense(xc, wc, act="silu").float().sum(), (xc, wc))
    assert torch.equal(gx[:, 100:356], hx) and float(gx[:, :100].abs().sum()) == 0.0 and torch.equal(gw, hw)


def test_dense_out_of_range_memory_is_not_used(native):
    # NaN all around the operands: rows and columns past the ends, and the K tail of a padded row, never reach a sum
    for rows, n, k in ((100, 130, 136), (1, 70, 200), (257, 322, 72)):
        buf = torch.full((rows + 600, k + 64), float("nan"), device="cuda", dtype=torch.bfloat16)
        wbuf = torch.full((n + 600, k + 64), float("nan"), device="cuda", dtype=torch.bfloat16)
        buf[:rows, :k], wbuf[:n, :k] = torch.randn(rows, k, device="cuda"), torch.randn(n, k, device="cuda")
        x, w = buf[:rows, :k], wbuf[:n, :k]
        y = fd.dense(x, w)
        assert bool(torch.isfinite(y).all()) and torch.equal(y, fd.dense(x.contiguous(), w.contiguous()))


def test_dense_infinities(native):
    # float16: a pre-activation past the type's range gives the limits of output and slope, not NaN
    x = torch.full((2, 64), 60.0, device="cuda", dtype=torch.float16)
    x[1] = -60.0
    w = torch.full((8, 64), 60.0, device="cuda", dtype=torch.float16).requires_grad_()
    for act in ("gelu", "gelu_tanh", "silu", "relu"):
        y = fd.dense(x, w, act=act)
        assert bool(torch.isinf(y[0]).all()) and float(y[1].abs().max()) == 0.0, act
        (gw,) = torch.autograd.grad(y, w, torch.tensor([[0.0], [1.0]], device="cuda").half().expand(2, 8))
        assert float(gw.abs().max()) == 0.0, act
    # a NaN row stays in its row
    x = torch.randn(40, 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(48, 64, device="cuda").to(torch.bfloat16)
    bad = x.clone()
    bad[7, 3] = float("nan")
    y, ref = fd.dense(bad, w, act="gelu"), fd.dense(x, w, act="gelu")
    keep = torch.arange(40, device="cuda") != 7
    assert bool(torch.isnan(y[7]).all()) and torch.equal(y[keep], ref[keep])


def test_dense_empty_and_streams(native):
    w = torch.randn(8, 64, device="cuda").to(torch.bfloat16).requires_grad_()
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    b = torch.randn(8, device="cuda").to(torch.bfloat16).requires_grad_()
    y = fd.dense(x, w, b, act="gelu")
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (0, 8) and gx.shape == (0, 64) and float(gw.abs().sum()) == 0 and float(gb.abs().sum()) == 0
    assert fd.dense(torch.randn(3, 64, device="cuda").to(torch.bfloat16), w[:0].detach()).shape == (3, 0)
    t = make(200, 300, 1000, torch.bfloat16, True, False, 0, 2)
    want = fd.dense(t["x"], t["w"], t["b"], "gelu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [fd.dense(t["x"], t["w"], t["b"], "gelu") for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, want) for g in got)


def test_dense_in_a_graph(native):
    # captured and replayed, each replay against the eager result on the same inputs
    t = make(64, 512, 2048, torch.bfloat16, True, True, 1, 9)
    args = (t["x"], t["w"], t["b"], "gelu_tanh", t["r"], t["g"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fd.dense(*args)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fd.dense(*args)
    for i in range(4):
        t["x"].copy_(torch.randn(64, 2048, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, fd.dense(*args)), i


def test_dense_refusals(native):
    x = torch.randn(6, 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(32, 64, device="cuda").to(torch.bfloat16)
    assert fd.dense(x.cpu(), w.cpu()) is None and fd.dense(x.float(), w.float()) is None
    assert fd.dense(x, w.half()) is None and fd.dense(x, w.cpu()) is None
    assert fd.dense(x, w, bias=torch.zeros(32, device="cuda", dtype=torch.float16)) is None
    assert fd.dense(x, w, residual=torch.zeros(6, 32, device="cuda")) is None
    with pytest.raises(ValueError, match="act"):
        fd.dense(x, w, act="tanh")
    with pytest.raises(ValueError, match="weight"):
        fd.dense(x, w[:, :63])
    with pytest.raises(ValueError, match="bias"):
        fd.dense(x, w, bias=x[0, :31])
    with pytest.raises(ValueError, match="residual"):
        fd.dense(x, w, residual=w[:5, :32])
    with pytest.raises(ValueError, match="groups"):
        fd.dense(x, w, gate=w[:4, :32])
