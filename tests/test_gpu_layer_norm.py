"""GPU parity of LayerNorm, forward and backward, against the formula in float64 on the CPU, and of its refusals.

Tolerances (set before the first run). A row's sum takes at most 32 additions in a lane, 6 over a wave and 16 over a
team, so a mean is off by at most 2^-18 mean|x| and a variance by 2^-18 of itself: with A = mean|x| rstd the normalised
value is off by 2^-18 (A + |xh|), y by that times |s|, two more float32 roundings, and the rounding u of the output's type
(2^-24, 2^-11, 2^-8). dx collects the same errors in g, its two means and xh, each no more than twice: 2^-17. The parameters'
gradients add at most a few hundred float32 terms a column: 2^-16 of the sum of magnitudes."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
fn = sub("enhancers.fused_norm")


def formula(x, w, b, dy, groups, plus, eps):
    """y, dx, dw, db and the magnitudes their errors go by, all float64."""
    x, dy = x.double(), dy.double()
    rows, k = x.shape
    per = lambda t: t.double().reshape(groups, 1, k).expand(groups, rows // groups, k).reshape(rows, k)  # noqa: E731
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh, a = (x - mean) * rstd, x.abs().mean(1, keepdim=True) * rstd
    s = torch.ones_like(x) if w is None else per(w) + plus
    off = torch.zeros_like(x) if b is None else per(b)
    g = dy * s
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    fold = lambda t: t.reshape(groups, rows // groups, k).sum(1)                                         # noqa: E731
    n1, n2 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    return {"y": (xh * s + off, 2.0 ** -18 * (a + xh.abs()) * s.abs() + 2.0 ** -23 * off.abs()),
            "dx": (rstd * (g - m1 - xh * m2),
                   2.0 ** -17 * rstd * (g.abs() + n1 + (xh.abs() + a) * (n2 + a * n1))),
            "dw": (fold(dy * xh), 2.0 ** -16 * fold(dy.abs() * (xh.abs() + a))),
            "db": (fold(dy), 2.0 ** -16 * fold(dy.abs()))}


def check(got, want, what):
    ref, tol = want
    unit = UNIT[got.dtype]
    err = (got.double().cpu().reshape(ref.shape) - ref).abs()
    assert bool((err <= tol + ref.abs() * unit).all()), (what, float((err - tol - ref.abs() * unit).max()))


def inputs(rows, k, dtype, pdtype, groups, params, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, k, generator=g) * torch.exp(torch.randn(k, generator=g) * 0.5)
         + torch.randn(k, generator=g)).to(dtype)
    shape = (k,) if groups == 1 else (groups, k)
    w = torch.randn(shape, generator=g).to(pdtype) if "w" in params else None
    b = torch.randn(shape, generator=g).to(pdtype) if "b" in params else None
    return x, w, b, torch.randn(rows, k, generator=g).to(dtype)


# widths: one value, below / at / past a pack, odd, 5120 and 2048 of the DiT shapes, every number of waves a row
@pytest.mark.parametrize("rows,k,dtype,pdtype,groups,params", [
    (1, 1, "float32", "float32", 1, "wb"), (3, 7, "bfloat16", "bfloat16", 1, "wb"), (5, 8, "float16", "float16", 1, "w"),
    (1, 5120, "bfloat16", "bfloat16", 1, "wb"), (130, 1531, "float32", "float32", 1, "wb"),
    (257, 1531, "bfloat16", "float32", 1, "wb"), (64, 2048, "bfloat16", "float32", 2, "wb"),
    (63, 5120, "bfloat16", "bfloat16", 3, "wb"), (40, 5123, "float16", "float16", 1, ""),
    (33, 2049, "bfloat16", "bfloat16", 33, "wb"), (20, 9000, "float16", "float32", 1, "b"),
    (7, 20001, "bfloat16", "bfloat16", 1, "wb"), (4, 32768, "bfloat16", "bfloat16", 1, "wb"),
    (4, 32767, "float32", "float32", 2, "wb"), (3000, 64, "bfloat16", "bfloat16", 1, "wb"),
    (2000, 513, "float32", "float32", 4, "wb"), (9, 4096, "float32", "float32", 1, "wb"),
    (9, 12288, "float32", "float32", 1, "wb"), (1200, 320, "float16", "float16", 600, "wb")])
@pytest.mark.parametrize("modulation", [False, True])
def test_layer_norm_and_gradients(native, rows, k, dtype, pdtype, groups, params, modulation):
    x, w, b, dy = inputs(rows, k, getattr(torch, dtype), getattr(torch, pdtype), groups, params, rows + 3 * k)
    want = formula(x, w, b, dy, groups, 1.0 if modulation else 0.0, 1e-6)
    leaves = [None if t is None else t.cuda().requires_grad_() for t in (x, w, b)]
    y = fn.layer_norm(*leaves, eps=1e-6, modulation=modulation)
    check(y, want["y"], "y")
    with torch.no_grad():
        plain = fn.layer_norm(*leaves, eps=1e-6, modulation=modulation)
    assert torch.equal(plain, y)
    asked = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None],
                     torch.autograd.grad(y, asked, dy.cuda(), retain_graph=True)))
    for name, got in grads.items():
        check(got, want[name], name)
    again = torch.autograd.grad(y, asked, dy.cuda())
    assert all(torch.equal(p, q) for p, q in zip(again, grads.values()))         # the same bits on every run


def test_layer_norm_gradient_against_differences(native):
    # along the gradient's own direction the loss changes by |gradient|; central differences of the float32 forward pass at
    # step 1e-2: their truncation and rounding stay below 1 %
    x, w, b, dy = (t.cuda() for t in inputs(12, 700, torch.float32, torch.float32, 3, "wb", 5))
    loss = lambda *t: (fn.layer_norm(*t, eps=1e-5, modulation=True).double() * dy.double()).sum()    # noqa: E731
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i, g in enumerate(grads):
        size = g.double().norm()
        step = g / size * 1e-2
        hi, lo = [x, w, b], [x, w, b]
        hi[i], lo[i] = hi[i] + step, lo[i] - step
        with torch.no_grad():
            diff = (loss(*hi) - loss(*lo)) / 2e-2
        assert abs(float(diff / size) - 1) < 1e-2, i


def test_layer_norm_strides_streams_and_partial_gradients(native):
    base = torch.randn(6, 40, 3 * 130, device="cuda").to(torch.bfloat16)
    w = torch.randn(130, device="cuda", dtype=torch.float32)
    view = base[:, :, 131:261]                                    # rows 390 values apart, 2-byte aligned
    assert torch.equal(fn.layer_norm(view, w), fn.layer_norm(view.contiguous(), w))
    turned = base.transpose(0, 2)[:130].transpose(0, 2)            # not unit stride after the slice of a transposed view
    assert torch.equal(fn.layer_norm(turned, w), fn.layer_norm(turned.contiguous(), w))
    wide = torch.randn(130, 96, device="cuda").T                   # columns contiguous
    assert torch.equal(fn.layer_norm(wide), fn.layer_norm(wide.contiguous()))
    one = torch.randn(130, device="cuda").expand(50, 130)          # every row the same memory, and a gradient that is one
    one.requires_grad_()
    y = fn.layer_norm(one, w)
    (gx,) = torch.autograd.grad(y.sum(), one)
    assert gx.shape == one.shape and bool(torch.isfinite(gx).all())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = view.clone().requires_grad_()
        y = fn.layer_norm(x, w)
        (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, fn.layer_norm(view, w)) and gx.shape == view.shape
    # only the parameters ask for gradients: dx is not computed, and only x does
    wg = w.clone().requires_grad_()
    (gw,) = torch.autograd.grad(fn.layer_norm(view, wg), wg, torch.ones(6, 40, 130, device="cuda", dtype=torch.bfloat16))
    xg = view.detach().clone().requires_grad_()
    both = torch.autograd.grad(fn.layer_norm(xg, wg), (xg, wg), torch.ones_like(xg))
    assert torch.equal(both[1], gw)
    xg2 = view.detach().clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(fn.layer_norm(xg2, w), xg2, torch.ones_like(xg2))[0], both[0])


def test_layer_norm_special_values(native):
    x = torch.randn(6, 300, device="cuda")
    x[1, 5], x[2, 7], x[3] = float("nan"), float("inf"), 4.0       # a constant row: xh = 0
    y = fn.layer_norm(x, bias=torch.full((300,), 0.5, device="cuda"))
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[2]).all())
    assert torch.equal(y[3], torch.full_like(y[3], 0.5))
    clean = fn.layer_norm(x[[0, 4, 5]], bias=torch.full((300,), 0.5, device="cuda"))
    assert torch.equal(y[[0, 4, 5]], clean)                        # no row reads another
    far = torch.randn(8, 2048, device="cuda") + 1000.0             # the mean far above the deviation
    ref = torch.nn.functional.layer_norm(far.double(), (2048,))
    # 2^-18 (A + |xh|) with A about 1000 (the formula's bound above)
    assert float((fn.layer_norm(far).double() - ref).abs().max()) <= 2.0 ** -18 * 1010
    empty = torch.empty(0, 64, device="cuda", requires_grad=True)
    wg = torch.ones(64, device="cuda", requires_grad=True)
    y = fn.layer_norm(empty, wg)
    gx, gw = torch.autograd.grad(y.sum(), (empty, wg))
    assert y.shape == (0, 64) and gx.shape == (0, 64) and float(gw.abs().sum()) == 0.0


def test_layer_norm_refusals(native):
    x = torch.randn(6, 32, device="cuda")
    w = torch.randn(32, device="cuda")
    assert fn.layer_norm(x.cpu()) is None and fn.layer_norm(x.double()) is None
    assert fn.layer_norm(x, w.half()) is None and fn.layer_norm(x, w.cpu()) is None
    assert fn.layer_norm(torch.randn(2, 32769, device="cuda")) is None
    with pytest.raises(ValueError, match="last dimension"):
        fn.layer_norm(x, w[:31])
    with pytest.raises(ValueError, match="groups"):
        fn.layer_norm(x, torch.randn(4, 32, device="cuda"))
    with pytest.raises(ValueError, match="differ"):
        fn.layer_norm(x, w, torch.randn(2, 32, device="cuda"))
    xg = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(fn.layer_norm(xg).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), xg)                           # differentiable once
