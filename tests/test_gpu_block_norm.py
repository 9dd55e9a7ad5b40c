"""GPU parity of the norms around a gated residual, forward and backward, against the formula in float64 and the bounds that
block_norm_formula.py derives, plus half a step of each output's type."""
import pytest
import torch

from block_norm_formula import formula
from conftest import sub

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
fn = sub("enhancers.fused_norm")
NAMES = ("x", "h", "pw", "gate", "w", "b")


def check(got, want, what):
    ref, tol = want
    err = (got.double().cpu().reshape(ref.shape) - ref).abs()
    # (float16's smallest steps are 2^-24 apart: half of one where a value is below its normal range)
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    room = tol + (ref.abs() + tol) * UNIT[got.dtype] + tiny
    assert bool((err <= room).all()), (what, float((err - room).max()))


def inputs(rows, k, dtype, pdtype, params, gate_groups, w_groups, seed):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)                                                 # noqa: E731
    x = (rnd(rows, k) * torch.exp(rnd(k) * 0.5) + rnd(k)).to(dtype)
    h = (rnd(rows, k) * 0.7 + 0.3).to(dtype)
    row = lambda n: (k,) if n == 1 else (n, k)                                                    # noqa: E731
    pw = (1 + 0.3 * rnd(k)).to(pdtype) if "p" in params else None
    gate = rnd(*row(gate_groups)).to(pdtype) if "g" in params else None
    w = rnd(*row(w_groups)).to(pdtype) if "w" in params else None
    b = rnd(*row(w_groups)).to(pdtype) if "b" in params else None
    return x, h, pw, gate, w, b, rnd(rows, k).to(dtype), rnd(rows, k).to(dtype)


def run(t, norm, post, modulation=False, scale=1.0, eps=1e-6):
    leaves = [v if v is None else v.cuda().requires_grad_() for v in t[:6]]
    x, h, pw, gate, w, b = leaves
    r, y = fn.residual_norm(x, h, gate=gate, post_weight=pw, weight=w, bias=b, eps=eps, modulation=modulation, norm=norm,
                            post=post, scale=scale)
    given = [v for v in leaves if v is not None]
    grads = torch.autograd.grad((r, y), given, (t[6].cuda(), t[7].cuda()))
    out = {"r": r, "y": y}
    out.update(zip(["d" + n for n, v in zip(NAMES, leaves) if v is not None], grads))
    return out


# widths: one value, below / at / past a pack, odd, the DiT widths, the widest rows; every number of waves and both pack counts
CASES = [
    (1, 1, "float32", "float32", "pgwb", 1, 1), (3, 7, "bfloat16", "bfloat16", "gwb", 1, 1), (5, 8, "float16", "float16", "pw", 1, 1),
    (1, 5120, "bfloat16", "bfloat16", "pw", 1, 1), (130, 1531, "float32", "float32", "pgwb", 1, 1),
    (257, 1531, "bfloat16", "float32", "pgwb", 1, 1), (64, 2048, "bfloat16", "float32", "pgwb", 2, 2),
    (63, 5120, "bfloat16", "bfloat16", "gwb", 3, 1), (40, 5123, "float16", "float16", "", 1, 1),
    (33, 2049, "bfloat16", "bfloat16", "pgw", 33, 33), (20, 8191, "float16", "float32", "pgb", 1, 4),
    (7, 16384, "bfloat16", "bfloat16", "pgwb", 1, 1), (600, 16381, "float16", "float16", "pgwb", 2, 2),
    (4, 8192, "float32", "float32", "pgwb", 2, 2), (700, 8189, "float32", "float32", "pgwb", 1, 1),
    (3000, 64, "bfloat16", "bfloat16", "pgwb", 1, 1), (2000, 513, "float32", "float32", "pgwb", 4, 4),
    (1200, 320, "float16", "float16", "pgwb", 600, 600), (1030, 4096, "bfloat16", "bfloat16", "pgwb", 1, 1),
    (2100, 250, "bfloat16", "bfloat16", "pgwb", 3, 3), (2600, 500, "float32", "float32", "pgwb", 1, 1),
    (2100, 1000, "bfloat16", "bfloat16", "pgwb", 1, 1), (1500, 2040, "float16", "float32", "pgwb", 1, 1),
    (777, 6144, "bfloat16", "bfloat16", "pgwb", 1, 1), (530, 7168, "float16", "float16", "pw", 1, 1)]


@pytest.mark.parametrize("rows,k,dtype,pdtype,params,gate_groups,w_groups", CASES)
@pytest.mark.parametrize("norm,post,modulation,scale", [("rms", "rms", False, 1.0), ("layer", None, True, 1.0),
                                                        ("rms", "layer", True, 0.5), ("layer", "rms", False, 1.0)])
def test_outputs_and_gradients(native, rows, k, dtype, pdtype, params, gate_groups, w_groups, norm, post, modulation, scale):
    if post is None:
        params = params.replace("p", "")
    t = inputs(rows, k, getattr(torch, dtype), getattr(torch, pdtype), params, gate_groups, w_groups, rows + 3 * k)
    got = run(t, norm, post, modulation, scale)
    want = formula(*t, max(gate_groups if "g" in params else 1, w_groups if set("wb") & set(params) else 1), norm, post, scale,
                   modulation)
    for name, v in got.items():
        check(v, want[name], name)


def test_rms_norm_alone(native):
    for rows, k, groups in ((1, 1, 1), (5, 4099, 1), (90, 2048, 3), (1000, 5120, 1)):
        x, _, _, _, w, b, _, dy = inputs(rows, k, torch.bfloat16, torch.bfloat16, "wb", 1, groups, rows + k)
        lx, lw, lb = (v.cuda().requires_grad_() for v in (x, w, b))
        y = fn.rms_norm(lx, lw, lb, modulation=groups > 1)
        dx, dw, db = torch.autograd.grad(y, (lx, lw, lb), dy.cuda())
        want = formula(x, None, None, None, w, b, None, dy, groups, "rms", None, modulation=groups > 1)
        for name, v in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
            check(v, want[name], name)
        with torch.no_grad():
            assert torch.equal(fn.rms_norm(lx, lw, lb, modulation=groups > 1), y)


def test_one_output_used(native):
    """A gradient of r alone, of y alone: the other's is nothing, and what has no gradient stays out."""
    t = inputs(70, 1000, torch.float32, torch.float32, "pgwb", 1, 1, 3)
    for use in ("r", "y"):
        leaves = [v.cuda().requires_grad_() for v in t[:6]]
        out = dict(zip("ry", fn.residual_norm(leaves[0], leaves[1], leaves[3], leaves[2], leaves[4], leaves[5], post="rms")))
        grads = torch.autograd.grad(out[use], leaves, t[6].cuda())
        want = formula(*t[:6], *((t[6], None) if use == "r" else (None, t[6])), 1, "rms", "rms")
        for n, v in zip(NAMES, grads):
            check(v, want["d" + n], (use, n))
    x, h = t[0].cuda(), t[1].cuda().requires_grad_()
    r, y = fn.residual_norm(x, h, post="rms")
    (dh,) = torch.autograd.grad(y, h, t[7].cuda())
    want = formula(t[0], t[1], None, None, None, None, None, t[7], 1, "rms", "rms")
    check(dh, want["dh"], "dh")


def test_rows_of_zeros_and_of_infinities(native):
    x = torch.zeros(6, 300, dtype=torch.bfloat16)
    h = torch.zeros(6, 300, dtype=torch.bfloat16)
    h[2, 7], h[3, 5], x[4] = float("inf"), float("nan"), 3.0e38
    r, y = fn.residual_norm(x.cuda(), h.cuda(), post="rms")
    r, y = r.cpu().float(), y.cpu().float()
    assert (r[[0, 1, 5]] == 0).all() and (y[[0, 1, 5]] == 0).all()               # 0 / sqrt(eps), and no NaN
    assert r[2].isnan().any() and y[3].isnan().all()                             # infinities and NaN stay in their rows
    assert torch.equal(r[4], x[4].float())


def test_strides_batches_streams_and_no_rows(native):
    t = inputs(24, 640, torch.bfloat16, torch.bfloat16, "pgwb", 2, 2, 9)
    whole = run(t, "rms", "layer")
    wide = [torch.full((24, 1280), 7.0, dtype=torch.bfloat16) for _ in range(2)]
    for v, w in zip(t[:2], wide):
        w[:, 320:960] = v
    x, h = (w.cuda()[:, 320:960].view(2, 12, 640) for w in wide)
    pw, gate, w, b = (v.cuda() for v in t[2:6])
    r, y = fn.residual_norm(x, h, gate.view(2, 1, 640), pw, w.view(2, 1, 640), b.view(2, 1, 640), post="layer")
    assert r.shape == (2, 12, 640) and torch.equal(r.view(24, 640), whole["r"]) and torch.equal(y.view(24, 640), whole["y"])
    # values across rows, one row expanded to all
    across = t[0].t().contiguous().cuda().t()
    assert torch.equal(fn.residual_norm(across, t[1].cuda(), gate, pw, w, b, post="layer")[1], whole["y"])
    r, y = fn.residual_norm(t[0][:1].cuda().expand(24, 640), t[1].cuda(), post="rms")
    assert torch.equal(y, fn.residual_norm(t[0][:1].repeat(24, 1).cuda(), t[1].cuda(), post="rms")[1])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        r, y = fn.residual_norm(t[0].cuda(), t[1].cuda(), gate, pw, w, b, post="layer")
    side.synchronize()
    assert torch.equal(r, whole["r"]) and torch.equal(y, whole["y"])
    empty = torch.empty(0, 640, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    leaf = pw.clone().requires_grad_()
    r, y = fn.residual_norm(empty, empty, post="rms", post_weight=leaf)
    (r.sum() + y.sum()).backward()
    assert r.shape == (0, 640) and empty.grad.shape == (0, 640) and (leaf.grad == 0).all()


def test_expanded_gradient_and_same_bits(native):
    """An expanded gradient is read as it lies; two passes give the same bits."""
    t = inputs(500, 2048, torch.bfloat16, torch.bfloat16, "pgwb", 1, 1, 2)
    a, b = run(t, "rms", "rms"), run(t, "rms", "rms")
    assert all(torch.equal(a[k], b[k]) for k in a)
    x, h = t[0].cuda().requires_grad_(), t[1].cuda().requires_grad_()
    r, y = fn.residual_norm(x, h, post="rms")
    row = t[7][:1].cuda()
    got = torch.autograd.grad((r, y), (x, h), (row.expand(500, 2048), row.expand(500, 2048)), retain_graph=True)
    want = torch.autograd.grad((r, y), (x, h), (row.repeat(500, 1), row.repeat(500, 1)))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_refusals(native):
    t = inputs(8, 64, torch.bfloat16, torch.bfloat16, "pgwb", 2, 2, 1)
    x, h, pw, gate, w, b = (v.cuda() for v in t[:6])
    call = fn.residual_norm
    assert call(t[0], t[1]) is None and call(x, h.float()) is None and call(x.double(), h.double()) is None
    assert call(x, h, gate.half()) is None and call(x, h, weight=w, bias=b.float()) is None
    four = gate.repeat(2, 1)
    assert call(x, h, four, weight=w, bias=b) is None                            # 4 groups and 2
    wide = torch.zeros(2, 16385, dtype=torch.bfloat16, device="cuda")
    assert call(wide, wide) is None and fn.rms_norm(wide.float()) is None
    for bad in (dict(norm="none"), dict(post="batch"), dict(post_weight=pw), dict(gate=gate[:, :63]), dict(gate=gate[:1].repeat(3, 1)),
                dict(post="rms", post_weight=gate), dict(weight=w, bias=b[0])):
        with pytest.raises(ValueError):
            call(x, h, **bad)
    with pytest.raises(ValueError):
        call(x, h[:4])
    with pytest.raises(ValueError):
        call(x, None)
    leaf = x.clone().requires_grad_()
    r, y = call(leaf, h)
    (dx,) = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
