"""The norms around a gated residual in float64, outputs and gradients from the formula, each with what float32 arithmetic in any
reasonable order may be off by (tests/test_gpu_block_norm.py; tests/test_block_norm_formula.py checks the formula itself).

Where the bounds come from. A row's sum takes at most 32 additions in a lane, 6 over a wave and 16 over a team, so a mean is off by at
most 2^-18 of the mean magnitude and a reciprocal root by 2^-18 of itself; a normalised value z = (t - m) / d then by 2^-18 (A +
|z|), A = mean|t| / d (no mean is taken off for RMS: A = 0). An error e(t) in t moves z by (e(t) + mean e(t) + |z| mean(|z| e(t))) / d.
The rest is products and sums of these, 2^-23 of the magnitude for each rounding or two. Sums over rows add at most a few
hundred float32 terms one after another: 2^-16 of the sum of magnitudes."""
import torch

SUM, STEP = 2.0 ** -18, 2.0 ** -23


def formula(x, h, pw, gate, w, b, dr, dy, groups, norm, post, scale=1.0, modulation=False, eps=1e-6):
    """{name: (value, bound)} of r, y, dx, dh, dpw, dgate, dw, db; None for what is not there."""
    rows, k = x.shape
    to = lambda t: None if t is None else t.double().cpu()                                        # noqa: E731
    x, h, pw, gate, w, b, dr, dy = map(to, (x, h, pw, gate, w, b, dr, dy))
    which = torch.arange(rows) // (rows // groups)
    per = lambda t, plus=0.0: None if t is None else (t.reshape(-1, k) + plus).expand(             # noqa: E731
        max(groups, t.numel() // k), k)[which]
    mean = lambda t: t.mean(1, keepdim=True)                                                      # noqa: E731

    def unit(t, e, kind):
        m = mean(t) if kind == "layer" else torch.zeros(rows, 1, dtype=torch.float64)
        d = torch.sqrt(mean((t - m) ** 2) + eps)
        z = (t - m) / d
        a = mean(t.abs()) / d if kind == "layer" else 0.0
        moved = mean(z.abs() * e) / d
        return z, d, SUM * (a + z.abs()) + (e + mean(e)) / d + z.abs() * moved, SUM + moved

    def through(g, eg, z, ez, d, ed, kind):
        m1, m2 = mean(g) if kind == "layer" else 0.0, mean(g * z)
        e1 = SUM * mean(g.abs()) + mean(eg) if kind == "layer" else 0.0
        e2 = SUM * mean((g * z).abs()) + mean(g.abs() * ez + eg * z.abs())
        inner = g - m1 - z * m2
        e = eg + e1 + z.abs() * e2 + ez * abs(m2) + 4 * STEP * (g.abs() + abs(m1) + (z * m2).abs())
        return inner / d, (e + ed * inner.abs()) / d

    one = torch.ones(rows, k, dtype=torch.float64)
    pw_, gate_, w_ = (one if t is None else t for t in (per(pw), per(gate), per(w, 1.0 if modulation else 0.0)))
    gp = pw_ * gate_
    out = {}
    if h is None:
        hh, ehh = torch.zeros_like(x), torch.zeros_like(x)
    elif post is None:
        hh, ehh = h, torch.zeros_like(h)
    else:
        hh, h_d, ehh, h_ed = unit(h, torch.zeros_like(h), post)
    r = scale * x + gp * hh
    er = gp.abs() * ehh + 2 * STEP * ((scale * x).abs() + (gp * hh).abs())
    rh, r_d, erh, r_ed = unit(r, er, norm)
    y = rh * w_ + (0.0 if b is None else per(b))
    out["r"] = (r, er) if h is not None else None
    out["y"] = (y, w_.abs() * erh + STEP * ((rh * w_).abs() + (0.0 if b is None else per(b).abs())))
    if dr is None and dy is None:
        return out
    dr, dy = (torch.zeros_like(x) if t is None else t for t in (dr, dy))
    g = dy * w_
    back, eback = through(g, STEP * g.abs(), rh, erh, r_d, r_ed, norm)
    dR, edR = dr + back, eback + STEP * (dr.abs() + back.abs())
    t, et = dR * gp, gp.abs() * edR + 2 * STEP * (dR * gp).abs()
    out["dx"] = (scale * dR, abs(scale) * edR + STEP * (scale * dR).abs())
    if h is not None:
        out["dh"] = (t, et) if post is None else through(t, et, hh, ehh, h_d, h_ed, post)

    def fold(v, e, like):
        n = like.numel() // k
        zero = torch.zeros(n, k, dtype=torch.float64)
        at = which if n == groups else torch.zeros_like(which)
        add = lambda q: zero.index_add(0, at, q).reshape(like.shape)                              # noqa: E731
        return add(v), add(e + 2.0 ** -16 * v.abs())

    if gate is not None:
        out["dgate"] = fold(dR * pw_ * hh, pw_.abs() * (edR * hh.abs() + dR.abs() * ehh), gate)
    if pw is not None:
        out["dpw"] = fold(dR * gate_ * hh, gate_.abs() * (edR * hh.abs() + dR.abs() * ehh), pw)
    if w is not None:
        out["dw"] = fold(dy * rh, dy.abs() * erh, w)
    if b is not None:
        out["db"] = fold(dy, torch.zeros_like(dy), b)
    return out
