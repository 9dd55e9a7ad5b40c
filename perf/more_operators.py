"""Operators of a gated block's training step, next to those of perf/operators.py, as cases to be timed: the norms before
and after a block with its gate and residual, forward and backward; a gated feed-forward layer (both projections, the
activation and the product), forward and backward; an update orthogonalised by Newton-Schulz products, by itself and as a
whole optimizer step over many matrices.

``listed()`` gives the fixed cases, ``draw(rng)`` another one of the same ranges, ``prepare(case, seed)`` what a program
holds before the call, ``run(state)`` one pass (in elementary torch operations in float32, or, with ``own`` set, through
the framework's entry points), ``work(case)`` the bytes and operations it cannot do without, ``exact(case, seed)`` the
outputs from the definition in float64."""
import importlib
import math

import torch

own = False

_PKG = "comfyui-weightferry_amd"
_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1.0e-6                                       # of the norms
_LR, _MOMENTUM, _DECAY = 1.0e-2, 0.95, 0.1          # of the optimizer step
_COEFFICIENTS, _STEPS, _TINY = (3.4445, -4.7750, 2.0315), 5, 1.0e-7


def _mod(name):
    return importlib.import_module(f"{_PKG}.enhancers.{name}")


# ------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one row of a 14B DiT's width between two RMS-normed sub-layers: the call itself counts
        {"name": "block_norm_1_row", "kind": "norm", "rows": 1, "width": 5120, "dtype": "bf16", "post": "rms", "norm": "rms",
         "gate": 0, "params": "weight", "groups": 1, "train": False},
        # between a 14B block's attention and its FFN: gated residual and the modulated LayerNorm, a guidance pair of 2048 tokens
        {"name": "block_norm_mod_4096_rows", "kind": "norm", "rows": 4096, "width": 5120, "dtype": "bf16", "post": "none",
         "norm": "layer", "gate": 1, "params": "modulation", "groups": 2, "train": False},
        # float32 training at sizes that fit nothing
        {"name": "block_norm_train_odd_f32", "kind": "norm", "rows": 1021, "width": 1531, "dtype": "f32", "post": "layer",
         "norm": "rms", "gate": 1, "params": "affine", "groups": 1, "train": True},
        # a 2B block with norms on both sides in training, 2 x 2576 tokens, gate and modulation one row a sample
        {"name": "block_norm_train_5152_rows", "kind": "norm", "rows": 5152, "width": 2048, "dtype": "bf16", "post": "rms",
         "norm": "rms", "gate": 1, "params": "modulation", "groups": 2, "train": True},
        # the largest: the same over a whole video latent at a 14B width
        {"name": "block_norm_train_16384_rows", "kind": "norm", "rows": 16384, "width": 5120, "dtype": "bf16", "post": "rms",
         "norm": "rms", "gate": 1, "params": "weight", "groups": 1, "train": True},
        # one row through a 14B block's gated FFN: both weights are read once
        {"name": "gated_1_row", "kind": "gated", "rows": 1, "n": 13824, "k": 5120, "dtype": "bf16", "act": "silu",
         "bias": False, "train": False},
        # a short text context (77 tokens) in float16, widths that fit no tile
        {"name": "gated_77_rows_f16", "kind": "gated", "rows": 77, "n": 2607, "k": 1531, "dtype": "f16", "act": "gelu",
         "bias": True, "train": False},
        # a 4096-token latent
        {"name": "gated_4096_rows", "kind": "gated", "rows": 4096, "n": 13824, "k": 5120, "dtype": "bf16", "act": "silu",
         "bias": False, "train": False},
        # training on one 832 x 480 latent frame (1560 tokens)
        {"name": "gated_train_1560_rows", "kind": "gated", "rows": 1560, "n": 13824, "k": 5120, "dtype": "bf16",
         "act": "gelu_tanh", "bias": True, "train": True},
        # a step of the rank-32 adapters of 28 blocks' q, k, v and output layers: 112 pairs of factors
        {"name": "muon_adapters", "kind": "muon", "count": 112, "rows": 32, "cols": 2048, "both": True, "dtype": "bf16"},
        # the direction alone, of matrices whose sides fit nothing (in bfloat16, as a gradient comes)
        {"name": "orthogonalize_odd", "kind": "orthogonalize", "count": 3, "rows": 1531, "cols": 1021, "both": False,
         "dtype": "bf16"},
        # a step of a 14B FFN's two weights
        {"name": "muon_ffn", "kind": "muon", "count": 1, "rows": 13824, "cols": 5120, "both": True, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm"] * 4 + ["gated"] * 4 + ["muon"] * 3 + ["orthogonalize"])
    if kind == "norm":
        width = rng.choice([_log_int(rng, 64, 8192), 8 * _log_int(rng, 8, 1024), 256 * _log_int(rng, 1, 32)])
        rows = min(_log_int(rng, 1, 32768), 16384 * 5120 // width)
        gate, params = rng.choice([0, 1, 1]), rng.choice(["none", "weight", "affine", "modulation", "modulation_f32"])
        groups = rng.choice([1, 2, 3, 8]) if gate or params.startswith("modulation") else 1
        return {"kind": kind, "rows": max(1, rows // groups) * groups, "width": width,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "post": rng.choice(["none", "rms", "rms", "layer"]),
                "norm": rng.choice(["rms", "layer"]), "gate": gate, "params": params, "groups": groups,
                "train": rng.random() < 0.6}
    side = lambda lo: rng.choice([_log_int(rng, lo, 13824), 64 * _log_int(rng, 1, 216),           # noqa: E731
                                  8 * _log_int(rng, 8, 1728)])
    if kind == "gated":
        rows, n, k, train = _log_int(rng, 1, 16384), side(64), side(64), rng.random() < 0.5
        while rows * n * k * (3 if train else 1) > 1560 * 13824 * 5120 * 3:
            rows = rows // 2 + 1
        return {"kind": kind, "rows": rows, "n": n, "k": k, "dtype": rng.choice(["bf16", "bf16", "f16"]),
                "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu", "none"]), "bias": rng.random() < 0.5,
                "train": train}
    rows, cols, both = side(16), side(16), rng.random() < 0.4
    if rng.random() < 0.3:
        rows = rng.choice([8, 16, 32, 64])                        # an adapter's factor
    count = _log_int(rng, 1, 128)
    most = _muon_flops(13824, 5120) * 2
    while min(rows, cols) > 5120 or (1 + both) * _muon_flops(rows, cols) > most:
        rows, cols = -(-rows * 3 // 4), -(-cols * 3 // 4)
    while count > 1 and (count * (1 + both) * _muon_flops(rows, cols) > most
                         or count * (1 + both) * rows * cols > 2 * 13824 * 5120):
        count = count // 2
    return {"kind": kind, "count": count, "rows": rows, "cols": cols, "both": both,
            "dtype": "bf16" if kind == "orthogonalize" else rng.choice(["bf16", "bf16", "f16"])}


# ----------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)


def _gradient(g, count, rows, cols):
    """Gradients as a matrix's training gives them: a few strong directions whose sizes fall off, in noise."""
    rank = max(1, min(32, rows // 2, cols // 2))
    left, right = (torch.randn(count, *s, generator=g, device="cuda") for s in ((rows, rank), (rank, cols)))
    fall = 1.0 / torch.arange(1, rank + 1, device="cuda")
    strong = torch.bmm(left * fall, right)
    return (strong + 0.1 * torch.randn(count, rows, cols, generator=g, device="cuda")) * 1.0e-3


def _shapes(case):
    r, c = case["rows"], case["cols"]
    return [(r, c), (c, r)] if case["both"] else [(r, c)]


def prepare(case, seed):
    g = _gen(seed)
    dt = _DTYPE[case["dtype"]]
    if case["kind"] == "norm":
        rows, width, groups = case["rows"], case["width"], case["groups"]
        # a residual stream, channels of different size and mean, and a sub-layer's output
        x = _randn(g, rows, width, dtype=torch.float32) * torch.exp(0.5 * _randn(g, width, dtype=torch.float32))
        s = {"case": case, "x": (x + _randn(g, width, std=0.5, dtype=torch.float32)).to(dt),
             "h": _randn(g, rows, width, std=0.7, mean=0.1, dtype=dt), "pw": None, "gate": None, "w": None, "b": None}
        mod = case["params"].startswith("modulation")
        wdt = torch.float32 if case["params"] == "modulation_f32" else dt
        shape = (groups, width) if mod else (width,)
        if case["post"] != "none":
            s["pw"] = _randn(g, width, std=0.3, mean=1.0, dtype=dt)
        if case["gate"]:
            s["gate"] = _randn(g, groups, width, std=0.5, dtype=dt)
        if case["params"] != "none":
            s["w"] = _randn(g, *shape, std=0.3, mean=0.0 if mod else 1.0, dtype=wdt)
        if case["params"] not in ("none", "weight"):
            s["b"] = _randn(g, *shape, std=0.3, dtype=wdt)
        if case["train"]:
            s["dr"], s["dy"] = (_randn(g, rows, width, std=0.01, dtype=dt) for _ in range(2))
            for t in (s["x"], s["h"], s["pw"], s["gate"], s["w"], s["b"]):
                if t is not None:
                    t.requires_grad_()
        return s
    if case["kind"] == "gated":
        rows, n, k = case["rows"], case["n"], case["k"]
        s = {"case": case, "x": _randn(g, rows, k, dtype=dt), "w": _randn(g, 2 * n, k, std=1.5 / math.sqrt(k), dtype=dt),
             "b": _randn(g, 2 * n, std=0.2, dtype=dt) if case["bias"] else None}
        if case["train"]:
            s["dy"] = _randn(g, rows, n, std=0.1, dtype=dt)
            for t in (s["x"], s["w"], s["b"]):
                if t is not None:
                    t.requires_grad_()
        return s
    s = {"case": case, "grads": [_gradient(g, case["count"], *shape).to(dt) for shape in _shapes(case)]}
    if case["kind"] == "muon":
        s["params"] = [_randn(g, case["count"], *shape, std=0.02, dtype=dt) for shape in _shapes(case)]
        s["momenta"] = [_gradient(g, case["count"], *shape) for shape in _shapes(case)]
        s["lists"] = [[m for t in s[k] for m in t.unbind(0)] for k in ("params", "grads", "momenta")]
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    case, x, h = s["case"], s["x"].float(), s["h"].float()
    dt, rows, width, groups = s["x"].dtype, case["rows"], case["width"], case["groups"]
    mod, train = case["params"].startswith("modulation"), case["train"]
    # a parameter as one row for each group, and a matrix as its groups of rows
    per_row = lambda t: None if t is None else t.float().view(-1, 1, width)                       # noqa: E731
    grouped = lambda t: t.view(groups, rows // groups, width)                                     # noqa: E731

    def unit(t, kind):
        if kind == "layer":
            t = t - t.mean(-1, keepdim=True)
        rstd = torch.rsqrt((t * t).mean(-1, keepdim=True) + _EPS)
        return t * rstd, rstd

    def unit_back(d, t, rstd, kind):
        inner = d - t * (d * t).mean(-1, keepdim=True)
        if kind == "layer":
            inner = inner - d.mean(-1, keepdim=True)
        return inner * rstd

    def summed(t, like):
        t = t.sum(1)
        return (t if t.shape[0] == like.numel() // width else t.sum(0)).view(like.shape).to(like.dtype)

    pw, gate, w, b = (per_row(s[k]) for k in ("pw", "gate", "w", "b"))
    if mod:
        w = 1.0 + w
    hh, h_rstd = unit(h, case["post"]) if case["post"] != "none" else (h, None)
    hh = grouped(hh)
    branch = hh if pw is None else hh * pw
    r = grouped(x) + (branch if gate is None else branch * gate)
    rh, r_rstd = unit(r, case["norm"])
    y = rh if w is None else rh * w
    if b is not None:
        y = y + b
    out = {"r": r.view(rows, width).to(dt), "y": y.view(rows, width).to(dt)}
    if train:
        dy = grouped(s["dy"].float())
        dr = grouped(s["dr"].float()) + unit_back(dy if w is None else dy * w, rh, r_rstd, case["norm"])
        dbranch = dr if gate is None else dr * gate
        dh = dbranch if pw is None else dbranch * pw
        if case["post"] != "none":
            dh = unit_back(dh, hh, h_rstd.view(groups, -1, 1), case["post"])
        out["dx"], out["dh"] = dr.view(rows, width).to(dt), dh.reshape(rows, width).to(dt)
        if pw is not None:
            out["dpw"] = summed(dbranch * hh, s["pw"])
        if gate is not None:
            out["dgate"] = summed(dr * branch, s["gate"])
        if w is not None:
            out["dw"] = summed(dy * rh, s["w"])
        if b is not None:
            out["db"] = summed(dy, s["b"])
    return out


def _act(h, act):
    if act == "gelu":
        return 0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * h * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (h + 0.044715 * h * h * h)))
    if act == "silu":
        return h * torch.sigmoid(h)
    return torch.clamp(h, min=0.0) if act == "relu" else h


def _act_slope(h, act):
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (h + 0.044715 * h * h * h))
        return 0.5 * (1.0 + t) + 0.5 * h * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * h * h)
    if act == "silu":
        sig = torch.sigmoid(h)
        return sig * (1.0 + h * (1.0 - sig))
    return (h > 0).float() if act == "relu" else torch.ones_like(h)


def _plain_gated(s):
    case, dt, n = s["case"], s["x"].dtype, s["case"]["n"]
    x, w = s["x"].float(), s["w"].float()
    h = x @ w.T
    if s["b"] is not None:
        h = h + s["b"].float()
    g, u = h[:, :n], h[:, n:]
    a = _act(g, case["act"])
    out = {"y": (a * u).to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        dh = torch.cat((dy * u * _act_slope(g, case["act"]), dy * a), 1)
        out["dx"], out["dw"] = (dh @ w).to(dt), (dh.T @ x).to(dt)
        if s["b"] is not None:
            out["db"] = dh.sum(0).to(dt)
    return out


def _plain_orthogonal(u):
    """u / |u| with each of its singular values put through the polynomial a v + b v^3 + c v^5, five times."""
    a, b, c = _COEFFICIENTS
    x = u / u.square().sum((1, 2), keepdim=True).sqrt().clamp(min=_TINY)
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    for _ in range(_STEPS):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.transpose(1, 2).contiguous() if tall else x


def _plain_muon(s):
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        g = g.float()
        m.copy_(_MOMENTUM * m + (1 - _MOMENTUM) * g)
        step = _plain_orthogonal(_MOMENTUM * m + (1 - _MOMENTUM) * g) * (_LR * 0.2 * math.sqrt(max(p.shape[1:])))
        p.copy_(p.float() * (1 - _LR * _DECAY) - step)
    return {"p": s["params"], "m": s["momenta"]}


# --------------------------------------------------------------------------------------------------- one pass
def _own_norm(s):
    case = s["case"]
    r, y = _mod("fused_norm").residual_norm(s["x"], s["h"], gate=s["gate"], post_weight=s["pw"], weight=s["w"], bias=s["b"],
                                            eps=_EPS, modulation=case["params"].startswith("modulation"), norm=case["norm"],
                                            post=None if case["post"] == "none" else case["post"])
    out = {"r": r, "y": y}
    if case["train"]:
        names = [k for k in ("x", "h", "pw", "gate", "w", "b") if s[k] is not None]
        out.update(zip(["d" + k for k in names], torch.autograd.grad((r, y), [s[k] for k in names], (s["dr"], s["dy"]))))
    return out


def _own_gated(s):
    act = s["case"]["act"]
    y = _mod("fused_dense").gated_dense(s["x"], s["w"], s["b"], act=None if act == "none" else act)
    out = {"y": y}
    if s["case"]["train"]:
        names = [k for k in ("x", "w", "b") if s[k] is not None]
        out.update(zip(["d" + k for k in names], torch.autograd.grad(y, [s[k] for k in names], s["dy"])))
    return out


def run(s):
    kind = s["case"]["kind"]
    if own:
        if kind == "norm":
            return _own_norm(s)
        if kind == "gated":
            return _own_gated(s)
        muon = _mod("fused_muon")
        if kind == "orthogonalize":
            return [muon.orthogonalize(g) for g in s["grads"]]
        muon.muon_step(*s["lists"], lr=_LR, momentum=_MOMENTUM, weight_decay=_DECAY, adjust="rms")
        return {"p": s["params"], "m": s["momenta"]}
    with torch.no_grad():
        if kind == "norm":
            return _plain_norm(s)
        if kind == "gated":
            return _plain_gated(s)
        if kind == "muon":
            return _plain_muon(s)
        return [_plain_orthogonal(g.float()).to(g.dtype) for g in s["grads"]]


# ------------------------------------------------------------------------------------------------------- work
def _muon_flops(rows, cols):
    """Of one matrix: a step's Gram matrix and its square are symmetric, so half of each is enough."""
    m, n = min(rows, cols), max(rows, cols)
    return _STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["kind"] == "norm":
        values, width = case["rows"] * case["width"], case["width"]
        n_params = {"none": 0, "weight": 1}.get(case["params"], 2)
        per = case["groups"] if case["params"].startswith("modulation") else 1
        params = n_params * per * width * (4 if case["params"] == "modulation_f32" else size)
        params += ((case["post"] != "none") + case["gate"] * case["groups"]) * width * size
        if not case["train"]:
            return {"bytes": 4 * values * size + params, "flops": 16 * values}      # x, h in; r, y out
        return {"bytes": 8 * values * size + 2 * params, "flops": 50 * values}      # and dr, dy in; dx, dh out
    if case["kind"] == "gated":
        rows, n, k = case["rows"], case["n"], case["k"]
        once = rows * k + 2 * n * k + rows * n + 2 * n * int(case["bias"])
        if not case["train"]:
            return {"bytes": once * size, "flops": 4 * rows * n * k}
        return {"bytes": 2 * once * size, "flops": 12 * rows * n * k}               # dy in; dx, dw, db out
    matrices = case["count"] * len(_shapes(case))
    values = matrices * case["rows"] * case["cols"]
    flops = matrices * _muon_flops(case["rows"], case["cols"])
    if case["kind"] == "orthogonalize":
        return {"bytes": 2 * values * size, "flops": flops}
    return {"bytes": values * (3 * size + 8), "flops": flops + 8 * values}          # p and m in and out, g in


# ------------------------------------------------------------------------------------------------------ exact
def _exact_norm(case, d):
    rows, width, groups = case["rows"], case["width"], case["groups"]
    which = torch.arange(rows, device="cuda") // (rows // groups)

    def spread(name, plus=0.0):                             # a parameter's row for each row of x
        if name not in d:
            return None
        t = d[name].view(-1, width) + plus
        return t[which] if t.shape[0] == groups else t.expand(rows, width)

    def fold(t, name):                                      # its gradient
        n = d[name].numel() // width
        zero = torch.zeros(n, width, device="cuda", dtype=torch.float64)
        return zero.index_add(0, which if n == groups else torch.zeros_like(which), t).view(d[name].shape)

    def moments(t, kind):                                   # what the norm takes off, and what it divides by
        mean = torch.mean(t, 1, keepdim=True) if kind == "layer" else torch.zeros(rows, 1, device="cuda", dtype=torch.float64)
        return mean, torch.sqrt(torch.sum((t - mean) ** 2, 1, keepdim=True) / width + _EPS)

    def through(dt, t, mean, div, kind):                    # the gradient of (t - mean) / div
        z = (t - mean) / div
        out = dt - z * torch.sum(dt * z, 1, keepdim=True) / width
        if kind == "layer":
            out = out - torch.sum(dt, 1, keepdim=True) / width
        return out / div

    one = torch.ones((), device="cuda", dtype=torch.float64)
    pw, gate, b = spread("pw"), spread("gate"), spread("b")
    w = spread("w", 1.0 if case["params"].startswith("modulation") else 0.0)
    pw, gate, w = (one if t is None else t for t in (pw, gate, w))
    post = case["post"]
    h_mean, h_div = moments(d["h"], post) if post != "none" else (0.0, 1.0)
    hh = (d["h"] - h_mean) / h_div
    r = d["x"] + gate * pw * hh
    r_mean, r_div = moments(r, case["norm"])
    rh = (r - r_mean) / r_div
    y = rh * w
    out = {"r": r, "y": y if b is None else y + b}
    if case["train"]:
        dr = d["dr"] + through(d["dy"] * w, r, r_mean, r_div, case["norm"])
        dhh = dr * gate * pw
        out["dx"] = dr
        out["dh"] = dhh if post == "none" else through(dhh, d["h"], h_mean, h_div, post)
        if "pw" in d:
            out["dpw"] = fold(dr * gate * hh, "pw")
        if "gate" in d:
            out["dgate"] = fold(dr * pw * hh, "gate")
        if "w" in d:
            out["dw"] = fold(d["dy"] * rh, "w")
        if "b" in d:
            out["db"] = fold(d["dy"], "b")
    return out


def _exact_gated(case, d):
    n, act = case["n"], case["act"]
    wg, wu = d["w"][:n], d["w"][n:]
    g, u = torch.matmul(d["x"], wg.t()), torch.matmul(d["x"], wu.t())
    if "b" in d:
        g, u = g + d["b"][:n], u + d["b"][n:]
    if act == "gelu":                                       # g Phi(g), and Phi(g) + g phi(g)
        phi = torch.special.ndtr(g)
        a, slope = g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    elif act == "gelu_tanh":                                # g sigmoid(2 z), z = sqrt(2 / pi) (g + 0.044715 g^3)
        z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        sig = 1 / (1 + torch.exp(-2 * z))
        a, slope = g * sig, sig + g * 2 * sig * (1 - sig) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g ** 2)
    elif act == "silu":
        sig = 1 / (1 + torch.exp(-g))
        a, slope = g * sig, sig + g * sig * (1 - sig)
    elif act == "relu":
        a, slope = torch.where(g > 0, g, 0.0), torch.where(g > 0, 1.0, 0.0).double()
    else:
        a, slope = g, torch.ones_like(g)
    out = {"y": a * u}
    if case["train"]:
        dg, du = d["dy"] * u * slope, d["dy"] * a
        out["dx"] = torch.matmul(dg, wg) + torch.matmul(du, wu)
        out["dw"] = torch.cat((torch.matmul(dg.t(), d["x"]), torch.matmul(du.t(), d["x"])))
        if "b" in d:
            out["db"] = torch.cat((dg.sum(0), du.sum(0)))
    return out


def _exact_orthogonal(u):
    """One matrix at a time, on the Gram matrix of its shorter side: with q = a + b gram + c gram^2 a step is gram <- q gram q,
    and the product of the steps' q times u / |u| is the result."""
    a, b, c = _COEFFICIENTS
    out = torch.empty_like(u)
    for i in range(u.shape[0]):
        x = u[i] / torch.linalg.norm(u[i]).clamp(min=_TINY)
        wide = x.shape[0] <= x.shape[1]
        gram = torch.mm(x, x.t()) if wide else torch.mm(x.t(), x)
        eye = torch.eye(gram.shape[0], device="cuda", dtype=torch.float64)
        total = eye
        for _ in range(_STEPS):
            q = a * eye + b * gram + c * torch.mm(gram, gram)
            total, gram = torch.mm(q, total), torch.mm(q, torch.mm(gram, q))
        out[i] = torch.mm(total, x) if wide else torch.mm(x, total)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["kind"] == "norm":
        return _exact_norm(case, d)
    if case["kind"] == "gated":
        return _exact_gated(case, d)
    grads = [g.double() for g in s["grads"]]
    if case["kind"] == "orthogonalize":
        return [_exact_orthogonal(g) for g in grads]
    out = {"p": [], "m": []}
    for p, g, m in zip(s["params"], grads, s["momenta"]):
        m = m.double() + (1 - _MOMENTUM) * (g - m.double())
        ahead = m + (1 - _MOMENTUM) * (g - m)
        size = 0.2 * math.sqrt(max(p.shape[1], p.shape[2]))
        out["m"].append(m)
        out["p"].append(p.double() - _LR * _DECAY * p.double() - _LR * size * _exact_orthogonal(ahead))
    return out
