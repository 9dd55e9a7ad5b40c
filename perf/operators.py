"""The operators of a training step next to the streamed, quantised inference path, as cases to be timed: LayerNorm with
its affine weights or a DiT block's modulation, forward and backward; a 16-bit linear with bias, activation and gated
residual in its epilogue, forward and backward; an AdamW step over many tensors with states in 8 or in 32 bits.

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
_LR, _BETAS, _EPS, _DECAY = 1.0e-4, (0.9, 0.999), 1.0e-8, 0.01
_BLOCK = 256                      # values that share a scale in the 8-bit states; tensors start on whole blocks


def _mod(name):
    return importlib.import_module(f"{_PKG}.enhancers.{name}")


# ------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one row of a 14B DiT's width: the head's norm on a pooled token, where the call itself counts
        {"name": "norm_1_row", "kind": "norm", "rows": 1, "width": 5120, "dtype": "bf16", "params": "affine",
         "groups": 1, "train": False},
        # the modulated norm before a 14B block's self-attention, guidance pair of 2048 tokens each
        {"name": "norm_mod_4096_rows", "kind": "norm", "rows": 4096, "width": 5120, "dtype": "bf16",
         "params": "modulation", "groups": 2, "train": False},
        # float32 training at sizes that fit nothing
        {"name": "norm_train_odd_f32", "kind": "norm", "rows": 1021, "width": 1531, "dtype": "f32", "params": "affine",
         "groups": 1, "train": True},
        # a 2B block's modulated norm in training, 896 x 1472 (2 x 2576 tokens), modulation in float32
        {"name": "norm_train_mod_5152_rows", "kind": "norm", "rows": 5152, "width": 2048, "dtype": "bf16",
         "params": "modulation_f32", "groups": 2, "train": True},
        # the largest: an affine norm over a whole video latent in training
        {"name": "norm_train_16384_rows", "kind": "norm", "rows": 16384, "width": 5120, "dtype": "bf16",
         "params": "affine", "groups": 1, "train": True},
        # one row through the first layer of a 14B block's FFN: the weight is read once
        {"name": "dense_1_row", "kind": "dense", "rows": 1, "n": 13824, "k": 5120, "dtype": "bf16", "act": "gelu_tanh",
         "bias": True, "residual": False, "groups": 0, "train": False},
        # a short text context (77 tokens) in float16, widths that fit no tile
        {"name": "dense_77_rows_f16", "kind": "dense", "rows": 77, "n": 2607, "k": 1531, "dtype": "f16", "act": "gelu",
         "bias": True, "residual": True, "groups": 0, "train": False},
        # a 4096-token latent through the FFN's first layer
        {"name": "dense_4096_rows", "kind": "dense", "rows": 4096, "n": 13824, "k": 5120, "dtype": "bf16",
         "act": "gelu_tanh", "bias": True, "residual": False, "groups": 0, "train": False},
        # training a 2B block's MLP: its second layer with the gated residual, 2 x 2576 tokens
        {"name": "dense_train_5152_rows", "kind": "dense", "rows": 5152, "n": 2048, "k": 8192, "dtype": "bf16",
         "act": "none", "bias": False, "residual": True, "groups": 2, "train": True},
        # training a 14B FFN's first layer on one 832 x 480 latent frame (1560 tokens)
        {"name": "dense_train_1560_rows", "kind": "dense", "rows": 1560, "n": 13824, "k": 5120, "dtype": "bf16",
         "act": "gelu_tanh", "bias": True, "residual": False, "groups": 0, "train": True},
        # a step of the rank-32 adapters of 28 blocks' q, k, v and output layers (224 tensors), 8-bit states
        {"name": "adamw_8bit_adapters", "kind": "adamw", "blocks": 28, "layers": 4, "m": 2048, "n": 2048, "rank": 32,
         "dtype": "f32", "bits": 8},
        # a step of a 14B FFN's own weights and biases (4 tensors), states in float32
        {"name": "adamw_32bit_ffn", "kind": "adamw", "blocks": 1, "layers": 2, "m": 13824, "n": 5120, "rank": 0,
         "dtype": "bf16", "bits": 32},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm"] * 4 + ["dense"] * 6 + ["adamw"] * 3)
    if kind == "norm":
        width = rng.choice([_log_int(rng, 64, 8192), 8 * _log_int(rng, 8, 1024), 256 * _log_int(rng, 1, 32)])
        rows = min(_log_int(rng, 1, 32768), 16384 * 5120 // width)
        params = rng.choice(["affine", "affine", "weight", "none", "modulation", "modulation_f32"])
        groups = rng.choice([1, 2, 3, 8]) if params.startswith("modulation") else 1
        return {"kind": kind, "rows": max(1, rows // groups) * groups, "width": width,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "params": params, "groups": groups,
                "train": rng.random() < 0.6}
    if kind == "dense":
        side = lambda: rng.choice([_log_int(rng, 64, 13824), 64 * _log_int(rng, 1, 216),       # noqa: E731
                                   8 * _log_int(rng, 8, 1728)])
        rows, n, k, train = _log_int(rng, 1, 16384), side(), side(), rng.random() < 0.5
        while rows * n * k * (3 if train else 1) > 1560 * 13824 * 5120 * 3:
            rows = rows // 2 + 1
        residual = rng.random() < 0.4
        groups = rng.choice([0, 1, 2]) if residual else 0
        if groups:
            rows = max(1, rows // groups) * groups
        return {"kind": kind, "rows": rows, "n": n, "k": k, "dtype": rng.choice(["bf16", "bf16", "f16"]),
                "act": rng.choice(["none", "gelu", "gelu_tanh", "silu", "relu"]), "bias": rng.random() < 0.7,
                "residual": residual, "groups": groups, "train": train}
    rank = rng.choice([0, 1, 4, 16, 32, 64])
    m, n = _log_int(rng, 256, 13824), _log_int(rng, 256, 5120)
    blocks = _log_int(rng, 1, 40) if rank else 1
    layers = rng.choice([1, 2, 4]) if rank else rng.choice([1, 2])
    while (m + n) * rank * blocks * layers > 2 * 13824 * 5120:
        blocks = blocks // 2
    return {"kind": kind, "blocks": blocks, "layers": layers, "m": m, "n": n, "rank": rank,
            "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "bits": rng.choice([8, 32])}


# ----------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)


def _shapes(case):
    """The tensors of an optimizer step: each layer's two factors of a rank-``rank`` adapter, or (rank 0) its weight and
    its bias, every second layer the other way round."""
    m, n, r = case["m"], case["n"], case["rank"]
    one = lambda a, b: [(r, b), (a, r)] if r else [(a, b), (a,)]                               # noqa: E731
    return [s for _ in range(case["blocks"]) for i in range(case["layers"])
            for s in (one(m, n) if i % 2 == 0 else one(n, m))]


def _starts(shapes):
    """Where each tensor starts in the flat states, in values, and their length: on whole blocks."""
    at, starts = 0, []
    for s in shapes:
        starts.append(at)
        at += -(-math.prod(s) // _BLOCK) * _BLOCK
    return starts, at


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "norm":
        dt, rows, width, groups = _DTYPE[case["dtype"]], case["rows"], case["width"], case["groups"]
        # a residual stream: channels of different size and mean
        x = _randn(g, rows, width, dtype=torch.float32) * torch.exp(0.5 * _randn(g, width, dtype=torch.float32))
        s = {"case": case, "x": (x + _randn(g, width, std=0.5, dtype=torch.float32)).to(dt), "w": None, "b": None}
        mod = case["params"].startswith("modulation")
        wdt = torch.float32 if case["params"] == "modulation_f32" else dt
        shape = (groups, width) if mod else (width,)
        if case["params"] != "none":
            s["w"] = _randn(g, *shape, std=0.3, mean=0.0 if mod else 1.0, dtype=wdt)
        if case["params"] not in ("none", "weight"):
            s["b"] = _randn(g, *shape, std=0.3, dtype=wdt)
        if case["train"]:
            s["dy"] = _randn(g, rows, width, std=0.01, dtype=dt)
            for t in (s["x"], s["w"], s["b"]):
                if t is not None:
                    t.requires_grad_()
        return s
    if case["kind"] == "dense":
        dt, rows, n, k = _DTYPE[case["dtype"]], case["rows"], case["n"], case["k"]
        s = {"case": case, "x": _randn(g, rows, k, dtype=dt), "w": _randn(g, n, k, std=1.5 / math.sqrt(k), dtype=dt),
             "b": _randn(g, n, std=0.2, dtype=dt) if case["bias"] else None,
             "res": _randn(g, rows, n, std=2.0, dtype=dt) if case["residual"] else None,
             "gate": _randn(g, case["groups"], n, std=0.5, dtype=dt) if case["groups"] else None}
        if case["train"]:
            s["dy"] = _randn(g, rows, n, std=0.1, dtype=dt)
            for t in (s["x"], s["w"], s["b"], s["res"], s["gate"]):
                if t is not None:
                    t.requires_grad_()
        return s
    dt, shapes = _DTYPE[case["dtype"]], _shapes(case)
    starts, total = _starts(shapes)
    flat, gflat = (torch.zeros(total, device="cuda", dtype=dt) for _ in range(2))
    view = lambda f: [f[a:a + math.prod(s)].view(s) for a, s in zip(starts, shapes)]           # noqa: E731
    s = {"case": case, "step": 100, "flat": flat, "gflat": gflat, "params": view(flat), "grads": view(gflat)}
    exp_avg, exp_avg_sq = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    for p, d, m, v in zip(s["params"], s["grads"], view(exp_avg), view(exp_avg_sq)):
        p.normal_(0.0, 0.02, generator=g)
        size = 10.0 ** (torch.rand((), generator=g, device="cuda") * 2 - 5)       # a tensor's gradients: 1e-5 .. 1e-3
        d.copy_(torch.randn(d.shape, generator=g, device="cuda") * size)
        v.copy_(torch.exp(torch.randn(v.shape, generator=g, device="cuda")) * size * size)
        m.copy_(torch.randn(m.shape, generator=g, device="cuda") * 0.3 * size)
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _encode_avg(exp_avg)
        s["v"], s["v_scale"] = _encode_sq(exp_avg_sq)
    else:
        s["m"], s["v"] = exp_avg, exp_avg_sq
    return s


# ------------------------------------------------------------------------------------------------- plain forms
# 8-bit states: m as sign(q) (q / 127)^2 scale, v as ((q / 255)^2 scale)^2, the scale a block's largest |m| or sqrt(v);
# a v that is not zero keeps a code that is not zero.
def _decode_avg(q, scale):
    c = q.view(-1, _BLOCK).float() * (1.0 / 127.0)
    return (c * c.abs() * scale[:, None]).view(-1)


def _decode_sq(q, scale):
    c = q.view(-1, _BLOCK).float() * (1.0 / 255.0)
    u = c * c * scale[:, None]
    return (u * u).view(-1)


def _encode_avg(m):
    m = m.view(-1, _BLOCK)
    scale = m.abs().amax(1)
    r = torch.where(scale > 0, scale, 1.0)[:, None]
    q = torch.round(torch.sqrt(m.abs() / r) * 127.0)
    return torch.where(m < 0, -q, q).to(torch.int8).view(-1), scale


def _encode_sq(v):
    u = torch.sqrt(v).view(-1, _BLOCK)
    scale = u.amax(1)
    r = torch.where(scale > 0, scale, 1.0)[:, None]
    q = torch.round(torch.sqrt(u / r) * 255.0)
    return torch.where(u > 0, q.clamp(min=1.0), q).to(torch.uint8).view(-1), scale


def _plain_norm(s):
    case, x = s["case"], s["x"].float()
    rows, groups, mod = case["rows"], case["groups"], case["params"].startswith("modulation")
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + 1.0e-6)
    xh = xc * rstd
    per_row = lambda t: t.float().view(groups, 1, -1)                                          # noqa: E731
    grouped = lambda t: t.view(groups, rows // groups, -1)                                     # noqa: E731
    w = None if s["w"] is None else per_row(s["w"]) + (1.0 if mod else 0.0)
    y = xh if w is None else (grouped(xh) * w).view(rows, -1)
    if s["b"] is not None:
        y = (grouped(y) + per_row(s["b"])).view(rows, -1)
    out = {"y": y.to(s["x"].dtype)}
    if case["train"]:
        dy = s["dy"].float()
        dxh = dy if w is None else (grouped(dy) * w).view(rows, -1)
        dx = rstd * (dxh - dxh.mean(1, keepdim=True) - xh * (dxh * xh).mean(1, keepdim=True))
        out["dx"] = dx.to(s["x"].dtype)
        if s["w"] is not None:
            out["dw"] = grouped(dy * xh).sum(1).view(s["w"].shape).to(s["w"].dtype)
        if s["b"] is not None:
            out["db"] = grouped(dy).sum(1).view(s["b"].shape).to(s["b"].dtype)
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
    sig = torch.sigmoid(h)
    return sig * (1.0 + h * (1.0 - sig)) if act == "silu" else (h > 0).float()


def _plain_dense(s):
    case, dt = s["case"], s["x"].dtype
    rows, n, act, groups = case["rows"], case["n"], case["act"], max(1, case["groups"])
    x, w = s["x"].float(), s["w"].float()
    grouped = lambda t: t.view(groups, rows // groups, n)                                      # noqa: E731
    h = x @ w.T
    if s["b"] is not None:
        h = h + s["b"].float()
    a = _act(h, act)
    gate = None if s["gate"] is None else s["gate"].float()[:, None, :]
    y = a if gate is None else (grouped(a) * gate).view(rows, n)
    if s["res"] is not None:
        y = s["res"].float() + y
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        da = dy if gate is None else (grouped(dy) * gate).view(rows, n)
        dh = da if act == "none" else da * _act_slope(h, act)
        out["dx"], out["dw"] = (dh @ w).to(dt), (dh.T @ x).to(dt)
        if s["b"] is not None:
            out["db"] = dh.sum(0).to(dt)
        if s["res"] is not None:
            out["dres"] = s["dy"]
        if gate is not None:
            out["dgate"] = grouped(dy * a).sum(1).to(dt)
    return out


def _plain_adamw(s):
    b1, b2 = _BETAS
    step, eight = s["step"], s["case"]["bits"] == 8
    g, p = s["gflat"].float(), s["flat"].float()
    m = _decode_avg(s["m"], s["m_scale"]) if eight else s["m"]
    v = _decode_sq(s["v"], s["v_scale"]) if eight else s["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    denom = torch.sqrt(v) * (1.0 / math.sqrt(1 - b2 ** step)) + _EPS
    s["flat"].copy_(p * (1 - _LR * _DECAY) - m / denom * (_LR / (1 - b1 ** step)))
    if eight:
        s["m"], s["m_scale"] = _encode_avg(m)
        s["v"], s["v_scale"] = _encode_sq(v)
        m, v = _decode_avg(s["m"], s["m_scale"]), _decode_sq(s["v"], s["v_scale"])
    else:
        s["m"], s["v"] = m, v
    return {"p": s["flat"], "m": m, "v": v}


# --------------------------------------------------------------------------------------------------- one pass
def _own_norm(s):
    y = _mod("fused_norm").layer_norm(s["x"], s["w"], s["b"], eps=1.0e-6,
                                      modulation=s["case"]["params"].startswith("modulation"))
    out = {"y": y}
    if s["case"]["train"]:
        names = [k for k in ("x", "w", "b") if s[k] is not None]
        out.update(zip(["d" + k for k in names], torch.autograd.grad(y, [s[k] for k in names], s["dy"])))
    return out


def _own_dense(s):
    act = s["case"]["act"]
    y = _mod("fused_dense").dense(s["x"], s["w"], s["b"], act=None if act == "none" else act, residual=s["res"],
                                  gate=s["gate"])
    out = {"y": y}
    if s["case"]["train"]:
        names = [k for k in ("x", "w", "b", "res", "gate") if s[k] is not None]
        out.update(zip(["d" + k for k in names], torch.autograd.grad(y, [s[k] for k in names], s["dy"])))
    return out


def _own_adamw(s):
    adamw = _mod("fused_adamw")
    state = adamw.AdamWState(s["m"], s["v"], s.get("m_scale"), s.get("v_scale"))
    adamw.adamw_step(s["params"], s["grads"], state, s["step"], lr=_LR, betas=_BETAS, eps=_EPS, weight_decay=_DECAY)
    m, v = state.values()
    return {"p": s["flat"], "m": m, "v": v}


def run(s):
    kind = s["case"]["kind"]
    if kind == "adamw":
        s["step"] += 1
        if own:
            return _own_adamw(s)
        with torch.no_grad():
            return _plain_adamw(s)
    if own:
        return (_own_norm if kind == "norm" else _own_dense)(s)
    with torch.no_grad():
        return (_plain_norm if kind == "norm" else _plain_dense)(s)


# ------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "norm":
        size, values = _SIZE[case["dtype"]], case["rows"] * case["width"]
        wsize = 4 if case["params"] == "modulation_f32" else size
        n_params = {"none": 0, "weight": 1}.get(case["params"], 2)
        params = n_params * case["groups"] * case["width"] * wsize
        if not case["train"]:
            return {"bytes": 2 * values * size + params, "flops": 8 * values}
        return {"bytes": 4 * values * size + 2 * params, "flops": 22 * values}     # x, dy in; y, dx out
    if case["kind"] == "dense":
        rows, n, k, size = case["rows"], case["n"], case["k"], _SIZE[case["dtype"]]
        vectors = n * (int(case["bias"]) + case["groups"])
        once = rows * k + n * k + rows * n * (2 if case["residual"] else 1) + vectors
        if not case["train"]:
            return {"bytes": once * size, "flops": 2 * rows * n * k}
        back = rows * n + rows * k + n * k + vectors                               # dy in; dx, dw and the rest out
        return {"bytes": (once + back) * size, "flops": 6 * rows * n * k}
    values, size = sum(math.prod(s) for s in _shapes(case)), _SIZE[case["dtype"]]
    state = 16 if case["bits"] == 32 else 4 + 8 + 16 / _BLOCK      # read and written; from 8 bits the values too
    return {"bytes": int(values * (3 * size + state)), "flops": 15 * values}


# ------------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["kind"] == "norm":
        x, rows, groups = d["x"], case["rows"], case["groups"]
        which = torch.arange(rows, device="cuda") // (rows // groups)
        var, mean = torch.var_mean(x, dim=1, keepdim=True, correction=0)
        xh = (x - mean) / torch.sqrt(var + 1.0e-6)
        w = None
        if "w" in d:
            w = d["w"].view(groups, -1)[which] + (1 if case["params"].startswith("modulation") else 0)
        y = xh if w is None else xh * w
        out = {"y": y + d["b"].view(groups, -1)[which] if "b" in d else y}
        if case["train"]:
            dxh = d["dy"] if w is None else d["dy"] * w
            inner = dxh - dxh.mean(1, keepdim=True) - xh * (dxh * xh).mean(1, keepdim=True)
            out["dx"] = inner / torch.sqrt(var + 1.0e-6)
            zero = torch.zeros(groups, case["width"], device="cuda", dtype=torch.float64)
            if "w" in d:
                out["dw"] = zero.index_add(0, which, d["dy"] * xh).view(d["w"].shape)
            if "b" in d:
                out["db"] = zero.index_add(0, which, d["dy"]).view(d["b"].shape)
        return out
    if case["kind"] == "dense":
        rows, groups, act = case["rows"], max(1, case["groups"]), case["act"]
        which = torch.arange(rows, device="cuda") // (rows // groups)
        h = torch.matmul(d["x"], d["w"].t())
        if "b" in d:
            h += d["b"]
        if act == "gelu":                                   # h Phi(h), and Phi(h) + h phi(h)
            phi = torch.special.ndtr(h)
            a, slope = h * phi, phi + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)
        elif act == "gelu_tanh":                            # h sigmoid(2 z), z = sqrt(2 / pi) (h + 0.044715 h^3)
            z = math.sqrt(2 / math.pi) * (h + 0.044715 * h ** 3)
            sig = 1 / (1 + torch.exp(-2 * z))
            a = h * sig
            slope = sig + h * 2 * sig * (1 - sig) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * h ** 2)
        elif act == "silu":
            sig = 1 / (1 + torch.exp(-h))
            a, slope = h * sig, sig + h * sig * (1 - sig)
        elif act == "relu":
            a, slope = torch.where(h > 0, h, 0.0), torch.where(h > 0, 1.0, 0.0).double()
        else:
            a, slope = h, torch.ones_like(h)
        gate = d["gate"][which] if "gate" in d else torch.ones_like(h)
        out = {"y": gate * a + d.get("res", 0)}
        if case["train"]:
            dh = d["dy"] * gate * slope
            out["dx"], out["dw"] = torch.matmul(dh, d["w"]), torch.matmul(dh.t(), d["x"])
            if "b" in d:
                out["db"] = dh.sum(0)
            if "res" in d:
                out["dres"] = d["dy"]
            if "gate" in d:
                zero = torch.zeros(groups, case["n"], device="cuda", dtype=torch.float64)
                out["dgate"] = zero.index_add(0, which, d["dy"] * a)
        return out
    # one AdamW step; 8-bit states are read from their codes, and the new ones are rounded to codes of the same kind
    step, (b1, b2), eight = s["step"] + 1, _BETAS, case["bits"] == 8
    p, g, m, v = d["flat"], d["gflat"], d["m"], d["v"]
    if eight:
        m = torch.sign(m) * (m / 127) ** 2 * d["m_scale"].repeat_interleave(_BLOCK)
        v = ((v / 255) ** 2 * d["v_scale"].repeat_interleave(_BLOCK)) ** 2
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    update = (m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + _EPS)
    p = p - _LR * _DECAY * p - _LR * update
    if eight:
        top = m.abs().view(-1, _BLOCK).amax(1).repeat_interleave(_BLOCK)
        m = torch.sign(m) * (torch.round(127 * torch.sqrt(m.abs() / top.clamp(min=1e-300))) / 127) ** 2 * top
        u = torch.sqrt(v)
        top = u.view(-1, _BLOCK).amax(1).repeat_interleave(_BLOCK)
        q = torch.round(255 * torch.sqrt(u / top.clamp(min=1e-300)))
        v = ((torch.where(u > 0, q.clamp(min=1), q) / 255) ** 2 * top) ** 2
    return {"p": p, "m": m, "v": v}
