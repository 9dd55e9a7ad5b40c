"""LayerNorm with affine weights or a DiT block's modulation in one kernel, forward and backward (wf_layer_norm,
wf_layer_norm_bwd), and the norms around a block's gated residual in another (wf_block_norm_fwd, wf_block_norm_bwd).

``layer_norm(x, weight, bias)`` is ``torch.nn.functional.layer_norm`` over the last dimension; with ``modulation=True`` it
is the block's ``LayerNorm(x) * (1 + scale) + shift``, ``scale`` and ``shift`` one row per batch entry (any number of
consecutive row groups), computed and rounded once instead of three times through memory. Gradients of ``x``, ``weight``
and ``bias`` come from one pass over ``x`` and ``dy``.

``residual_norm(x, branch, ...)`` is what lies between two sub-layers: the norm after one (none, RMS or LayerNorm), the gated
residual, and the norm before the next (RMS or LayerNorm, affine or modulated); ``rms_norm(x, weight, bias)`` the second
norm alone. The reference has no training path; its int8 quantiser's LayerNorm
(enhancers/fused_kernels.py:84-136) feeds int8 products only."""
import ctypes

import torch

from .. import _native
from .operands import CODES, Sizes, applier, gradient, groups_of, once, plain, ptr, rows_of, wants_grad, whole

MAX_WIDTH = 32768


def _ask(rows, width, rows_per_group, code):
    need = ctypes.c_int64()
    _native.call("wf_layer_norm_bwd_workspace", rows, width, rows_per_group, code, ctypes.byref(need))
    return need.value


_bytes = Sizes(_ask)


def _launch(x2, w, b, code, pcode, groups, eps, modulation, stats):
    rows, width = x2.shape
    dev = x2.device
    y = torch.empty((rows, width), dtype=x2.dtype, device=dev)
    if rows:
        with _native.on_device(dev):
            rc = _native.lib().wf_layer_norm(x2.data_ptr(), x2.stride(0), code, ptr(w), ptr(b), pcode, modulation,
                                             rows // groups, eps, y.data_ptr(), ptr(stats), rows, width,
                                             _native.stream_of(dev))
        if rc:
            _native.must(rc, "wf_layer_norm")
    return y


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, how):
        code, pcode, groups, eps, modulation = how
        x2, w = rows_of(x, x.shape[-1]), whole(weight)
        stats = torch.empty((x2.shape[0], 2), dtype=torch.float32, device=x2.device)
        y = _launch(x2, w, whole(bias), code, pcode, groups, eps, modulation, stats)
        ctx.how = (code, pcode, groups, modulation, x.shape, None if weight is None else weight.shape,
                   None if bias is None else bias.shape)
        ctx.save_for_backward(x2, w, stats)
        return y if x.dim() == 2 else y.view(x.shape)

    @once
    def backward(ctx, dy):
        dy = gradient(dy)
        x2, w, stats = ctx.saved_tensors
        code, pcode, groups, modulation, shape, wshape, bshape = ctx.how
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        rows, width = x2.shape
        dev, dt = x2.device, x2.dtype
        pdt = torch.float32 if pcode == 2 else dt
        new = torch.empty if rows else torch.zeros
        dx = (torch.empty_like(dy) if dy.is_contiguous() else new(shape, dtype=dt, device=dev)) if need_x else None
        dw = new(wshape, dtype=pdt, device=dev) if need_w else None
        db = new(bshape, dtype=pdt, device=dev) if need_b else None
        if rows:
            d2, ws, need = rows_of(dy, width), None, 0
            if need_w or need_b:
                need = _bytes((rows, width, rows // groups, code))
                ws = torch.empty(need, dtype=torch.uint8, device=dev)
            with _native.on_device(dev):
                rc = _native.lib().wf_layer_norm_bwd(x2.data_ptr(), x2.stride(0), d2.data_ptr(), d2.stride(0), code, ptr(w),
                                                     pcode, modulation, rows // groups, stats.data_ptr(), ptr(dx), ptr(dw),
                                                     ptr(db), rows, width, ptr(ws), need, _native.stream_of(dev))
            if rc:
                _native.must(rc, "wf_layer_norm_bwd")
        return dx, dw, db, None


_apply = applier(_LayerNorm)


def layer_norm(x, weight=None, bias=None, eps=1e-5, modulation=False):
    """LayerNorm of ``x`` [..., K] over its last dimension, times ``weight`` plus ``bias``; with ``modulation`` times
    1 + ``weight``. ``weight`` and ``bias`` are [K], or [..., G, K] with a row for each of G groups of consecutive rows of
    ``x``; of x's type or both float32. Any strides; float16, bfloat16 and float32. None when it is not the kernel's case
    (not a plain GPU tensor, another type, K > 32768, more than 65535 groups); ValueError when the shapes do not fit
    together."""
    dt, dev = x.dtype, x.device
    pcode = code = CODES.get(dt)
    dims = x.dim()
    if code is None or dims == 0 or dev.type != "cuda" or not plain(dev, x, weight, bias):
        return None
    width = x.shape[-1]
    if not 0 < width <= MAX_WIDTH:
        return None
    rows = x.shape[0] if dims == 2 else x.numel() // width
    groups, first = 1, None
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.dtype != dt:
            if t.dtype != torch.float32:
                return None
            pcode = 2
        groups = groups_of(t, rows, width, what)
        if first is not None and first.numel() != t.numel():
            raise ValueError(f"weight {tuple(first.shape)} and bias {tuple(t.shape)} differ")
        if first is not None and first.dtype != t.dtype:
            return None
        first = t
    if groups > 65535 or rows >= 1 << 31:
        return None
    if wants_grad(x, weight, bias):
        return _apply(x, weight, bias, (code, pcode, groups, float(eps), 1 if modulation else 0))
    y = _launch(rows_of(x, width), whole(weight), whole(bias), code, pcode, groups, eps, 1 if modulation else 0, None)
    return y if dims == 2 else y.view(x.shape)


# ------------------------------------------------------------------------- the norms around a gated residual
NORMS = {"rms": 1, "layer": 2}
MAX_ROW_BYTES = 32768


def _ask_block(code, rows, width, groups, sums):
    q, need = _native.BlockNorm(dt=code, norm=1, groups=groups), ctypes.c_int64()
    _native.call("wf_block_norm_bwd_workspace", ctypes.byref(q), rows, width, sums, ctypes.byref(need))
    return need.value


_bytes_block = Sizes(_ask_block)


def _block(how, post_weight, gate, weight, bias):
    """The call's parameters as the library takes them."""
    code, post, norm, plus_one, scale, eps, groups, gate_groups, weight_groups = how
    wcode = code if weight is None and bias is None else CODES[(bias if weight is None else weight).dtype]
    return _native.BlockNorm(code, post, norm, plus_one, code if post_weight is None else CODES[post_weight.dtype],
                             code if gate is None else CODES[gate.dtype], wcode, scale, eps, groups, gate_groups,
                             weight_groups, ptr(post_weight), ptr(gate), ptr(weight), ptr(bias))


def _launch_block(x2, h2, params, how, stats):
    """(r, or None without a branch, and y)"""
    rows, width = x2.shape
    dev = x2.device
    y = torch.empty((rows, width), dtype=x2.dtype, device=dev)
    r = None if h2 is None else torch.empty_like(y)
    if rows:
        with _native.on_device(dev):
            rc = _native.lib().wf_block_norm_fwd(ctypes.byref(_block(how, *params)), x2.data_ptr(), x2.stride(0), ptr(h2),
                                                 0 if h2 is None else h2.stride(0), ptr(r), y.data_ptr(), ptr(stats), rows,
                                                 width, _native.stream_of(dev))
        if rc:
            _native.must(rc, "wf_block_norm_fwd")
    return r, y


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, post_weight, gate, weight, bias, how):
        ctx.set_materialize_grads(False)
        width = x.shape[-1]
        x2, h2 = rows_of(x, width), None if branch is None else rows_of(branch, width)
        params = whole(post_weight), whole(gate), whole(weight), whole(bias)
        stats = torch.empty((x2.shape[0], 4), dtype=torch.float32, device=x2.device)
        r, y = _launch_block(x2, h2, params, how, stats)
        ctx.how = how, x.shape, tuple(None if t is None else (t.shape, t.dtype) for t in (post_weight, gate, weight, bias))
        ctx.save_for_backward(x2, h2, *params[:3], stats)
        return y.view(x.shape) if r is None else (r.view(x.shape), y.view(x.shape))

    @once
    def backward(ctx, *grads):
        grads = [None if d is None else gradient(d) for d in grads]
        dr, dy = grads if len(grads) == 2 else (None, grads[0])
        if dr is None and dy is None:
            return (None,) * 7
        x2, h2, post_weight, gate, weight, stats = ctx.saved_tensors
        how, shape, specs = ctx.how
        need = ctx.needs_input_grad
        rows, width = x2.shape
        dev = x2.device
        new = torch.empty if rows else torch.zeros
        dx = new(shape, dtype=x2.dtype, device=dev) if need[0] else None
        dh = new(shape, dtype=x2.dtype, device=dev) if need[1] else None
        dparams = [new(spec[0], dtype=spec[1], device=dev) if want else None for want, spec in zip(need[2:6], specs)]
        if rows:
            q = _block(how, post_weight, gate, weight, None)
            if specs[3] is not None:
                q.weight_dt = CODES[specs[3][1]]
            d2 = [None if d is None else rows_of(d, width) for d in (dr, dy)]
            sums = sum(t is not None for t in dparams)
            size = _bytes_block((how[0], rows, width, how[6], sums)) if sums else 0
            ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
            with _native.on_device(dev):
                rc = _native.lib().wf_block_norm_bwd(
                    ctypes.byref(q), x2.data_ptr(), x2.stride(0), ptr(h2), 0 if h2 is None else h2.stride(0), ptr(d2[0]),
                    0 if d2[0] is None else d2[0].stride(0), ptr(d2[1]), 0 if d2[1] is None else d2[1].stride(0),
                    stats.data_ptr(), ptr(dx), ptr(dh), *map(ptr, dparams), rows, width, ptr(ws), size,
                    _native.stream_of(dev))
            if rc:
                _native.must(rc, "wf_block_norm_bwd")
        return (dx, dh, *dparams, None)


_apply_block = applier(_BlockNorm)


def _block_norm(x, branch, gate, post_weight, weight, bias, eps, modulation, norm, post, scale):
    if norm not in NORMS or (post is not None and post not in NORMS):
        raise ValueError(f"norm={norm!r}, post={post!r}: one of {', '.join(map(repr, NORMS))}; post may be None")
    if post is None and post_weight is not None:
        raise ValueError("post_weight without the norm that it scales (post)")
    dt, dev, dims = x.dtype, x.device, x.dim()
    code = CODES.get(dt)
    if code is None or dims == 0 or dev.type != "cuda" or not plain(dev, x, branch, gate, post_weight, weight, bias):
        return None
    if branch is not None:
        if branch.shape != x.shape:
            raise ValueError(f"branch has shape {tuple(branch.shape)}: {tuple(x.shape)} is wanted")
        if branch.dtype != dt:
            return None
    width = x.shape[-1]
    if not 0 < width * x.element_size() <= MAX_ROW_BYTES:
        return None
    rows = x.numel() // width
    if any(t is not None and t.dtype != dt and t.dtype != torch.float32 for t in (gate, post_weight, weight, bias)):
        return None
    if post_weight is not None and tuple(post_weight.shape) != (width,):
        raise ValueError(f"post_weight has shape {tuple(post_weight.shape)}: ({width},) is wanted")
    gate_groups = 1 if gate is None else groups_of(gate, rows, width, "gate")
    weight_groups = 1
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            weight_groups = groups_of(t, rows, width, what)
    if weight is not None and bias is not None:
        if weight.numel() != bias.numel():
            raise ValueError(f"weight {tuple(weight.shape)} and bias {tuple(bias.shape)} differ")
        if weight.dtype != bias.dtype:
            return None
    groups = max(gate_groups, weight_groups)
    if min(gate_groups, weight_groups) not in (1, groups) or groups > 65535 or rows >= 1 << 31:
        return None
    how = (code, 0 if post is None else NORMS[post], NORMS[norm], 1 if modulation else 0, float(scale), float(eps), groups,
           gate_groups, weight_groups)
    if wants_grad(x, branch, post_weight, gate, weight, bias):
        return _apply_block(x, branch, post_weight, gate, weight, bias, how)
    r, y = _launch_block(rows_of(x, width), None if branch is None else rows_of(branch, width),
                         (whole(post_weight), whole(gate), whole(weight), whole(bias)), how, None)
    return y.view(x.shape) if r is None else (r.view(x.shape), y.view(x.shape))


def residual_norm(x, branch, gate=None, post_weight=None, weight=None, bias=None, eps=1e-6, modulation=False, norm="rms",
                  post=None, scale=1.0):
    """``(r, y)`` with r = ``scale`` x + ``gate`` * ``post_weight`` * post(branch) and y = norm(r) * ``weight`` + ``bias`` (with
    ``modulation`` times 1 + ``weight``): a sub-layer's output ``branch`` [..., K], like ``x``, is normed, gated and added to the
    residual stream, and normed for the next sub-layer, in one pass. ``norm``: "rms" (t / sqrt(mean t^2 + eps)) or "layer";
    ``post``: the same, or None for the branch as it is. ``post_weight`` [K]; ``gate``, and ``weight`` and ``bias``: [K], or
    [..., G, K] with a row for each of G groups of consecutive rows. Parameters of x's type or float32. y comes from r before
    its rounding. Records gradients of all six tensors. None when it is not the kernel's case (not plain GPU tensors, other types,
    rows of more than 32768 bytes, gate and weight in different numbers of groups, more than 65535); ValueError when the
    shapes do not fit together."""
    if branch is None:
        raise ValueError("no branch: rms_norm and layer_norm are the norm alone")
    return _block_norm(x, branch, gate, post_weight, weight, bias, eps, modulation, norm, post, scale)


def rms_norm(x, weight=None, bias=None, eps=1e-6, modulation=False):
    """``x / sqrt(mean x^2 + eps) * weight + bias`` over the last dimension, with ``modulation`` times 1 + ``weight``: what
    ``layer_norm`` takes and gives, for rows of at most 32768 bytes."""
    return _block_norm(x, None, None, None, weight, bias, eps, modulation, "rms", None, 1.0)
