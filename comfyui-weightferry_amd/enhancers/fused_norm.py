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
_POSTS = {None: 0, **NORMS}
MAX_ROW_BYTES = 32768


def _block(*how):
    """A call's kinds, types and groups as the library takes them: its address, and what keeps that valid."""
    q = _native.BlockNorm(*how)
    return ctypes.addressof(q), q


_blocks = Sizes(_block)


def _ask_block(how, rows, width, sums):
    need, q = ctypes.c_int64(), _blocks(how)             # (q is held until the call is done: another thread may clear the cache)
    _native.call("wf_block_norm_bwd_workspace", q[0], rows, width, sums, ctypes.byref(need))
    return need.value


_bytes_block = Sizes(_ask_block)


def _launch_block(x2, h2, post_weight, gate, weight, bias, how, stats):
    """(r, or None without a branch, and y)"""
    rows, width = x2.shape
    dev = x2.device
    # (the like of a contiguous tensor takes two thirds of the time)
    y = torch.empty_like(x2) if x2.is_contiguous() else torch.empty((rows, width), dtype=x2.dtype, device=dev)
    r = None if h2 is None else torch.empty_like(y)
    if rows:
        q = _blocks(how)
        with _native.on_device(dev):
            rc = _native.lib().wf_block_norm_fwd(q[0], x2.data_ptr(), x2.stride(0), ptr(h2), 0 if h2 is None else h2.stride(0),
                                                 ptr(post_weight), ptr(gate), ptr(weight), ptr(bias), ptr(r), y.data_ptr(),
                                                 ptr(stats), rows, width, _native.stream_of(dev))
        if rc:
            _native.must(rc, "wf_block_norm_fwd")
    return r, y


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, post_weight, gate, weight, bias, how):
        ctx.set_materialize_grads(False)
        shape = x.shape
        width = shape[-1]
        x2, h2 = rows_of(x, width), None if branch is None else rows_of(branch, width)
        pw, g, w = whole(post_weight), whole(gate), whole(weight)
        stats = torch.empty((x2.shape[0], 4), dtype=torch.float32, device=x2.device)
        r, y = _launch_block(x2, h2, pw, g, w, whole(bias), how, stats)
        ctx.how = how, shape, tuple(None if t is None else (t.shape, t.dtype) for t in (post_weight, gate, weight, bias))
        ctx.save_for_backward(x2, h2, pw, g, w, stats)
        if len(shape) == 2:
            return y if r is None else (r, y)
        return y.view(shape) if r is None else (r.view(shape), y.view(shape))

    @once
    def backward(ctx, *grads):
        dr, dy = grads if len(grads) == 2 else (None, grads[0])
        if dr is None and dy is None:
            return (None,) * 7
        x2, h2, post_weight, gate, weight, stats = ctx.saved_tensors
        how, shape, specs = ctx.how
        need = ctx.needs_input_grad
        rows, width = x2.shape
        dt, dev = x2.dtype, x2.device
        dr = None if dr is None else rows_of(gradient(dr), width)
        dy = None if dy is None else rows_of(gradient(dy), width)
        new = torch.empty if rows else torch.zeros
        dx = new(shape, dtype=dt, device=dev) if need[0] else None
        dh = new(shape, dtype=dt, device=dev) if need[1] else None
        dparams, sums = [], 0
        for want, spec in zip(need[2:6], specs):
            dparams.append(new(spec[0], dtype=spec[1], device=dev) if want else None)
            sums += want
        if rows:
            size = _bytes_block((how, rows, width, sums)) if sums else 0
            ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
            q = _blocks(how)
            with _native.on_device(dev):
                rc = _native.lib().wf_block_norm_bwd(
                    q[0], x2.data_ptr(), x2.stride(0), ptr(h2), 0 if h2 is None else h2.stride(0), ptr(post_weight), ptr(gate),
                    ptr(weight), ptr(dr), 0 if dr is None else dr.stride(0), ptr(dy), 0 if dy is None else dy.stride(0),
                    stats.data_ptr(), ptr(dx), ptr(dh), *map(ptr, dparams), rows, width, ptr(ws), size, _native.stream_of(dev))
            if rc:
                _native.must(rc, "wf_block_norm_bwd")
        return (dx, dh, *dparams, None)


_apply_block = applier(_BlockNorm)


def _block_norm(x, branch, gate, post_weight, weight, bias, eps, modulation, norm, post, scale):
    norm_code, post_code = NORMS.get(norm), _POSTS.get(post)
    if norm_code is None or post_code is None:
        raise ValueError(f"norm={norm!r}, post={post!r}: one of {', '.join(map(repr, NORMS))}; post may be None")
    dt, dev, shape = x.dtype, x.device, x.shape
    code = CODES.get(dt)
    if code is None or not shape or dev.type != "cuda" or not plain(dev, x, branch, gate, post_weight, weight, bias):
        return None
    if branch is not None:
        if branch.shape != shape:
            raise ValueError(f"branch has shape {tuple(branch.shape)}: {tuple(shape)} is wanted")
        if branch.dtype != dt:
            return None
    width = shape[-1]
    if not 0 < width * (4 if code == 2 else 2) <= MAX_ROW_BYTES:
        return None
    dims = len(shape)
    rows = shape[0] if dims == 2 else x.numel() // width
    gate_code = post_weight_code = weight_code = code
    gate_groups = weight_groups = 1
    if post_weight is not None:
        if not post_code:
            raise ValueError("post_weight without the norm that it scales (post)")
        if post_weight.shape != (width,):
            raise ValueError(f"post_weight has shape {tuple(post_weight.shape)}: ({width},) is wanted")
        post_weight_code = CODES.get(post_weight.dtype)
    if gate is not None:
        gate_groups, gate_code = groups_of(gate, rows, width, "gate"), CODES.get(gate.dtype)
    if weight is not None:
        weight_groups, weight_code = groups_of(weight, rows, width, "weight"), CODES.get(weight.dtype)
    if bias is not None:
        groups = groups_of(bias, rows, width, "bias")
        if weight is not None:
            if groups != weight_groups:
                raise ValueError(f"weight {tuple(weight.shape)} and bias {tuple(bias.shape)} differ")
            if bias.dtype != weight.dtype:
                return None
        weight_groups, weight_code = groups, CODES.get(bias.dtype)
    for c in (post_weight_code, gate_code, weight_code):
        if c != code and c != 2:
            return None
    groups = gate_groups if gate_groups > weight_groups else weight_groups
    if groups > 1 and (gate_groups not in (1, groups) or weight_groups not in (1, groups) or groups > 65535) or rows >= 1 << 31:
        return None
    how = (code, post_code, norm_code, 1 if modulation else 0, post_weight_code, gate_code, weight_code, float(scale), float(eps),
           groups, gate_groups, weight_groups)
    if wants_grad(x, branch, post_weight, gate, weight, bias):
        return _apply_block(x, branch, post_weight, gate, weight, bias, how)
    r, y = _launch_block(rows_of(x, width), None if branch is None else rows_of(branch, width), whole(post_weight), whole(gate),
                         whole(weight), whole(bias), how, None)
    if dims == 2:
        return y if r is None else (r, y)
    return y.view(shape) if r is None else (r.view(shape), y.view(shape))


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
