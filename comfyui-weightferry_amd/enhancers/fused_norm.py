"""LayerNorm with affine weights or a DiT block's modulation in one kernel, forward and backward (wf_layer_norm,
wf_layer_norm_bwd).

``layer_norm(x, weight, bias)`` is ``torch.nn.functional.layer_norm`` over the last dimension; with ``modulation=True`` it
is the block's ``LayerNorm(x) * (1 + scale) + shift``, ``scale`` and ``shift`` one row per batch entry (any number of
consecutive row groups), computed and rounded once instead of three times through memory. Gradients of ``x``, ``weight``
and ``bias`` come from one pass over ``x`` and ``dy``. The reference has no training path; its int8 quantiser's LayerNorm
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
