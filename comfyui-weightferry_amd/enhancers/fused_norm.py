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
from .operands import CODES, groups_of, plain, ptr, rows_of, wants_grad

MAX_WIDTH = 32768


def _forward(x2, weight, bias, code, pcode, groups, eps, modulation, keep):
    rows, width = x2.shape
    dev = x2.device
    y = torch.empty((rows, width), dtype=x2.dtype, device=dev)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=dev) if keep else None
    if rows:
        with _native.on_device(dev):
            _native.call("wf_layer_norm", x2.data_ptr(), x2.stride(0), code, ptr(weight), ptr(bias), pcode,
                         1 if modulation else 0, rows // groups, eps, y.data_ptr(), ptr(stats), rows, width,
                         _native.stream_of(dev))
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, modulation):
        x2 = rows_of(x, x.shape[-1])
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        p = w if w is not None else b
        ctx.code, ctx.pcode = CODES[x.dtype], CODES[x.dtype if p is None else p.dtype]
        ctx.groups, ctx.modulation, ctx.shape = groups, modulation, x.shape
        ctx.wshape = None if weight is None else weight.shape
        ctx.bshape = None if bias is None else bias.shape
        y, stats = _forward(x2, w, b, ctx.code, ctx.pcode, groups, eps, modulation, True)
        ctx.save_for_backward(x2, w, stats)
        return y.view(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, w, stats = ctx.saved_tensors
        rows, width = x2.shape
        dev = x2.device
        dt = x2.dtype
        pdt = torch.float32 if ctx.pcode == 2 else dt
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        new = torch.empty if rows else torch.zeros
        dx = new((rows, width), dtype=dt, device=dev) if need_x else None
        dw = new(ctx.wshape, dtype=pdt, device=dev) if need_w else None
        db = new(ctx.bshape, dtype=pdt, device=dev) if need_b else None
        if rows:
            d2 = rows_of(dy, width)
            ws = None
            if need_w or need_b:
                need = ctypes.c_int64()
                _native.call("wf_layer_norm_bwd_workspace", rows, width, rows // ctx.groups, ctx.code, ctypes.byref(need))
                ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
            with _native.on_device(dev):
                _native.call("wf_layer_norm_bwd", x2.data_ptr(), x2.stride(0), d2.data_ptr(), d2.stride(0), ctx.code,
                             ptr(w), ctx.pcode, 1 if ctx.modulation else 0, rows // ctx.groups, stats.data_ptr(), ptr(dx),
                             ptr(dw), ptr(db), rows, width, ptr(ws), 0 if ws is None else ws.numel(),
                             _native.stream_of(dev))
        return None if dx is None else dx.view(ctx.shape), dw, db, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, modulation=False):
    """LayerNorm of ``x`` [..., K] over its last dimension, times ``weight`` plus ``bias``; with ``modulation`` times
    1 + ``weight``. ``weight`` and ``bias`` are [K], or [..., G, K] with a row for each of G groups of consecutive rows of
    ``x``; of x's type or both float32. Any strides; float16, bfloat16 and float32. None when it is not the kernel's case
    (not a plain GPU tensor, another type, K > 32768, more than 65535 groups); ValueError when the shapes do not fit
    together."""
    code = CODES.get(x.dtype)
    if code is None or not x.is_cuda or x.dim() == 0 or not plain(x, x.device):
        return None
    width = x.shape[-1]
    if not 0 < width <= MAX_WIDTH or x.numel() // width >= 1 << 31:
        return None
    rows = x.numel() // width
    groups, pcode, shared = 1, code, None
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if not plain(t, x.device) or (t.dtype != x.dtype and t.dtype != torch.float32):
            return None
        groups = groups_of(t, rows, width, what)
        if shared is not None and (shared.dtype != t.dtype or shared.numel() != t.numel()):
            raise ValueError(f"weight {shared.dtype} {tuple(shared.shape)} and bias {t.dtype} {tuple(t.shape)} differ")
        shared, pcode = t, CODES[t.dtype]
    if groups > 65535:
        return None
    if wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, groups, float(eps), bool(modulation))
    y, _ = _forward(rows_of(x, width), None if weight is None else weight.contiguous(),
                    None if bias is None else bias.contiguous(), code, pcode, groups, float(eps), modulation, False)
    return y if x.dim() == 2 else y.view(x.shape)
