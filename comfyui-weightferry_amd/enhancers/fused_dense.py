"""A linear layer on 16-bit weights with everything around the product in its epilogue, forward and backward (wf_dense,
wf_dense_grad):

    y = residual + gate * act(x @ weight.T + bias)

is what a DiT block does around each of its products (GELU after the MLP's first layer, the gated residual after an output
projection); here the sums stay in float32 from the matrix unit to the one rounding of ``y``. The backward pass is one
element-wise kernel (dh, and the gradients of bias and gate) and two products on the transposed operands.
The reference leaves these layers to ComfyUI's ``torch.nn.functional.linear``; its own epilogues are the int8 path's
(enhancers/fused_int8.py:191-268)."""
import ctypes

import torch

from .. import _native
from .operands import CODES, groups_of, plain, ptr, rows_of, wants_grad

ACTIVATIONS = {None: 0, "gelu": 1, "gelu_tanh": 2, "silu": 3, "relu": 4}
MAX_ROWS, MAX_K = 1 << 24, 1 << 20


def _product(x, x_row, x_col, w, w_row, w_col, code, m, n, k, out, bias=None, act=0, gate=None, groups=1, resid=None,
             h=None):
    """out [m, n] by wf_dense; an operand is a tensor with the strides (in values) of its rows and of k."""
    dev = out.device
    need = ctypes.c_int64()
    xp, wp = x.data_ptr(), w.data_ptr()
    _native.call("wf_dense_workspace", xp, x_row, x_col, wp, w_row, w_col, code, m, n, k, ctypes.byref(need))
    ws = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
    with _native.on_device(dev):
        _native.call("wf_dense", xp, x_row, x_col, wp, w_row, w_col, code, m, n, k, ptr(bias),
                     code if bias is None else CODES[bias.dtype], act, ptr(gate),
                     code if gate is None else CODES[gate.dtype], m // groups, ptr(resid),
                     0 if resid is None else resid.stride(0), out.data_ptr(), ptr(h), ptr(ws), need.value,
                     _native.stream_of(dev))
    return out


def _matrix(w):
    """A weight as it can be read: any strides that are not negative (an expanded one is made real)."""
    return w if w.stride(0) and w.stride(1) else w.contiguous()


def _forward(x2, weight, bias, act, resid, gate, groups, keep):
    rows, k = x2.shape
    n = weight.shape[0]
    y = torch.empty((rows, n), dtype=x2.dtype, device=x2.device)
    h = torch.empty_like(y) if keep else None
    if rows and n:
        _product(x2, x2.stride(0), 1, weight, weight.stride(0), weight.stride(1), CODES[x2.dtype], rows, n, k, y, bias,
                 act, gate, groups, resid, h)
    return y, h


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, gate, act, groups):
        x2, w = rows_of(x, x.shape[-1]), _matrix(weight)
        n = w.shape[0]
        b = None if bias is None else bias.contiguous()
        g = None if gate is None else gate.contiguous()
        r = None if residual is None else rows_of(residual, n)
        keep = act != 0 or ctx.needs_input_grad[4]       # the activation's slope and the gate's gradient read h
        y, h = _forward(x2, w, b, act, r, g, groups, keep)
        ctx.save_for_backward(x2, w, h, g)
        ctx.act, ctx.groups, ctx.shape = act, groups, x.shape
        ctx.bias = None if bias is None else (bias.shape, bias.dtype)
        ctx.gate = None if gate is None else gate.shape
        return y.view(*x.shape[:-1], n)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, w, h, gate = ctx.saved_tensors
        rows, k = x2.shape
        n, dt, dev, code = w.shape[0], x2.dtype, x2.device, CODES[x2.dtype]
        need_x, need_w, need_b, need_r, need_g = ctx.needs_input_grad[:5]
        none = rows == 0 or n == 0
        new = torch.zeros if none else torch.empty
        dx = new((rows, k), dtype=dt, device=dev) if need_x else None
        dw = new((n, k), dtype=dt, device=dev) if need_w else None
        db = new(ctx.bias[0], dtype=ctx.bias[1], device=dev) if need_b else None
        dg = new(ctx.gate, dtype=gate.dtype, device=dev) if need_g else None
        if not none:
            dh = d2 = rows_of(dy, n)
            changed = (ctx.act != 0 or gate is not None) and (need_x or need_w)
            if changed:
                dh = torch.empty((rows, n), dtype=dt, device=dev)
            if changed or need_b or need_g:
                ws = None
                if need_b or need_g:
                    need = ctypes.c_int64()
                    _native.call("wf_dense_grad_workspace", rows, n, rows // ctx.groups, ctypes.byref(need))
                    ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
                with _native.on_device(dev):
                    _native.call("wf_dense_grad", d2.data_ptr(), d2.stride(0), ptr(h), code, ctx.act, ptr(gate),
                                 code if gate is None else CODES[gate.dtype], rows // ctx.groups,
                                 dh.data_ptr() if changed else None, ptr(db),
                                 code if db is None else CODES[db.dtype], ptr(dg), rows, n, ptr(ws),
                                 0 if ws is None else ws.numel(), _native.stream_of(dev))
            if need_x:
                _product(dh, dh.stride(0), 1, w, w.stride(1), w.stride(0), code, rows, k, n, dx)
            if need_w:
                _product(dh, 1, dh.stride(0), x2, 1, x2.stride(0), code, n, k, rows, dw)
        return (None if dx is None else dx.view(ctx.shape), dw, db, dy if need_r else None, dg, None, None)


def dense(x, weight, bias=None, act=None, residual=None, gate=None):
    """``residual + gate * act(x @ weight.T + bias)`` for ``x`` [..., K] and ``weight`` [N, K], bfloat16 or float16, any
    strides. ``act``: None, "gelu", "gelu_tanh", "silu" or "relu". ``bias`` [N]; ``residual`` [..., N]; ``gate`` [N], or
    [..., G, N] with a row for each of G groups of consecutive rows; bias and gate of x's type or float32. Records gradients
    of all five. None when it is not the kernel's case (not plain GPU tensors, other types, K above 2^20, rows or N above
    2^24, or above 2^20 with gradients); ValueError when the shapes do not fit together or ``act`` is unknown."""
    if act not in ACTIVATIONS:
        raise ValueError(f"act={act!r}: one of {', '.join(map(repr, ACTIVATIONS))}")
    dt, dev = x.dtype, x.device
    if (dt != torch.bfloat16 and dt != torch.float16) or not x.is_cuda or x.dim() == 0 or not plain(x, dev):
        return None
    if weight.dtype != dt or not plain(weight, dev):
        return None
    k = x.shape[-1]
    if weight.dim() != 2 or weight.shape[1] != k or k == 0:
        raise ValueError(f"weight has shape {tuple(weight.shape)}: [N, {k}] fits x {tuple(x.shape)}")
    n, rows = weight.shape[0], x.numel() // k
    groups = 1
    if bias is not None:
        if (bias.dtype != dt and bias.dtype != torch.float32) or not plain(bias, dev):
            return None
        if bias.numel() != n:
            raise ValueError(f"bias has shape {tuple(bias.shape)}: {n} values are wanted")
    if residual is not None:
        if residual.dtype != dt or not plain(residual, dev):
            return None
        if residual.shape[:-1] != x.shape[:-1] or residual.shape[-1] != n:
            raise ValueError(f"residual has shape {tuple(residual.shape)}: {(*x.shape[:-1], n)} is wanted")
    if gate is not None:
        if (gate.dtype != dt and gate.dtype != torch.float32) or not plain(gate, dev):
            return None
        groups = groups_of(gate, rows, n, "gate") if n else 1
    grads = wants_grad(x, weight, bias, residual, gate)
    if max(rows, n) > (MAX_K if grads else MAX_ROWS) or k > MAX_K or groups > 65535:
        return None
    code = ACTIVATIONS[act]
    if grads:
        return _Dense.apply(x, weight, bias, residual, gate, code, groups)
    y, _ = _forward(rows_of(x, k), _matrix(weight), None if bias is None else bias.contiguous(), code,
                    None if residual is None else rows_of(residual, n), None if gate is None else gate.contiguous(),
                    groups, False)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], n)
