"""A linear layer on 16-bit weights with everything around the product in its epilogue, forward and backward (wf_dense,
wf_dense_bwd):

    y = residual + gate * act(x @ weight.T + bias)

is what a DiT block does around each of its products (GELU after the MLP's first layer, the gated residual after an output
projection); here the sums stay in float32 from the matrix unit to the one rounding of ``y``. The backward pass is one
element-wise kernel (dh, and the gradients of bias and gate) and two products on the transposed operands, which are loaded
as they lie. The reference leaves these layers to ComfyUI's ``torch.nn.functional.linear``; its own epilogues are the int8
path's (enhancers/fused_int8.py:191-268)."""
import ctypes

import torch

from .. import _native
from .operands import CODES, Sizes, applier, gradient, groups_of, once, plain, ptr, rows_of, wants_grad, whole

ACTIVATIONS = {None: 0, "gelu": 1, "gelu_tanh": 2, "silu": 3, "relu": 4}
MAX_ROWS, MAX_K = 1 << 24, 1 << 20


def _ask(*key):
    need = ctypes.c_int64()
    _native.call("wf_dense_workspace", *key, ctypes.byref(need))
    return need.value


def _ask_bwd(*key):
    need = ctypes.c_int64()
    _native.call("wf_dense_bwd_workspace", *key, ctypes.byref(need))
    return need.value


# (of an address the library's answer depends on its alignment to 16 bytes only, so that stands for it in the key)
_bytes, _bytes_bwd = Sizes(_ask), Sizes(_ask_bwd)


def _matrix(w):
    """A weight as it can be read: any strides that are not zero (an expanded one is made real)."""
    return w if w.stride(0) and w.stride(1) else w.contiguous()


def _launch(x2, w, b, code, act, resid, gate, groups, keep):
    """(y, the pre-activations or None)"""
    rows, k = x2.shape
    n, dev = w.shape[0], x2.device
    y = torch.empty((rows, n), dtype=x2.dtype, device=dev)
    h = torch.empty_like(y) if keep else None
    if rows and n:
        xp, wp, xr = x2.data_ptr(), w.data_ptr(), x2.stride(0)
        w_row, w_col = w.stride()
        epilogue = (1 if act else 0) | (2 if keep else 0) | (0 if gate is None and resid is None else 4)
        need = _bytes((xp & 15, xr, 1, wp & 15, w_row, w_col, code, rows, n, k, epilogue))
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        with _native.on_device(dev):
            rc = _native.lib().wf_dense(xp, xr, 1, wp, w_row, w_col, code, rows, n, k, ptr(b),
                                        code if b is None else CODES[b.dtype], act, ptr(gate),
                                        code if gate is None else CODES[gate.dtype], rows // groups, ptr(resid),
                                        0 if resid is None else resid.stride(0), y.data_ptr(), ptr(h), ptr(ws), need,
                                        _native.stream_of(dev))
        if rc:
            _native.must(rc, "wf_dense")
    return y, h


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, gate, how):
        code, act, groups = how
        x2, w, g = rows_of(x, x.shape[-1]), _matrix(weight), whole(gate)
        n = w.shape[0]
        keep = act != 0 or ctx.needs_input_grad[4]       # the activation's slope and the gate's gradient read h
        y, h = _launch(x2, w, whole(bias), code, act, None if residual is None else rows_of(residual, n), g, groups, keep)
        ctx.save_for_backward(x2, w, h, g)
        ctx.how = (code, act, groups, x.shape, None if bias is None else (bias.shape, bias.dtype),
                   None if gate is None else gate.shape)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], n)

    @once
    def backward(ctx, dy):
        dy = gradient(dy)
        x2, w, h, gate = ctx.saved_tensors
        code, act, groups, shape, bias, gshape = ctx.how
        need_x, need_w, need_b, need_r, need_g = ctx.needs_input_grad[:5]
        rows, k = x2.shape
        n, dt, dev = w.shape[0], x2.dtype, x2.device
        new = torch.empty if rows and n else torch.zeros
        dx = new(shape, dtype=dt, device=dev) if need_x else None
        dw = new((n, k), dtype=dt, device=dev) if need_w else None
        db = new(bias[0], dtype=bias[1], device=dev) if need_b else None
        dg = new(gshape, dtype=gate.dtype, device=dev) if need_g else None
        if rows and n and (need_x or need_w or need_b or need_g):
            d2, rpg, gated = rows_of(dy, n), rows // groups, 0 if gate is None else 1
            xp, wp, dp, xr, dr = x2.data_ptr(), w.data_ptr(), d2.data_ptr(), x2.stride(0), d2.stride(0)
            w_row, w_col = w.stride()
            need = _bytes_bwd((xp & 15, xr, wp & 15, w_row, w_col, dp & 15, dr, code, act, gated, rpg, rows, n, k,
                               1 if need_x else 0, 1 if need_w else 0, 1 if need_b or need_g else 0))
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            with _native.on_device(dev):
                rc = _native.lib().wf_dense_bwd(xp, xr, wp, w_row, w_col, dp, dr, ptr(h), code, act, ptr(gate),
                                                code if gate is None else CODES[gate.dtype], rpg, rows, n, k, ptr(dx),
                                                ptr(dw), ptr(db), code if bias is None else CODES[bias[1]], ptr(dg), ptr(ws),
                                                need, _native.stream_of(dev))
            if rc:
                _native.must(rc, "wf_dense_bwd")
        return dx, dw, db, dy if need_r else None, dg, None


_apply = applier(_Dense)


def dense(x, weight, bias=None, act=None, residual=None, gate=None):
    """``residual + gate * act(x @ weight.T + bias)`` for ``x`` [..., K] and ``weight`` [N, K], bfloat16 or float16, any
    strides. ``act``: None, "gelu", "gelu_tanh", "silu" or "relu". ``bias`` [N]; ``residual`` [..., N]; ``gate`` [N], or
    [..., G, N] with a row for each of G groups of consecutive rows; bias and gate of x's type or float32. Records gradients
    of all five. None when it is not the kernel's case (not plain GPU tensors, other types, K above 2^20, rows or N above
    2^24, or above 2^20 with gradients); ValueError when the shapes do not fit together or ``act`` is unknown."""
    act_code = ACTIVATIONS.get(act)
    if act_code is None:
        raise ValueError(f"act={act!r}: one of {', '.join(map(repr, ACTIVATIONS))}")
    dt, dev, dims = x.dtype, x.device, x.dim()
    if (dt != torch.bfloat16 and dt != torch.float16) or dims == 0 or dev.type != "cuda":
        return None
    if weight.dtype != dt or not plain(dev, x, weight, bias, residual, gate):
        return None
    xshape = x.shape
    k = xshape[-1]
    if weight.dim() != 2 or weight.shape[1] != k or k == 0:
        raise ValueError(f"weight has shape {tuple(weight.shape)}: [N, {k}] fits x {tuple(xshape)}")
    n = weight.shape[0]
    rows = xshape[0] if dims == 2 else x.numel() // k
    groups = 1
    if bias is not None:
        if bias.dtype != dt and bias.dtype != torch.float32:
            return None
        if bias.numel() != n:
            raise ValueError(f"bias has shape {tuple(bias.shape)}: {n} values are wanted")
    if residual is not None:
        if residual.dtype != dt:
            return None
        if residual.shape[:-1] != xshape[:-1] or residual.shape[-1] != n:
            raise ValueError(f"residual has shape {tuple(residual.shape)}: {(*xshape[:-1], n)} is wanted")
    if gate is not None:
        if gate.dtype != dt and gate.dtype != torch.float32:
            return None
        groups = groups_of(gate, rows, n, "gate") if n else 1
    grads = wants_grad(x, weight, bias, residual, gate)
    most = MAX_K if grads else MAX_ROWS
    if rows > most or n > most or k > MAX_K or groups > 65535:
        return None
    code = CODES[dt]
    if grads:
        return _apply(x, weight, bias, residual, gate, (code, act_code, groups))
    y, _ = _launch(rows_of(x, k), _matrix(weight), whole(bias), code, act_code,
                   None if residual is None else rows_of(residual, n), whole(gate), groups, False)
    return y if dims == 2 else y.view(*xshape[:-1], n)
