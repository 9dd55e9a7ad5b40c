"""Orthogonalised updates: every singular value of a matrix's momentum moved towards one by a few Newton-Schulz products (wf_muon,
wf_orthogonalize), as the Muon optimizer steps the matrices of a model while ``fused_adamw`` steps the rest.

``Muon`` is the optimizer; ``muon_step`` one step on given matrices, those of one shape through every launch together;
``orthogonalize`` the direction alone. Momenta are float32. The reference trains nothing."""
import array
import ctypes
import math
import operator
import warnings

import torch

from .. import _native
from .operands import CODES, Sizes, duals, plain, wants_grad, whole

COEFFICIENTS = (3.4445, -4.7750, 2.0315)     # steep at zero: small singular values grow by 3.4 a step; all end between 0.7 and 1.2
_TYPES = frozenset((torch.Tensor, torch.nn.Parameter))
_dtype, _index, _contiguous = operator.attrgetter("dtype"), torch.Tensor.get_device, torch.Tensor.is_contiguous
_capturing = torch.cuda.is_current_stream_capturing
_data_ptr, _numel, _shape = torch.Tensor.data_ptr, torch.Tensor.numel, operator.attrgetter("shape")
MAX_SHORT, MAX_LONG, MAX_VALUES = 16384, 1 << 20, 1 << 30


def _ask(count, rows, cols):
    need = ctypes.c_int64()
    _native.call("wf_muon_workspace", count, rows, cols, ctypes.byref(need))
    return need.value


_bytes = Sizes(_ask)


def _fits(rows, cols):
    return min(rows, cols) <= MAX_SHORT and max(rows, cols) <= MAX_LONG and (rows + 256) * (cols + 8) < MAX_VALUES


_known = {}


def _polynomial(steps, coefficients, eps):
    """The coefficients as the library takes them; ValueError for what it would refuse."""
    steps, abc = operator.index(steps), tuple(map(float, coefficients))
    held = _known.get((steps, abc))
    if held is None:
        if len(abc) != 3 or not 1 <= steps <= 32:
            raise ValueError(f"steps={steps} (1 to 32), coefficients={abc} (three)")
        held = (ctypes.c_double * 3)(*abc)
        if _native.lib().wf_orthogonalize(None, 0, 1, 1, 0, steps, held, 1.0, None, 0, None):
            raise ValueError(_native.last_error())
        if len(_known) > 256:
            _known.clear()
        _known[steps, abc] = held
    if not 0 < eps < math.inf:
        raise ValueError(f"eps={eps}")
    return held


def orthogonalize(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """``x`` [..., M, N] over its Frobenius norm (at least ``eps``), matrix by matrix, then ``steps`` times a X + (b A + c A A) X
    with A = X X^T: each singular value v put through a v + b v^3 + c v^5. float16, bfloat16 or float32, any strides. No gradient is
    recorded (a UserWarning says so where one would have been). With a
    shorter side up to 64 nothing is rounded before the result; above, whatever x's type, the products take float16: the result is off
    by about 1e-3 of its norm for flat and falling spectra, up to 4e-3 where few directions hold nearly all of x, and 1.5e-2 where two
    or three entries do. None when it is not the kernel's case (no plain GPU tensor, another type, a shorter side above 16384, a
    longer one above 2^20, 2^30 values); ValueError for coefficients that let singular values grow past 1.9."""
    abc = _polynomial(steps, coefficients, eps)
    code, dev = CODES.get(x.dtype), x.device
    if x.dim() < 2:
        raise ValueError(f"x has shape {tuple(x.shape)}: matrices are wanted")
    rows, cols = x.shape[-2:]
    if code is None or dev.type != "cuda" or not plain(dev, x) or not _fits(rows, cols):
        return None
    if wants_grad(x):
        warnings.warn("orthogonalize records no gradient: its result is a constant to autograd", stacklevel=2)
    x = whole(x.detach())
    out = torch.empty_like(x)
    if not x.numel():
        return out
    count, size = x.numel() // (rows * cols), rows * cols * x.element_size()
    table = array.array("q", [0]) * (3 * count)
    table[0::3] = array.array("q", range(out.data_ptr(), out.data_ptr() + count * size, size))
    table[1::3] = array.array("q", range(x.data_ptr(), x.data_ptr() + count * size, size))
    need = _bytes((count, rows, cols))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    with _native.on_device(dev):
        _native.call("wf_orthogonalize", table.buffer_info()[0], count, rows, cols, code, steps, abc, eps, ws.data_ptr(), need,
                     _native.stream_of(dev))
    return out


def muon_momenta(params):
    """Zero momenta for ``params``: float32, of their shapes."""
    return [torch.zeros(p.shape, dtype=torch.float32, device=p.device) for p in params]


def _size(adjust, rows, cols):
    if adjust == "spectral":
        return math.sqrt(max(1.0, rows / cols))
    if adjust == "rms":
        return 0.2 * math.sqrt(max(rows, cols))
    raise ValueError(f"adjust={adjust!r}: 'spectral' or 'rms'")


def _odd_one(params, grads, momenta, dt, dev):
    """What is wrong with the first matrix that does not fit."""
    for p, g, m in zip(params, grads, momenta):
        if p.dim() != 2:
            return f"parameter {tuple(p.shape)}: matrices are wanted (fused_adamw steps the others)"
        for t, want in ((p, dt), (g, dt), (m, torch.float32)):
            if t.dtype != want or t.device != dev or not t.is_contiguous() or t.numel() != p.numel() or type(t) not in _TYPES:
                return (f"parameter {tuple(p.shape)} {p.dtype} on {p.device}, gradient {tuple(g.shape)} {g.dtype} on {g.device}, "
                        f"momentum {tuple(m.shape)} {m.dtype} on {m.device}: plain contiguous matrices of one shape, {dt} and "
                        f"float32 momenta on {dev}, are wanted")
    return "a gradient has another shape than its parameter"


def _ready(params, grads, momenta, lr, momentum, nesterov, weight_decay, steps, coefficients, eps, adjust):
    """A step's launches, once everything about it has been found in order (ValueError if not): nothing has changed until they
    are called."""
    if not len(params) == len(grads) == len(momenta):
        raise ValueError(f"{len(params)} parameters, {len(grads)} gradients and {len(momenta)} momenta")
    if not (0 <= momentum < 1 and math.isfinite(lr) and math.isfinite(weight_decay)):
        raise ValueError(f"lr={lr}, momentum={momentum}, weight_decay={weight_decay}")
    abc = _polynomial(steps, coefficients, eps)
    _size(adjust, 1, 1)
    if not params:
        return lambda: None
    dt, dev = params[0].dtype, params[0].device
    code = CODES.get(dt)
    if code is None or dev.type != "cuda":
        raise ValueError(f"parameters of type {dt} on {dev}: float32, bfloat16 or float16 on a GPU")
    with _native.on_device(dev):
        if _capturing():
            raise RuntimeError("a step cannot be captured into a graph: its rates and addresses are the call's, and a replay would "
                               "repeat them")
    if not plain(dev):
        raise ValueError("a step inside a functorch transform or a trace, which would not see it")
    # (questions of all tensors at once: with hundreds of adapters they are the step's host time, a microsecond a matrix)
    every = params + grads + momenta
    if duals(every):
        raise ValueError("a forward-mode tangent, which the step would leave behind")
    shapes, many = list(map(_shape, params)), len(params)
    if (set(map(_dtype, params + grads)) != {dt} or set(map(_dtype, momenta)) != {torch.float32}
            or set(map(_index, every)) != {dev.index} or not all(map(_contiguous, every))
            or not _TYPES.issuperset(map(type, every)) or shapes != list(map(_shape, grads))):
        raise ValueError(_odd_one(params, grads, momenta, dt, dev))
    by_shape = {}
    for i, key in enumerate(zip(shapes, map(_numel, momenta))):
        which = by_shape.get(key)
        if which is None:
            by_shape[key] = [i]
        else:
            which.append(i)
    need, order, calls = 0, [], []
    for (shape, values), which in by_shape.items():
        if len(shape) != 2 or shape[0] * shape[1] != values:
            raise ValueError(_odd_one(params, grads, momenta, dt, dev))
        rows, cols = shape
        if values:
            if not _fits(rows, cols):
                raise ValueError(f"a matrix of {rows} x {cols}: the shorter side is at most {MAX_SHORT}, the longer {MAX_LONG}, "
                                 f"and there are fewer than {MAX_VALUES} values")
            # (contiguous, but not what its memory holds: only a single value can be both without a private call)
            if values == 1 and any(t[i].is_neg() for t in (params, grads, momenta) for i in which):
                raise ValueError("a negative view: what it stands for is not in its memory")
            need = max(need, _bytes((len(which), rows, cols)))
            calls.append((24 * len(order), len(which), rows, cols, lr * _size(adjust, rows, cols)))
            order += which
    at, table = list(map(_data_ptr, every)), array.array("q", bytes(24 * len(order)))
    if len(order) > 1:
        pick = operator.itemgetter(*order)
        at_p, at_g, at_m = (pick(at[k * many:(k + 1) * many]) for k in range(3))
    else:
        at_p, at_g, at_m = ([at[i + k * many] for i in order] for k in range(3))
    for k, column in enumerate((at_p, at_g, at_m)):
        table[k::3] = array.array("q", column)
    if len({*at_p, *at_m}) != 2 * len(order):
        raise ValueError("a parameter or a momentum is there twice: each is stepped on its own")
    if dt == torch.float32 and not set(at_g).isdisjoint(at_m):
        raise ValueError("a gradient is a momentum's memory, which the step changes before it has read the gradient for the last time")

    def launch():
        if not calls:
            return
        base = table.buffer_info()[0]
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        with _native.on_device(dev):
            for offset, count, rows, cols, rate in calls:
                _native.call("wf_muon", base + offset, count, rows, cols, code, momentum, 1 if nesterov else 0,
                             1.0 - lr * weight_decay, rate, steps, abc, eps, ws.data_ptr(), need, _native.stream_of(dev))
        # what autograd saved of them is stale now, as after torch's own in-place operations
        torch.autograd.graph.increment_version(params)
        torch.autograd.graph.increment_version(momenta)
    return launch


def muon_step(params, grads, momenta, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.1, steps=5, coefficients=COEFFICIENTS,
              eps=1e-7, adjust="spectral"):
    """A step on ``params`` and ``momenta`` in place: m = momentum m + (1 - momentum) g; the update is m, or with ``nesterov``
    momentum m + (1 - momentum) g, orthogonalised as by ``orthogonalize``; p = (1 - lr weight_decay) p - lr s update, s =
    sqrt(max(1, rows / cols)) ("spectral") or 0.2 sqrt(max(rows, cols)) ("rms": updates as large as AdamW's). ``params`` and ``grads``:
    contiguous GPU matrices of one type (float32, bfloat16 or float16); ``momenta``: contiguous, float32, as many values
    (``muon_momenta``); all on one device, no parameter or momentum twice, none sharing its memory with another tensor.
    ValueError for anything else. Asynchronous on torch's current stream; RuntimeError while that is captured into a graph."""
    _ready(list(params), list(grads), list(momenta), lr, momentum, nesterov, weight_decay, steps, coefficients, eps, adjust)()


_OPTIONS = ("lr", "momentum", "nesterov", "weight_decay", "steps", "coefficients", "eps", "adjust")


class Muon(torch.optim.Optimizer):
    """The optimizer over ``muon_step``: a parameter group is one call. Parameters without a gradient are left alone."""

    def __init__(self, params, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.1, steps=5, coefficients=COEFFICIENTS, eps=1e-7,
                 adjust="spectral"):
        _polynomial(steps, coefficients, eps)
        _size(adjust, 1, 1)
        super().__init__(params, {"lr": lr, "momentum": momentum, "nesterov": nesterov, "weight_decay": weight_decay, "steps": steps,
                                  "coefficients": tuple(coefficients), "eps": eps, "adjust": adjust})
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"parameter {tuple(p.shape)}: matrices are wanted (fused_adamw steps the others)")

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # (torch casts a loaded state to its parameter's type; momenta are kept as they were saved)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                self.state[p] = {k: v.to(p.device, copy=True) if isinstance(v, torch.Tensor) else v
                                 for k, v in state_dict["state"][i].items()}

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        ready = []                                       # of every group, before the first of them changes anything
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            held = [self.state.get(p) or {"momentum": torch.zeros(p.shape, dtype=torch.float32, device=p.device)} for p in params]
            launch = _ready(params, [p.grad for p in params], [h["momentum"] for h in held],
                            **{k: v for k, v in group.items() if k in _OPTIONS})
            ready.append((launch, params, held))
        for launch, params, held in ready:
            launch()
            for p, h in zip(params, held):
                self.state[p] = h
        return loss
