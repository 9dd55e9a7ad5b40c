"""AdamW over many tensors in one launch, its moments in float32 or in 8 bits (wf_adamw).

Next to a model whose weights are quantised to 4-8 bits, float32 moments would be the largest thing in memory: 8 bytes a
trained value. In 8 bits they take 2, and 8 bytes a block of 256 values for its two scales. ``AdamW`` is the optimizer;
``adamw_step`` one step on given tensors, ``adamw_state`` / ``AdamWState`` the moments: flat over all tensors, each tensor
starting on a whole block. The reference trains nothing."""
import array
import math
import operator
from typing import NamedTuple, Optional

import torch

from .. import _native
from .operands import CODES, plain

BLOCK = 256
_TYPES = frozenset((torch.Tensor, torch.nn.Parameter))
_dtype, _index, _contiguous = operator.attrgetter("dtype"), torch.Tensor.get_device, torch.Tensor.is_contiguous
_capturing = torch.cuda.is_current_stream_capturing
_data_ptr, _numel = torch.Tensor.data_ptr, torch.Tensor.numel


class AdamWState(NamedTuple):
    """The moments of a list of tensors: float32 without scales, or int8 / uint8 codes with a float32 scale a block."""
    exp_avg: torch.Tensor
    exp_avg_sq: torch.Tensor
    exp_avg_scale: Optional[torch.Tensor] = None
    exp_avg_sq_scale: Optional[torch.Tensor] = None

    @property
    def bits(self):
        return 32 if self.exp_avg_scale is None else 8

    def values(self):
        """Both moments in float32: the state's own tensors, or what its codes stand for."""
        if self.bits == 32:
            return self.exp_avg, self.exp_avg_sq
        _check_state(self)
        dev = self.exp_avg.device
        if dev.type != "cuda":
            raise ValueError(f"codes on {dev}: the kernel that reads them needs them on a GPU")
        m, v = (torch.empty(self.exp_avg.numel(), dtype=torch.float32, device=dev) for _ in range(2))
        with _native.on_device(dev):
            _native.call("wf_adamw_values", self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(),
                         self.exp_avg_scale.data_ptr(), self.exp_avg_sq_scale.data_ptr(), self.exp_avg_scale.numel(),
                         m.data_ptr(), v.data_ptr(), _native.stream_of(dev))
        return m, v


def _blocks(n):
    return -(-n // BLOCK)


def adamw_state(params, bits=8):
    """Zero moments for ``params`` (one device), in 8 or 32 bits."""
    if bits not in (8, 32):
        raise ValueError(f"bits={bits}: 8 or 32")
    params = list(params)
    if not params:
        raise ValueError("no parameters")
    dev, blocks = params[0].device, sum(_blocks(p.numel()) for p in params)
    zeros = lambda n, dt: torch.zeros(n, dtype=dt, device=dev)                                 # noqa: E731
    if bits == 32:
        return AdamWState(zeros(blocks * BLOCK, torch.float32), zeros(blocks * BLOCK, torch.float32))
    return AdamWState(zeros(blocks * BLOCK, torch.int8), zeros(blocks * BLOCK, torch.uint8),
                      zeros(blocks, torch.float32), zeros(blocks, torch.float32))


def _check_state(state):
    """ValueError unless the state's tensors belong together."""
    m, v, ms, vs = state
    n, dev = m.numel(), m.device
    types = (torch.float32, torch.float32) if ms is None else (torch.int8, torch.uint8)
    ok = (m.dtype, v.dtype) == types and v.numel() == n and n % BLOCK == 0 and v.device == dev
    ok = ok and m.is_contiguous() and v.is_contiguous() and (ms is None) == (vs is None)
    if ok and ms is not None:
        ok = all(s.dtype == torch.float32 and s.numel() == n // BLOCK and s.is_contiguous() and s.device == dev
                 for s in (ms, vs))
    if not ok:
        raise ValueError("the state's tensors do not belong together: float32 moments without scales, or int8 and uint8 "
                         "codes with a float32 scale a block of 256, contiguous, on one device")


def _odd_one(params, grads, dt, dev):
    """What is wrong with the first parameter or gradient that does not fit."""
    for p, g in zip(params, grads):
        for t in (p, g):
            if t.dtype != dt or t.device != dev or not t.is_contiguous() or t.numel() != p.numel() or type(t) not in _TYPES:
                return (f"parameter {tuple(p.shape)} {p.dtype} on {p.device} with gradient {tuple(g.shape)} {g.dtype} on "
                        f"{g.device}: plain contiguous tensors of one size, {dt} on {dev}, are wanted")
    return "parameters and gradients do not fit together"


def _ready(params, grads, state, step, lr, betas, eps, weight_decay):
    """A step's launch, once everything about it has been found in order (ValueError if not): nothing has changed until it is
    called."""
    if len(params) != len(grads):
        raise ValueError(f"{len(params)} parameters and {len(grads)} gradients")
    _check_state(state)
    if not step >= 1 or step != int(step):
        raise ValueError(f"step={step}: the first step is 1")
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and 0 <= eps < math.inf and math.isfinite(lr)
            and math.isfinite(weight_decay)):
        raise ValueError(f"lr={lr}, betas={tuple(betas)}, eps={eps}, weight_decay={weight_decay}")
    if not params:
        return lambda: None
    dt, dev = params[0].dtype, state.exp_avg.device
    code = CODES.get(dt)
    if code is None or dev.type != "cuda":
        raise ValueError(f"parameters of type {dt} with moments on {dev}: float32, bfloat16 or float16 on a GPU")
    if _capturing():
        raise RuntimeError("a step cannot be captured into a graph: its step count, rates and addresses are the call's, and a "
                           "replay would repeat them")
    if not plain(dev):
        raise ValueError("a step inside a functorch transform or a trace, which would not see it")
    # (questions of all tensors at once: with hundreds of adapters they are the step's host time, 0.6 us a parameter; the numbers
    # of values are compared, not the shapes: that alone would be a third more)
    both, index, sizes = params + grads, dev.index, list(map(_numel, params))
    if (set(map(_dtype, both)) != {dt} or set(map(_index, both)) != {index} or not all(map(_contiguous, both))
            or sizes != list(map(_numel, grads)) or not _TYPES.issuperset(map(type, both))):
        raise ValueError(_odd_one(params, grads, dt, dev))
    table = array.array("q", [0]) * (3 * len(params))
    table[0::3] = array.array("q", map(_data_ptr, params))
    table[1::3] = array.array("q", map(_data_ptr, grads))
    table[2::3] = array.array("q", sizes)

    def launch():
        with _native.on_device(dev):
            _native.call("wf_adamw", table.buffer_info()[0], len(params), code, state.bits, state.exp_avg.data_ptr(),
                         state.exp_avg_sq.data_ptr(), None if state.exp_avg_scale is None else state.exp_avg_scale.data_ptr(),
                         None if state.exp_avg_sq_scale is None else state.exp_avg_sq_scale.data_ptr(),
                         state.exp_avg.numel() // BLOCK, int(step), lr, betas[0], betas[1], eps, weight_decay,
                         _native.stream_of(dev))
        # what autograd saved of them is stale now, as after torch's own in-place operations
        torch.autograd.graph.increment_version(params)
    return launch


def adamw_step(params, grads, state, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
    """Step ``step`` (1 is the first) on ``params`` and ``state`` in place: decoupled weight decay, bias-corrected moments.
    ``params`` and ``grads``: contiguous GPU tensors of one type (float32, bfloat16 or float16) on one device, a gradient as
    many values as its parameter, in the order that ``state`` was made for. ValueError for anything else. Asynchronous on
    torch's current stream; RuntimeError while that is captured into a graph, whose replays would repeat this very step."""
    _ready(list(params), list(grads), state, step, lr, betas, eps, weight_decay)()


class AdamW(torch.optim.Optimizer):
    """The optimizer over ``adamw_step``: a parameter group is one call. Every parameter of a group has to have a gradient
    in each step or in none (their moments are one array); a group without gradients is left alone."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=8):
        if bits not in (8, 32):
            raise ValueError(f"bits={bits}: 8 or 32")
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay, "bits": bits})

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # (torch casts a loaded state to its parameter's type; codes and float32 moments are kept as they were saved)
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
        steps = []                                       # of every group, before the first of them changes anything
        for group in self.param_groups:
            params = group["params"]
            grads = [p.grad for p in params]
            missing = sum(g is None for g in grads)
            if missing == len(grads):
                continue
            if missing:
                raise ValueError(f"{missing} of a group's {len(grads)} parameters have no gradient")
            held = self.state.get(params[0]) or {"step": 0, **adamw_state(params, group["bits"])._asdict()}
            step = held["step"] + 1
            launch = _ready(params, grads, AdamWState(*(held[f] for f in AdamWState._fields)), step, group["lr"],
                            group["betas"], group["eps"], group["weight_decay"])
            steps.append((launch, params[0], held, step))
        for launch, first, held, step in steps:
            launch()
            held["step"] = step
            self.state[first] = held
        return loss
