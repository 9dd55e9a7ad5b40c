"""What the training-step operators (fused_norm, fused_dense, fused_adamw) ask of their tensors. The kernels read memory,
so tensors that are more than memory (subclasses, functorch wrappers, forward-mode duals, negative views) are not their
case, and neither is a call that is being traced: a kernel launched through ctypes is no operation that a trace records.
These questions run once per call, so each is asked in its cheapest form."""
import torch
from torch.autograd import forward_ad

CODES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}      # the library's dtype codes
_TYPES = frozenset((torch.Tensor, torch.nn.Parameter))
_level = torch._C._functorch.maybe_current_level
_wrapped = torch._C._functorch.is_functorch_wrapped_tensor
_grad_enabled = torch.is_grad_enabled
_jit_traces, _modes, _mode = torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._get_dispatch_mode
_TRACERS = (torch._C._TorchDispatchModeKey.PROXY, torch._C._TorchDispatchModeKey.FAKE)


def _dual(t):
    return _wrapped(t) or t._is_zerotensor() or forward_ad.unpack_dual(t).tangent is not None


def duals(tensors):
    """Whether forward mode is at work and one of ``tensors`` (an iterable) carries a tangent, which an operation in place on its memory alone
    would leave behind."""
    return forward_ad._current_level >= 0 and any(map(_dual, tensors))


def plain(device, *tensors):
    """Whether each of ``tensors`` is None or an ordinary tensor on ``device``, outside functorch's transforms and traces."""
    if _level() is not None or _jit_traces():
        return False
    if _modes() and any(_mode(k) is not None for k in _TRACERS):    # proxies or fake tensors record what runs
        return False
    deep = forward_ad._current_level >= 0                            # forward mode is at work somewhere
    for t in tensors:
        if t is None:
            continue
        if type(t) not in _TYPES or t.device != device or t.is_neg():
            return False
        if deep and _dual(t):
            return False
    return True


def gradient(dy):
    """``dy``, the gradient that a backward pass is given, as its kernels read it. RuntimeError for one that is more than its
    memory -- a forward-mode tangent, a functorch wrapper, a subclass with its own operations -- whose rest the pass would
    lose in silence: the forward pass could not know of it."""
    if dy.is_neg():
        dy = dy.resolve_neg()
    if type(dy) not in _TYPES and type(dy).__torch_dispatch__ is torch.Tensor.__torch_dispatch__:
        dy = dy.as_subclass(torch.Tensor)                            # a subclass in name only
    if not plain(dy.device, dy):
        raise RuntimeError(f"a gradient that is no plain tensor ({type(dy).__name__}; or it carries a forward-mode tangent, or "
                           "a functorch transform or a trace is at work): the backward pass of this operator takes values alone")
    return dy


def rows_of(t, width):
    """``t`` [..., width] as a matrix whose rows are runs of values, a view where its strides allow one."""
    t2 = t if t.dim() == 2 else t.reshape(-1 if width else t.shape[:-1].numel(), width)
    return t2 if t2.stride(1) == 1 or width == 1 else t2.contiguous()


def whole(t):
    """``t`` contiguous, or None for None."""
    return t if t is None or t.is_contiguous() else t.contiguous()


def groups_of(t, rows, width, what):
    """The number of row groups that a parameter [width] or [..., groups, width] stands for; ValueError when it is not one
    row a group of ``rows // groups`` consecutive rows."""
    shape = t.shape
    if not shape or shape[-1] != width:
        raise ValueError(f"{what} has shape {tuple(shape)}: its last dimension has to be {width}")
    groups = 1 if len(shape) == 1 else t.numel() // width
    if groups == 0 or rows % groups:
        raise ValueError(f"{what} has shape {tuple(shape)}: {rows} rows are no whole number of its {groups} groups")
    return groups


def wants_grad(*tensors):
    if _grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def ptr(t):
    return None if t is None else t.data_ptr()


def once(backward):
    """A Function's backward that is differentiable once: with create_graph, torch's own wrapper (whose result refuses a
    second derivative); without, as it nearly always is, the bare function."""
    wrapped = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *dys):
        return wrapped(ctx, *dys) if _grad_enabled() else backward(ctx, *dys)
    return staticmethod(run)


def applier(function):
    """``function.apply`` without its Python layer, which unwraps functorch's tensors (``plain`` has refused them by then)
    and costs as much as a launch's checks."""
    return super(torch.autograd.Function, function).apply


class Sizes:
    """Workspace bytes by call shape: the library's answer depends on nothing else, so it is asked once a shape."""

    def __init__(self, ask):
        self._ask, self._known = ask, {}

    def __call__(self, key):
        need = self._known.get(key)
        if need is None:
            if len(self._known) > 4096:
                self._known.clear()
            need = self._known[key] = self._ask(*key)
        return need
