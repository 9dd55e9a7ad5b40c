"""What the training-step operators (fused_norm, fused_dense, fused_adamw) ask of their tensors. The kernels read memory,
so tensors that are more than memory (subclasses, functorch wrappers, forward-mode duals) are not their case."""
import torch

CODES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}      # the library's dtype codes


def plain(t, device):
    """Whether ``t`` is an ordinary tensor on ``device``."""
    return (type(t) in (torch.Tensor, torch.nn.Parameter) and t.device == device
            and not torch._C._functorch.is_functorch_wrapped_tensor(t) and not t._is_zerotensor() and not t.is_neg()
            and torch.autograd.forward_ad.unpack_dual(t).tangent is None)


def rows_of(t, width):
    """``t`` [..., width] as a matrix whose rows are runs of values, a view where its strides allow one."""
    t2 = t if t.dim() == 2 else t.reshape(-1, width)
    return t2 if t2.stride(1) == 1 or width == 1 else t2.contiguous()


def groups_of(t, rows, width, what):
    """The number of row groups that a parameter [width] or [..., groups, width] stands for; ValueError when it is not one
    row a group of ``rows // groups`` consecutive rows."""
    if t.dim() == 0 or t.shape[-1] != width:
        raise ValueError(f"{what} has shape {tuple(t.shape)}: its last dimension has to be {width}")
    groups = t.numel() // width
    if groups == 0 or rows % groups:
        raise ValueError(f"{what} has shape {tuple(t.shape)}: {rows} rows are no whole number of its {groups} groups")
    return groups


def wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def ptr(t):
    return None if t is None else t.data_ptr()
