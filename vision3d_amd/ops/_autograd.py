"""When a call of an operator goes through its autograd function."""
import torch
from torch.autograd import forward_ad


def recorded(*tensors) -> bool:
    """Whether a call on these tensors (None among them) is one that autograd has to know of: one requires a gradient, or
    carries a tangent of a forward-mode derivative -- which the autograd functions refuse, and a plain call would drop
    without a word."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
