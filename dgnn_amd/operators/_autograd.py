"""When an operator call has to go through its autograd.Function."""
import torch
from torch.autograd import forward_ad


def differentiated(*tensors):
    """True if the call is part of a backward graph or of forward-mode differentiation.  A dual tensor does not require grad:
    past the Function, which raises for it, its tangent would be dropped and the derivative read as zero."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                return True
    # (no dual level is open: what unpack_dual would find out for each tensor, a microsecond of a small call's seven)
    if getattr(forward_ad, "_current_level", 0) < 0:
        return False
    return any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)
