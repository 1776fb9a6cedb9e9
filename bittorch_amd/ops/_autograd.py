"""What autograd wants of a call."""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad


def has_tangent(*tensors: Optional[Tensor]) -> bool:
    """Whether one of them carries a forward-mode derivative (``forward_ad.make_dual``): it need not require a gradient, and no gradient
    mode turns it off."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def differentiated(*tensors: Optional[Tensor]) -> bool:
    """Whether the call belongs to autograd: for a backward pass, or in forward mode, which the autograd functions refuse."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or has_tangent(*tensors)
