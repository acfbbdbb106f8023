"""When a call may go straight to the kernels.

A call through torch.ops.lsrm_hip.* passes the dispatcher's Python layers,
which cost 7 us without and some 60 us with gradients, and ctypes another 10: more
than the kernels of a few tokens.  Plain tensors in eager mode need none of what
they add, so the operators for single tokens and small batches call the C++
binding (lsrm_hip.native()) themselves; tracing (torch.compile, export), tensor
subclasses and dispatch modes take the registered operator.  Both run the same
kernels.
"""

from __future__ import annotations

import torch
from torch.utils._python_dispatch import _get_current_dispatch_mode

_PLAIN = (torch.Tensor, torch.nn.Parameter)


def eager(*tensors) -> bool:
    return not torch.compiler.is_compiling() and _get_current_dispatch_mode() is None and \
        all(t is None or type(t) in _PLAIN for t in tensors)


def needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
