"""The end of a transformer block: what follows gate_merge and the output
projection, and precedes the next projection.

residual_rms_norm adds the block's output, with dropout in training, to the
residual stream and takes the root-mean-square norm of the sum;
residual_rms_norm_fp8 is its serving form, whose rows leave in 8 bits with
scales.  Both run on gfx950 HIP kernels, one pass over the rows each way
(eager: lsrm_hip.native(); traced: torch.ops.lsrm_hip.residual_norm_fwd /
_bwd / _fp8).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

import lsrm_hip as _hip

from ._dispatch import eager, needs_grad


def _check(x, residual, weight, eps):
    _hip.norm.check_rows(x, residual, weight)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")


def residual_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                      eps: float = 1e-6, dropout_p: float = 0.0,
                      rng_state: Optional[torch.Tensor] = None
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [.., hidden], residual of the same shape (or None), weight [hidden],
    one of bf16 / fp16 / fp32 -> (y, h): h = residual + dropout(x), rounded to
    the dtype, is the new residual stream, and y = h / sqrt(mean(h^2) + eps) *
    weight.  Differentiable in x, residual and weight, through y and h.

    dropout_p > 0 needs rng_state, int64 [2] on the device: a seed and an
    offset, read when the kernel runs.  The mask is a function of them and of
    the element's row and column alone and is not stored; the backward draws
    it again from the values that the forward read, so the state may be
    changed in between (rng_state[1] += 1 for the next call, in a captured
    graph too).  Elements stay with probability 1 - round(65536 dropout_p) /
    65536 and are divided by it."""
    least = _hip.norm.drop_least(dropout_p)
    if least == 0:
        rng_state = None
    if not eager(x, residual, weight, rng_state):
        _check(x, residual, weight, eps)
        if least > 0:
            _hip.norm.check_rng(x, rng_state)
        return torch.ops.lsrm_hip.residual_norm_fwd(x, residual, weight, float(eps), least,
                                                    rng_state)[:2]
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    return _hip.native().residual_norm(x, residual, weight, eps, least, rng_state)


def residual_rms_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor],
                          weight: torch.Tensor, eps: float = 1e-6, group_size: int = 0
                          ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (y8 float8_e4m3fn [.., hidden], scales fp32 [.., hidden / group_size],
    h): y8 holds y / scale, where scale = max |y| / 448 over the row
    (group_size 0) or over each 32, 64 or 128 channels.  For inference: refuses
    inputs that require gradients while gradients are recorded."""
    if needs_grad(x, residual, weight):
        raise RuntimeError("residual_rms_norm_fp8 has no backward; call it under no_grad")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if eager(x, residual, weight):
        return _hip.native().residual_norm_fp8(x, residual, weight, eps, group_size)
    _check(x, residual, weight, eps)
    return torch.ops.lsrm_hip.residual_norm_fp8(x, residual, weight, float(eps),
                                                int(group_size))
