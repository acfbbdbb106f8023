"""Binding of the residual norm kernels (lsrm_residual_norm_*,
include/lsrm_hip.h)."""

from __future__ import annotations

from typing import Optional

import torch

import lsrm_hip as _hip


def drop_least(p: float) -> int:
    """The draw of 16 bits that an element has to reach to stay."""
    if not 0.0 <= p < 1.0:
        raise ValueError("dropout probability must be in [0, 1)")
    return min(65535, round(p * 65536))


def check_rows(x, residual, weight) -> torch.device:
    dev = _hip._dev_check(x, residual, weight)
    if x.dtype not in _hip._DTYPE_CODE or weight.dtype != x.dtype or \
            (residual is not None and residual.dtype != x.dtype):
        raise TypeError("x, residual and weight must share one of bf16 / fp16 / fp32")
    if x.dim() < 1 or weight.dim() != 1 or x.shape[-1] != weight.shape[0] or \
            (residual is not None and residual.shape != x.shape):
        raise ValueError("x and residual [.., hidden] of one shape and weight [hidden] expected")
    if not 0 < x.shape[-1] <= 16384:
        raise ValueError("hidden must be in 1 .. 16384")
    return dev


def check_rng(x, rng_state) -> None:
    if rng_state is None:
        raise ValueError("dropout needs rng_state")
    _hip._dev_check(x, rng_state)
    if rng_state.dtype != torch.int64 or tuple(rng_state.shape) != (2,):
        raise ValueError("rng_state must be int64 [2] (seed, offset)")


def residual_norm_fwd(x, residual: Optional[torch.Tensor], weight, eps: float, least: int,
                      rng_state: Optional[torch.Tensor]):
    """-> (y, h, rstd [rows] fp32, rng_used [2] int64)."""
    dev = check_rows(x, residual, weight)
    if least > 0:
        check_rng(x, rng_state)
        rng_state = rng_state.contiguous()
    x, weight = x.contiguous(), weight.contiguous()
    residual = None if residual is None else residual.contiguous()
    hidden = x.shape[-1]
    n = x.numel() // hidden
    y, h = torch.empty_like(x), torch.empty_like(x)
    rstd = torch.empty(n, dtype=torch.float32, device=dev)
    used = torch.empty(2 if least > 0 else 0, dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        _hip._check(_hip.lib().lsrm_residual_norm_fwd(
            x.data_ptr(), _hip._ptr(residual), weight.data_ptr(), _hip._DTYPE_CODE[x.dtype], n,
            hidden, eps, least, rng_state.data_ptr() if least > 0 else None,
            used.data_ptr() if least > 0 else None, y.data_ptr(), h.data_ptr(), rstd.data_ptr(),
            _hip._stream(dev)), "lsrm_residual_norm_fwd")
    return y, h, rstd, used


def residual_norm_fp8(x, residual: Optional[torch.Tensor], weight, eps: float, group: int):
    """-> (y8 float8_e4m3fn, scales fp32 [.., groups], h)."""
    dev = check_rows(x, residual, weight)
    hidden = x.shape[-1]
    if group not in (0, 32, 64, 128) or (group and hidden % group):
        raise ValueError("group_size must be 0 (the row), 32, 64 or 128 and divide hidden")
    x, weight = x.contiguous(), weight.contiguous()
    residual = None if residual is None else residual.contiguous()
    n = x.numel() // hidden
    h = torch.empty_like(x)
    y8 = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty(x.shape[:-1] + (hidden // group if group else 1,), dtype=torch.float32,
                         device=dev)
    with torch.cuda.device(dev):
        _hip._check(_hip.lib().lsrm_residual_norm_fp8(
            x.data_ptr(), _hip._ptr(residual), weight.data_ptr(), _hip._DTYPE_CODE[x.dtype], n,
            hidden, eps, group, y8.data_ptr(), scales.data_ptr(), h.data_ptr(),
            _hip._stream(dev)), "lsrm_residual_norm_fp8")
    return y8, scales, h


def residual_norm_bwd(dy: Optional[torch.Tensor], dh: Optional[torch.Tensor], h, weight, rstd,
                      least: int, rng_used: Optional[torch.Tensor]):
    """-> (dx or None, d_residual, d_weight); dx is None without dropout (it
    equals d_residual)."""
    dev = check_rows(h, None, weight)
    _hip._dev_check(h, dy, dh, rstd)
    for t in (dy, dh):
        if t is not None and (t.shape != h.shape or t.dtype != h.dtype):
            raise ValueError("gradients must match the outputs in shape and dtype")
    hidden = h.shape[-1]
    n = h.numel() // hidden
    if rstd.dtype != torch.float32 or rstd.numel() != n:
        raise ValueError("rstd must be float32 [rows]")
    if least > 0:
        check_rng(h, rng_used)
    h, weight, rstd = h.contiguous(), weight.contiguous(), rstd.contiguous()
    dy = None if dy is None else dy.contiguous()
    dh = None if dh is None else dh.contiguous()
    d_residual, d_weight = torch.empty_like(h), torch.empty_like(weight)
    dx = torch.empty_like(h) if least > 0 else None
    with torch.cuda.device(dev):
        ws = _hip._workspace(_hip.lib().lsrm_residual_norm_bwd_workspace_size(n, hidden), dev)
        _hip._check(_hip.lib().lsrm_residual_norm_bwd(
            _hip._ptr(dy), _hip._ptr(dh), h.data_ptr(), weight.data_ptr(), rstd.data_ptr(),
            _hip._DTYPE_CODE[h.dtype], n, hidden, least,
            rng_used.data_ptr() if least > 0 else None, _hip._ptr(dx), d_residual.data_ptr(),
            d_weight.data_ptr(), ws.data_ptr(), ws.numel(), _hip._stream(dev)),
            "lsrm_residual_norm_bwd")
    return dx, d_residual, d_weight
