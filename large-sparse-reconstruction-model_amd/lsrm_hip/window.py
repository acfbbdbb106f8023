"""Binding of the sliding-window attention kernels (lsrm_window_*,
include/lsrm_hip.h)."""

from __future__ import annotations

from typing import Optional

import torch

import lsrm_hip as _hip

MAX_STRIDE = 1 << 22  # elements between tokens that the kernels take


def token_rows(t: torch.Tensor):
    """(tensor, elements between its tokens) for [N, H, D]: the tensor itself
    where a token's heads are contiguous and its rows can be read in 16-byte
    pieces (a slice of a fused projection, say), else a contiguous copy."""
    n, h, d = t.shape
    dense = h * d
    if t.is_contiguous():
        stride = dense
    elif t.stride(2) == 1 and (h == 1 or t.stride(1) == d):
        stride = t.stride(0) if n > 1 else dense
    else:
        stride = -1
    if stride < dense or stride % 8 or stride > MAX_STRIDE or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format), dense
    return t, stride


def check_qkv(q, k, v) -> torch.device:
    dev = _hip._dev_check(q, k, v)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[2] != k.shape[2]:
        raise ValueError("q [Nq, Hq, D], k and v [Nk, Hkv, D] expected")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or \
            v.dtype != q.dtype:
        raise TypeError("q, k and v must share dtype float16 or bfloat16")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1] != 0:
        raise ValueError("num_q_heads must be a multiple of num_kv_heads")
    return dev


def bias_args(q, hq, bias_table, bias_buckets):
    """(table, buckets, number of buckets, range) of the C entry points."""
    if (bias_table is None) != (bias_buckets is None):
        raise ValueError("bias_table and bias_buckets go together")
    if bias_table is None:
        return None, None, 0, -1
    _hip._dev_check(q, bias_table, bias_buckets)
    if bias_table.dim() != 2 or bias_table.shape[1] != hq or bias_table.shape[0] == 0:
        raise ValueError(f"bias_table must be [num_buckets, num_q_heads = {hq}]")
    if bias_table.dtype != q.dtype:
        raise TypeError("bias_table must share the dtype of q")
    if bias_buckets.dim() != 1 or bias_buckets.numel() % 2 != 1:
        raise ValueError("bias_buckets must be [2 * max_distance + 1]")
    return (bias_table.contiguous(), _hip._i32(bias_buckets), bias_table.shape[0],
            bias_buckets.numel() // 2)


def _offsets(q, cu_seqlens_q, cu_seqlens_k):
    _hip._dev_check(q, cu_seqlens_q, cu_seqlens_k)
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape != cu_seqlens_k.shape or \
            cu_seqlens_q.numel() == 0:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must both have batch_size + 1 entries")
    return _hip._i32(cu_seqlens_q), _hip._i32(cu_seqlens_k)


def window_validate(n_q: int, n_k: int, cu_seqlens_q, cu_seqlens_k, bias_buckets=None,
                    n_buckets: int = 0) -> int:
    """Device check of the offsets and the bucket map (one host
    synchronisation); returns the lsrm_meta_error bits."""
    dev = _hip._dev_check(cu_seqlens_q, cu_seqlens_k, bias_buckets)
    cu_q, cu_k = _hip._i32(cu_seqlens_q), _hip._i32(cu_seqlens_k)
    buckets = None if bias_buckets is None else _hip._i32(bias_buckets)
    flags = torch.empty(1, dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        _hip._check(_hip.lib().lsrm_window_validate(
            cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, n_q, n_k, _hip._ptr(buckets),
            0 if buckets is None else buckets.numel() // 2, n_buckets, flags.data_ptr(),
            _hip._stream(dev)), "lsrm_window_validate")
    return int(flags.item())


def window_attn_fwd(q, k, v, cu_seqlens_q, cu_seqlens_k, left: int, right: int, sinks: int,
                    bias_table: Optional[torch.Tensor], bias_buckets: Optional[torch.Tensor],
                    softmax_scale: float, with_low: bool = False):
    """-> (out [Nq, Hq, D], lse [Hq, Nq] fp32 in log2 units, out_low int8: with
    with_low the 8 bits of out that follow its rounding, for the backward, else
    empty)."""
    dev = check_qkv(q, k, v)
    cu_q, cu_k = _offsets(q, cu_seqlens_q, cu_seqlens_k)
    nq, hq, d = q.shape
    nk, hkv, _ = k.shape
    table, buckets, n_buckets, r = bias_args(q, hq, bias_table, bias_buckets)
    q, qs = token_rows(q)
    k, ks = token_rows(k)
    v, vs = token_rows(v)
    out = torch.empty((nq, hq, d), dtype=q.dtype, device=dev)
    lse = torch.empty((hq, nq), dtype=torch.float32, device=dev)
    low = torch.empty((nq, hq, d) if with_low else (0,), dtype=torch.int8, device=dev)
    with torch.cuda.device(dev):
        _hip._check(_hip.lib().lsrm_window_attn_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _hip._DTYPE_CODE[q.dtype], qs, ks, vs, nq,
            nk, hq, hkv, d, cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, left, right,
            sinks, _hip._ptr(table), n_buckets, _hip._ptr(buckets), r, softmax_scale,
            out.data_ptr(), low.data_ptr() if with_low else None, lse.data_ptr(),
            _hip._stream(dev)), "lsrm_window_attn_fwd")
    return out, lse, low


def window_attn_bwd(do, q, k, v, o, low, lse, cu_seqlens_q, cu_seqlens_k, left: int, right: int,
                    sinks: int, bias_table: Optional[torch.Tensor],
                    bias_buckets: Optional[torch.Tensor], softmax_scale: float):
    """-> (dq, dk, dv, d_table or None), contiguous.  low: the forward's out_low
    (empty: gradients from the rounded output alone)."""
    dev = check_qkv(q, k, v)
    _hip._dev_check(q, do, o, low, lse)
    if low.dtype != torch.int8 or low.numel() not in (0, q.numel()):
        raise ValueError("low must be int8 of q's shape, or empty")
    low = low.contiguous()
    cu_q, cu_k = _offsets(q, cu_seqlens_q, cu_seqlens_k)
    nq, hq, d = q.shape
    nk, hkv, _ = k.shape
    if do.dtype != q.dtype:
        do = do.to(q.dtype)
    for name, t in (("do", do), ("o", o)):
        if t.shape != q.shape or t.dtype != q.dtype:
            raise ValueError(f"{name} must match q in shape and dtype")
    if tuple(lse.shape) != (hq, nq) or lse.dtype != torch.float32:
        raise ValueError("lse must be float32 [Hq, Nq]")
    table, buckets, n_buckets, r = bias_args(q, hq, bias_table, bias_buckets)
    q, qs = token_rows(q)
    k, ks = token_rows(k)
    v, vs = token_rows(v)
    do, o, lse = do.contiguous(), o.contiguous(), lse.contiguous()
    if do.data_ptr() % 16:
        do = do.clone()
    if o.data_ptr() % 16:
        o = o.clone()
    dq = torch.empty((nq, hq, d), dtype=q.dtype, device=dev)
    dk = torch.empty((nk, hkv, d), dtype=q.dtype, device=dev)
    dv = torch.empty_like(dk)
    d_table = None if table is None else torch.empty_like(table)
    batch = cu_q.numel() - 1
    with torch.cuda.device(dev):
        ws = _hip._workspace(_hip.lib().lsrm_window_attn_bwd_workspace_size(
            nq, nk, hq, hkv, d, batch, left, sinks, r), dev)
        _hip._check(_hip.lib().lsrm_window_attn_bwd(
            do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
            low.data_ptr() if low.numel() else None, lse.data_ptr(), _hip._DTYPE_CODE[q.dtype],
            qs, ks, vs, nq, nk, hq, hkv, d,
            cu_q.data_ptr(), cu_k.data_ptr(), batch, left, right, sinks, _hip._ptr(table),
            n_buckets, _hip._ptr(buckets), r, softmax_scale, dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), _hip._ptr(d_table), ws.data_ptr(), ws.numel(), _hip._stream(dev)),
            "lsrm_window_attn_bwd")
    return dq, dk, dv, d_table


def _cache_strides(name, t):
    """(batch, token, head) strides of a cache [B, capacity, Hkv, D]."""
    b, cap, h, d = t.shape
    if t.numel() == 0:
        return 0, 0, 0
    # the stride of a dimension of one element is never used
    strides = [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]
    if (d > 1 and strides[3] != 1) or any(s % 8 for s in strides[:3]) or \
            strides[1] > MAX_STRIDE or t.data_ptr() % 16:
        raise ValueError(f"{name}: channels must be contiguous, the other strides multiples of 8 "
                         "elements and the start 16-byte aligned (a cache is not copied)")
    return strides[0], strides[1], strides[2]


def window_decode(q, k_cache, v_cache, seqlens, left: int, sinks: int,
                  bias_table: Optional[torch.Tensor], bias_buckets: Optional[torch.Tensor],
                  softmax_scale: float):
    """-> (out [B, Hq, D], lse [Hq, B] fp32 in log2 units)."""
    dev = _hip._dev_check(q, k_cache, v_cache, seqlens)
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape or \
            q.shape[0] != k_cache.shape[0] or q.shape[2] != k_cache.shape[3]:
        raise ValueError("q [B, Hq, D], k_cache and v_cache [B, capacity, Hkv, D] expected")
    if q.dtype not in (torch.float16, torch.bfloat16) or k_cache.dtype != q.dtype or \
            v_cache.dtype != q.dtype:
        raise TypeError("q and the caches must share dtype float16 or bfloat16")
    batch, hq, d = q.shape
    _, capacity, hkv, _ = k_cache.shape
    if hkv == 0 or hq % hkv != 0:
        raise ValueError("num_q_heads must be a multiple of num_kv_heads")
    if tuple(seqlens.shape) != (batch,) or seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError("seqlens must be int32 [B]")
    table, buckets, n_buckets, r = bias_args(q, hq, bias_table, bias_buckets)
    q, qs = token_rows(q)
    lens = _hip._i32(seqlens)
    ks, vs = _cache_strides("k_cache", k_cache), _cache_strides("v_cache", v_cache)
    out = torch.empty((batch, hq, d), dtype=q.dtype, device=dev)
    lse = torch.empty((hq, batch), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        ws_n = _hip.lib().lsrm_window_decode_workspace_size(batch, capacity, hq, hkv, d, left,
                                                            sinks)
        ws = _hip._workspace(ws_n, dev) if ws_n else None
        _hip._check(_hip.lib().lsrm_window_decode(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _hip._DTYPE_CODE[q.dtype], qs,
            *ks, *vs, lens.data_ptr(), batch, capacity, hq, hkv, d, left, sinks,
            _hip._ptr(table), n_buckets, _hip._ptr(buckets), r, softmax_scale, out.data_ptr(),
            lse.data_ptr(), _hip._ptr(ws), ws_n, _hip._stream(dev)), "lsrm_window_decode")
    return out, lse
