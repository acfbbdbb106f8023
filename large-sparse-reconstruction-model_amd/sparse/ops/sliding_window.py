"""Sliding-window attention with visible first tokens and a learned bias of
the relative position.

Where sparse_window_attention lets every block attend to itself, here the
window follows the token: a query at position p of its sequence sees the keys
p - left .. p + right, and the sequence's first `num_sinks` tokens wherever it
stands.  Sequences are packed as for native_sparse_attend ([total, heads, dim],
int32 offsets); with fewer queries than keys the last query stands at the last
key (new tokens behind a cached past).  sliding_window_decode is the form for
one new token of every sequence against a cache.  Forward and backward run on
gfx950 HIP kernels (eager: lsrm_hip.native(); traced: the operators
torch.ops.lsrm_hip.window_attn_fwd / window_attn_bwd / window_decode).
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

import lsrm_hip as _hip

from . import native_sparse_attention as _nsa
from ._dispatch import eager, needs_grad


def relative_position_buckets(num_buckets: int, max_distance: int, bidirectional: bool = False,
                              device=None) -> torch.Tensor:
    """Bucket of every relative position (key minus query), clamped to
    -max_distance .. max_distance -> int32 [2 * max_distance + 1].

    One side has n = num_buckets positions' worth of buckets (bidirectional:
    half of them for keys behind the query, half for keys ahead; else keys
    ahead share the bucket of distance 0).  Distances below n // 2 have a
    bucket each; bucket n // 2 + b begins at the first distance d with
    log(d / (n // 2)) / log(max_distance / (n // 2)) * (n - n // 2) >= b,
    decided in whole numbers; the last one takes every larger distance."""
    side = num_buckets // 2 if bidirectional else num_buckets
    near = side // 2
    far = side - near
    if near < 1 or (bidirectional and num_buckets % 2) or max_distance <= near:
        raise ValueError("need at least 2 (bidirectional: an even number, 4) buckets and "
                         "max_distance above half of a side's buckets")
    if max_distance > 512:
        raise ValueError("max_distance is at most 512")
    first = []  # first distance of every far bucket after the first one
    d = near
    for b in range(1, far):
        while d ** far * near ** b < max_distance ** b * near ** far:
            d += 1
        first.append(d)
    out = []
    for rel in range(-max_distance, max_distance + 1):
        d = abs(rel) if bidirectional else max(0, -rel)
        bucket = d if d < near else near + sum(d >= f for f in first)
        out.append(bucket + (side if bidirectional and rel > 0 else 0))
    return torch.tensor(out, dtype=torch.int32, device=device)


def sliding_window_attention(
    q: torch.Tensor,  # [total_q, num_q_heads, dim]
    k: torch.Tensor,  # [total_k, num_kv_heads, dim]
    v: torch.Tensor,  # [total_k, num_kv_heads, dim]
    cu_seqlens_q: torch.Tensor,  # [batch_size + 1]
    cu_seqlens_k: torch.Tensor,  # [batch_size + 1]
    window: Tuple[int, int],
    num_sinks: int = 0,
    bias_table: Optional[torch.Tensor] = None,  # [num_buckets, num_q_heads]
    bias_buckets: Optional[torch.Tensor] = None,  # [2 * max_distance + 1]
    softmax_scale: Optional[float] = None,
    return_lse: bool = False,
):
    """Query i of a sequence of Lq queries and Lk keys stands at p = i + Lk -
    Lq and attends to the keys j <= p + right with j >= p - left or j <
    num_sinks; window = (left, right), -1 for no bound on a side ((left, 0) is
    causal).  With a bias, score(i, j) = scale q.k + bias_table[bias_buckets[
    clamp(j - p)], head] (relative_position_buckets; entries below -1e30 mask).

    Returns out [total_q, num_q_heads, dim] (and lse [num_q_heads, total_q],
    fp32, log2 units, not differentiable, when return_lse), differentiable in
    q, k, v and bias_table.  Rows that see no key, and rows behind the last
    sequence, give out = 0, lse = -inf and no gradients."""
    left, right = (int(x) for x in window)
    if left < -1 or right < -1:
        raise ValueError("window sides must be >= 0, or -1 for no bound")
    if not 0 <= num_sinks <= 64:
        raise ValueError("num_sinks must be in 0 .. 64")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(q.shape[-1])
    if not 0.0 < softmax_scale < math.inf:
        raise ValueError("softmax_scale must be positive")
    args = (q, k, v, cu_seqlens_q, cu_seqlens_k, left, right, int(num_sinks), bias_table,
            bias_buckets, float(softmax_scale))
    if eager(q, k, v, cu_seqlens_q, cu_seqlens_k, bias_table, bias_buckets):
        # The kernels take any offsets (they clamp what they read), so they run
        # while the host waits for the check (none under graph capture).
        out, lse, bits = _hip.native().window_attention(*args, return_lse,
                                                             _nsa._validate)
        if bits:
            raise ValueError(
                f"invalid sliding-window metadata: {_hip.describe_meta_error(bits)}")
    else:
        _hip.window.check_qkv(q, k, v)
        out, lse, _low = torch.ops.lsrm_hip.window_attn_fwd(
            *args, needs_grad(q, k, v, bias_table))
    return (out, lse) if return_lse else out


def sliding_window_decode(
    q: torch.Tensor,  # [batch, num_q_heads, dim]
    k_cache: torch.Tensor,  # [batch, capacity, num_kv_heads, dim]
    v_cache: torch.Tensor,  # [batch, capacity, num_kv_heads, dim]
    seqlens: torch.Tensor,  # [batch]
    window_left: int,
    num_sinks: int = 0,
    bias_table: Optional[torch.Tensor] = None,  # [num_buckets, num_q_heads]
    bias_buckets: Optional[torch.Tensor] = None,  # [2 * max_distance + 1]
    softmax_scale: Optional[float] = None,
    return_lse: bool = False,
):
    """One query per sequence, at the last of its seqlens[b] cached tokens (its
    own key and value among them): the row that sliding_window_attention with
    window (window_left, 0) gives there.  -1: no bound on the left.

    Lengths are read on the device and clamped to 0 .. capacity (no host
    synchronisation, so the call can be captured and replayed with lengths
    that grow); an empty sequence gives out = 0, lse = -inf.  Caches may have
    any strides with contiguous channels and are read only where the query
    sees them.  Returns out [batch, num_q_heads, dim] (and lse [num_q_heads,
    batch], fp32, log2 units, when return_lse); for inference."""
    if window_left < -1:
        raise ValueError("window_left must be >= 0, or -1 for no bound")
    if not 0 <= num_sinks <= 64:
        raise ValueError("num_sinks must be in 0 .. 64")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(q.shape[-1])
    if not 0.0 < softmax_scale < math.inf:
        raise ValueError("softmax_scale must be positive")
    if needs_grad(q, k_cache, v_cache, bias_table):
        raise RuntimeError("sliding_window_decode has no backward; call it under no_grad")
    args = (q, k_cache, v_cache, seqlens, int(window_left), int(num_sinks), bias_table,
            bias_buckets, float(softmax_scale))
    if eager(q, k_cache, v_cache, seqlens, bias_table, bias_buckets):
        out, lse = _hip.native().window_decode(*args, return_lse)
    else:
        out, lse = torch.ops.lsrm_hip.window_decode(*args)
    return (out, lse) if return_lse else out
