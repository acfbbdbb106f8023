"""The C ABI registered as PyTorch operators (namespace ``lsrm_hip``).

Each operator wraps one lsrm_hip call (which goes through liblsrm_hip.so):
the dispatcher sees it as an opaque kernel with a schema, a fake (meta)
implementation for shape propagation (torch.compile, FakeTensor, meta
tensors) and, for the two differentiable ones, an autograd formula.  The
sparse.ops front end routes every call through ``torch.ops.lsrm_hip.*``.

Operators (the reference interface each one stands in for):
  sel_attn_fwd     kvcentric:931-1010   native_sparse_attn_forward -> (o, lse)
  sel_attn_bwd     kvcentric:1018-1263  native_sparse_attn_backward -> (dq, dk, dv, delta)
  block_mean_pool  spatial_sparse_attention.py:27-37  sparse3d_compression
  block_mean_pool2 spatial_sparse_attention.py:49-66  the key and value pair
  select_blocks    the benchmark's per-query-block selection -> (topk_idx, compact)
  block_score      block_score.py:16-98  get_block_score
  gate_merge       spatial_sparse_attention.py:256-269 (the gated branch sum)
  gate_merge_bwd   its gradients -> [d_gate, d_cmp, d_slc(, d_win)]
  window_attn_fwd  sliding-window attention with visible first tokens and a
                   learned relative position bias -> (o, lse, o_low)
  window_attn_bwd  its gradients -> [dq, dk, dv(, d_table)]
  window_decode    the same for single query tokens against a cache -> (o, lse)
  residual_norm_fwd  dropout, residual addition and root-mean-square norm
                   -> (y, h, rstd, rng_used)
  residual_norm_bwd  its gradients -> [(dx,) d_residual, d_weight]
  residual_norm_fp8  the norm's rows in 8 bits -> (y8, scales, h)
  block_ids        the self-block rows of sparse_window_attention
                   (block_window_attention.py:14-31)
Tensors on the CPU raise (there is no CPU implementation).
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import (
    block_ids as _block_ids,
    block_mean_pool as _block_mean_pool,
    block_mean_pool2 as _block_mean_pool2,
    block_score as _block_score,
    gate_merge as _gate_merge,
    gate_merge_bwd as _gate_merge_bwd,
    sel_attn_bwd as _sel_attn_bwd,
    sel_attn_fwd as _sel_attn_fwd,
    residual_norm_bwd as _residual_norm_bwd,
    residual_norm_fp8 as _residual_norm_fp8,
    residual_norm_fwd as _residual_norm_fwd,
    select_blocks as _select_blocks,
    window_attn_bwd as _window_attn_bwd,
    window_attn_fwd as _window_attn_fwd,
    window_decode as _window_decode,
)

NS = "lsrm_hip"


# ------------------------------------------------------------- attention --

@torch.library.custom_op(f"{NS}::sel_attn_fwd", mutates_args=())
def sel_attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, topk_idx: torch.Tensor,
                 cu_seqblocks: torch.Tensor, cu_block_tokens: torch.Tensor,
                 cu_seqlens_q: torch.Tensor, softmax_scale: float, key_centric: bool = False
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """out [Nq, Hq, D] (q's dtype), lse [Hq, Nq] fp32 in log2 units
    (key_centric: the key-centric plan for per-token rows without locality)."""
    return _sel_attn_fwd(q, k, v, topk_idx, cu_seqblocks, cu_block_tokens, cu_seqlens_q,
                         softmax_scale, key_centric)


@sel_attn_fwd.register_fake
def _(q, k, v, topk_idx, cu_seqblocks, cu_block_tokens, cu_seqlens_q, softmax_scale,
      key_centric=False):
    return torch.empty_like(q), q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32)


@torch.library.custom_op(f"{NS}::sel_attn_bwd", mutates_args=())
def sel_attn_bwd(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                 o: torch.Tensor, lse: torch.Tensor, topk_idx: torch.Tensor,
                 cu_seqblocks: torch.Tensor, cu_block_tokens: torch.Tensor,
                 cu_seqlens_q: torch.Tensor, softmax_scale: float, key_centric: bool = False
                 ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv, delta [Hq, Nq] fp32 = rowsum(o * do))."""
    return _sel_attn_bwd(do, q, k, v, o, lse, topk_idx, cu_seqblocks, cu_block_tokens,
                         cu_seqlens_q, softmax_scale, key_centric)


@sel_attn_bwd.register_fake
def _(do, q, k, v, o, lse, topk_idx, cu_seqblocks, cu_block_tokens, cu_seqlens_q,
      softmax_scale, key_centric=False):
    return (torch.empty_like(q), torch.empty_like(k), torch.empty_like(v),
            q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32))


def _fwd_setup(ctx, inputs, output):
    q, k, v, topk_idx, cu_seqblocks, cu_block_tokens, cu_seqlens_q, scale = inputs[:8]
    o, lse = output
    ctx.save_for_backward(q, k, v, o, lse, topk_idx, cu_seqblocks, cu_block_tokens,
                          cu_seqlens_q)
    ctx.scale = scale
    ctx.key_centric = bool(inputs[8]) if len(inputs) > 8 else False


def _fwd_backward(ctx, do, _dlse):
    q, k, v, o, lse, topk_idx, cu_seqblocks, cu_block_tokens, cu_seqlens_q = ctx.saved_tensors
    dq, dk, dv, _ = torch.ops.lsrm_hip.sel_attn_bwd(
        do.contiguous().to(q.dtype), q, k, v, o, lse, topk_idx, cu_seqblocks, cu_block_tokens,
        cu_seqlens_q, ctx.scale, ctx.key_centric)
    return dq, dk, dv, None, None, None, None, None, None


sel_attn_fwd.register_autograd(_fwd_backward, setup_context=_fwd_setup)


# ------------------------------------------------------ sliding windows --

@torch.library.custom_op(f"{NS}::window_attn_fwd", mutates_args=())
def window_attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor, left: int,
                    right: int, sinks: int, bias_table: Optional[torch.Tensor],
                    bias_buckets: Optional[torch.Tensor], softmax_scale: float,
                    with_low: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """out [Nq, Hq, D] (q's dtype), lse [Hq, Nq] fp32 in log2 units, out_low
    int8 (empty without with_low; calls that will be differentiated want it)."""
    return _window_attn_fwd(q, k, v, cu_seqlens_q, cu_seqlens_k, left, right, sinks, bias_table,
                            bias_buckets, softmax_scale, with_low)


@window_attn_fwd.register_fake
def _(q, k, v, cu_seqlens_q, cu_seqlens_k, left, right, sinks, bias_table, bias_buckets,
      softmax_scale, with_low=False):
    return (q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32),
            q.new_empty(q.shape if with_low else (0,), dtype=torch.int8))


@torch.library.custom_op(f"{NS}::window_attn_bwd", mutates_args=())
def window_attn_bwd(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    o: torch.Tensor, low: torch.Tensor, lse: torch.Tensor,
                    cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor, left: int,
                    right: int, sinks: int, bias_table: Optional[torch.Tensor],
                    bias_buckets: Optional[torch.Tensor],
                    softmax_scale: float) -> List[torch.Tensor]:
    """[dq, dk, dv] (+ [d_table] when bias_table is given)."""
    out = _window_attn_bwd(do, q, k, v, o, low, lse, cu_seqlens_q, cu_seqlens_k, left, right, sinks,
                           bias_table, bias_buckets, softmax_scale)
    return [t for t in out if t is not None]


@window_attn_bwd.register_fake
def _(do, q, k, v, o, low, lse, cu_seqlens_q, cu_seqlens_k, left, right, sinks, bias_table,
      bias_buckets, softmax_scale):
    out = [q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)]
    if bias_table is not None:
        out.append(bias_table.new_empty(bias_table.shape))
    return out


def _window_setup(ctx, inputs, output):
    (q, k, v, cu_q, cu_k, ctx.left, ctx.right, ctx.sinks, table, buckets, ctx.scale) = inputs[:11]
    o, lse, low = output
    ctx.mark_non_differentiable(lse, low)
    ctx.biased = table is not None
    ctx.save_for_backward(q, k, v, o, low, lse, cu_q, cu_k,
                          *([table, buckets] if ctx.biased else []))


def _window_backward(ctx, do, _dlse, _dlow):
    q, k, v, o, low, lse, cu_q, cu_k, *bias = ctx.saved_tensors
    grads = torch.ops.lsrm_hip.window_attn_bwd(
        do.to(q.dtype), q, k, v, o, low, lse, cu_q, cu_k, ctx.left, ctx.right, ctx.sinks,
        *(bias if ctx.biased else (None, None)), ctx.scale)
    return (grads[0], grads[1], grads[2], None, None, None, None, None,
            grads[3] if ctx.biased else None, None, None, None)


window_attn_fwd.register_autograd(_window_backward, setup_context=_window_setup)


@torch.library.custom_op(f"{NS}::window_decode", mutates_args=())
def window_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  seqlens: torch.Tensor, left: int, sinks: int,
                  bias_table: Optional[torch.Tensor], bias_buckets: Optional[torch.Tensor],
                  softmax_scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """out [B, Hq, D] (q's dtype), lse [Hq, B] fp32 in log2 units."""
    return _window_decode(q, k_cache, v_cache, seqlens, left, sinks, bias_table, bias_buckets,
                          softmax_scale)


@window_decode.register_fake
def _(q, k_cache, v_cache, seqlens, left, sinks, bias_table, bias_buckets, softmax_scale):
    return q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32)


# --------------------------------------------------- pooling, selection --

@torch.library.custom_op(f"{NS}::block_mean_pool", mutates_args=())
def block_mean_pool(x: torch.Tensor, cu_block_tokens: torch.Tensor,
                    out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """[N, C] -> [n_blocks, C] block means (bit-exact contract of
    lsrm_block_mean_pool)."""
    return _block_mean_pool(x, cu_block_tokens, out_dtype)


@block_mean_pool.register_fake
def _(x, cu_block_tokens, out_dtype=None):
    return x.new_empty((cu_block_tokens.shape[0] - 1, x.shape[1]), dtype=out_dtype or x.dtype)


@torch.library.custom_op(f"{NS}::block_mean_pool2", mutates_args=())
def block_mean_pool2(x_a: torch.Tensor, x_b: torch.Tensor, cu_block_tokens: torch.Tensor,
                     out_a_dtype: Optional[torch.dtype] = None,
                     out_b_dtype: Optional[torch.dtype] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of one block partition in one launch pair (each
    output equals block_mean_pool of its input)."""
    return _block_mean_pool2(x_a, x_b, cu_block_tokens, out_a_dtype, out_b_dtype)


@block_mean_pool2.register_fake
def _(x_a, x_b, cu_block_tokens, out_a_dtype=None, out_b_dtype=None):
    nb = cu_block_tokens.shape[0] - 1
    return (x_a.new_empty((nb, x_a.shape[1]), dtype=out_a_dtype or x_a.dtype),
            x_b.new_empty((nb, x_b.shape[1]), dtype=out_b_dtype or x_b.dtype))


@torch.library.custom_op(f"{NS}::select_blocks", mutates_args=())
def select_blocks(q: torch.Tensor, k: torch.Tensor, cu_seqblocks: torch.Tensor,
                  cu_block_tokens: torch.Tensor, topk: int, forced_blocks: List[int],
                  force_self: bool, pooled_k: Optional[torch.Tensor] = None
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(topk_idx [Hkv, N, topk], compact [Hkv, n_blocks, topk]) int32."""
    return _select_blocks(q, k, cu_seqblocks, cu_block_tokens, topk, forced_blocks,
                          force_self, pooled_k)


@select_blocks.register_fake
def _(q, k, cu_seqblocks, cu_block_tokens, topk, forced_blocks, force_self, pooled_k=None):
    hkv, n, nb = k.shape[1], q.shape[0], cu_block_tokens.shape[0] - 1
    return (q.new_empty((hkv, n, topk), dtype=torch.int32),
            q.new_empty((hkv, nb, topk), dtype=torch.int32))


@torch.library.custom_op(f"{NS}::block_score", mutates_args=())
def block_score(q: torch.Tensor, compressed_k: torch.Tensor, lse: torch.Tensor, topk: int,
                cu_seqlens_q: torch.Tensor, compressed_cu_seqlens: torch.Tensor,
                sm_scale: float) -> torch.Tensor:
    """get_block_score -> [Hkv, Nq, topk] int32."""
    return _block_score(q, compressed_k, lse, topk, cu_seqlens_q, compressed_cu_seqlens,
                        sm_scale)


@block_score.register_fake
def _(q, compressed_k, lse, topk, cu_seqlens_q, compressed_cu_seqlens, sm_scale):
    return q.new_empty((compressed_k.shape[1], q.shape[0], topk), dtype=torch.int32)


@torch.library.custom_op(f"{NS}::block_ids", mutates_args=())
def block_ids(cu_seqblocks: torch.Tensor, cu_block_tokens: torch.Tensor, n_tokens: int,
              hkv: int) -> torch.Tensor:
    """Batch-local block id of every token, [hkv, n_tokens, 1] int32."""
    return _block_ids(cu_seqblocks, cu_block_tokens, n_tokens, hkv)


@block_ids.register_fake
def _(cu_seqblocks, cu_block_tokens, n_tokens, hkv):
    return cu_block_tokens.new_empty((hkv, n_tokens, 1), dtype=torch.int32)


# ------------------------------------------------------------ gate merge --

@torch.library.custom_op(f"{NS}::gate_merge", mutates_args=())
def gate_merge(gate: torch.Tensor, o_cmp: torch.Tensor, o_slc: torch.Tensor,
               o_win: Optional[torch.Tensor] = None) -> torch.Tensor:
    return _gate_merge(gate, o_cmp, o_slc, o_win)


@gate_merge.register_fake
def _(gate, o_cmp, o_slc, o_win=None):
    return torch.empty_like(o_cmp)


@torch.library.custom_op(f"{NS}::gate_merge_bwd", mutates_args=())
def gate_merge_bwd(dout: torch.Tensor, gate: torch.Tensor, o_cmp: torch.Tensor,
                   o_slc: torch.Tensor, o_win: Optional[torch.Tensor] = None
                   ) -> List[torch.Tensor]:
    """[d_gate, d_cmp, d_slc] (+ [d_win] when o_win is given)."""
    out = _gate_merge_bwd(dout, gate, o_cmp, o_slc, o_win)
    return [t for t in out if t is not None]


@gate_merge_bwd.register_fake
def _(dout, gate, o_cmp, o_slc, o_win=None):
    out = [torch.empty_like(gate), torch.empty_like(o_cmp), torch.empty_like(o_slc)]
    if o_win is not None:
        out.append(torch.empty_like(o_win))
    return out


def _gm_setup(ctx, inputs, output):
    gate, o_cmp, o_slc, o_win = inputs
    ctx.has_win = o_win is not None
    ctx.save_for_backward(gate, o_cmp, o_slc, *([o_win] if ctx.has_win else []))


def _gm_backward(ctx, dout):
    saved = ctx.saved_tensors
    grads = torch.ops.lsrm_hip.gate_merge_bwd(dout.contiguous(), *saved)
    return grads[0], grads[1], grads[2], (grads[3] if ctx.has_win else None)


gate_merge.register_autograd(_gm_backward, setup_context=_gm_setup)


# --------------------------------------------------------- residual norm --

@torch.library.custom_op(f"{NS}::residual_norm_fwd", mutates_args=())
def residual_norm_fwd(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                      eps: float, drop_least: int, rng_state: Optional[torch.Tensor]
                      ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """y, h (x's dtype), rstd [rows] fp32, and the generator state used."""
    return _residual_norm_fwd(x, residual, weight, eps, drop_least, rng_state)


@residual_norm_fwd.register_fake
def _(x, residual, weight, eps, drop_least, rng_state):
    return (x.new_empty(x.shape), x.new_empty(x.shape),
            x.new_empty((x.numel() // x.shape[-1],), dtype=torch.float32),
            x.new_empty((2 if drop_least > 0 else 0,), dtype=torch.int64))


@torch.library.custom_op(f"{NS}::residual_norm_bwd", mutates_args=())
def residual_norm_bwd(dy: Optional[torch.Tensor], dh: Optional[torch.Tensor], h: torch.Tensor,
                      weight: torch.Tensor, rstd: torch.Tensor, drop_least: int,
                      rng_used: Optional[torch.Tensor]) -> List[torch.Tensor]:
    """[dx (with dropout only), d_residual, d_weight]."""
    out = _residual_norm_bwd(dy, dh, h, weight, rstd, drop_least, rng_used)
    return [t for t in out if t is not None]


@residual_norm_bwd.register_fake
def _(dy, dh, h, weight, rstd, drop_least, rng_used):
    out = [h.new_empty(h.shape), weight.new_empty(weight.shape)]
    return ([h.new_empty(h.shape)] if drop_least > 0 else []) + out


@torch.library.custom_op(f"{NS}::residual_norm_fp8", mutates_args=())
def residual_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                      eps: float, group: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """y8 (float8_e4m3fn), scales fp32, h."""
    return _residual_norm_fp8(x, residual, weight, eps, group)


@residual_norm_fp8.register_fake
def _(x, residual, weight, eps, group):
    scales = x.shape[:-1] + (x.shape[-1] // group if group else 1,)
    return (x.new_empty(x.shape, dtype=torch.float8_e4m3fn),
            x.new_empty(scales, dtype=torch.float32), x.new_empty(x.shape))


def _rn_setup(ctx, inputs, output):
    _x, residual, weight, _eps, least, _rng = inputs
    _y, h, rstd, used = output
    ctx.mark_non_differentiable(rstd, used)
    ctx.set_materialize_grads(False)
    ctx.least, ctx.has_residual = least, residual is not None
    ctx.save_for_backward(h, weight, rstd, used)


def _rn_backward(ctx, dy, dh, _drstd, _dused):
    h, weight, rstd, used = ctx.saved_tensors
    if dy is None and dh is None:
        return None, None, None, None, None, None
    grads = torch.ops.lsrm_hip.residual_norm_bwd(
        None if dy is None else dy.to(h.dtype), None if dh is None else dh.to(h.dtype), h,
        weight, rstd, ctx.least, used if ctx.least > 0 else None)
    # without dropout x and the residual have one gradient
    return (grads[0], grads[-2] if ctx.has_residual else None, grads[-1], None, None, None)


residual_norm_fwd.register_autograd(_rn_backward, setup_context=_rn_setup)

OPS = ("sel_attn_fwd", "sel_attn_bwd", "block_mean_pool", "block_mean_pool2", "select_blocks",
       "block_score",
       "block_ids", "gate_merge", "gate_merge_bwd", "window_attn_fwd", "window_attn_bwd", "window_decode",
       "residual_norm_fwd", "residual_norm_bwd", "residual_norm_fp8")
