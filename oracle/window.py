"""Sliding-window attention with visible first tokens and a bucketed relative
position bias, by definition in 64 bits, with its gradients and the bounds
that a kernel's roundings put on their errors.

Query i of Lq stands at p = i + Lk - Lq and sees key j where j <= p + right
and (j >= p - left or j < sinks); a negative side has no bound.
"""

from __future__ import annotations

import math

import torch

MASKED = -1e30  # table entries below mask their keys


def visible(lq: int, lk: int, left: int, right: int, sinks: int) -> torch.Tensor:
    """[lq, lk] truth values."""
    rel = torch.arange(lk)[None, :] - (torch.arange(lq) + lk - lq)[:, None]
    seen = torch.ones(lq, lk, dtype=torch.bool)
    if right >= 0:
        seen &= rel <= right
    if left >= 0:
        seen &= (rel >= -left) | (torch.arange(lk) < sinks)[None, :]
    return seen


def bias_map(lq: int, lk: int, buckets: torch.Tensor) -> torch.Tensor:
    """Bucket of every (query, key) pair."""
    r = buckets.numel() // 2
    rel = torch.arange(lk)[None, :] - (torch.arange(lq) + lk - lq)[:, None]
    return buckets.long()[rel.clamp(-r, r) + r]


def _pieces(cu_q, cu_k):
    cq, ck = cu_q.tolist(), cu_k.tolist()
    return [(a, b, c, d) for a, b, c, d in zip(cq, cq[1:], ck, ck[1:])]


def window_attn_ref(q, k, v, cu_q, cu_k, left, right, sinks, table=None, buckets=None,
                    scale=None, do=None, unit=0.0):
    """CPU tensors of any float type -> dict of out, lse (log2 units) and,
    with do, dq, dk, dv, dtable, in 64 bits; and for unit > 0 (the largest
    relative error of one rounding to the kernel's type) an elementwise bound
    "<name>_err" of each: P and dS rounded once for the products, outputs
    rounded once, and the LSE from rounded P."""
    q, k, v = (t.double() for t in (q, k, v))
    nq, hq, d = q.shape
    nk, hkv, _ = k.shape
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    u, tiny = unit, 2.0 ** -18  # tiny: sums and exponentials in 32 bits
    # Values of fp16 below 2^-14 are multiples of 2^-24: P and dS that small are
    # off by up to half of that (in the forward P is relative to a row's
    # reference, whose own P of 1 is part of the sum that divides it).
    step = 2.0 ** -25 if unit == 2.0 ** -11 else 0.0
    r = {"out": torch.zeros(nq, hq, d, dtype=torch.float64),
         "lse": torch.full((hq, nq), -math.inf, dtype=torch.float64)}
    r["out_err"] = torch.zeros_like(r["out"])
    if do is not None:
        do = do.double()
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            r[n], r[n + "_err"] = torch.zeros_like(t), torch.zeros_like(t)
        if table is not None:
            r["dtable"] = torch.zeros(table.shape, dtype=torch.float64)
            r["dtable_err"] = torch.zeros_like(r["dtable"])
    for q0, q1, k0, k1 in _pieces(cu_q, cu_k):
        lq, lk = q1 - q0, k1 - k0
        if lq == 0 or lk == 0:
            continue
        seen = visible(lq, lk, left, right, sinks)
        where = None if table is None else bias_map(lq, lk, buckets)
        for h in range(hq):
            qh, kh, vh = q[q0:q1, h], k[k0:k1, h // g], v[k0:k1, h // g]
            s = scale * qh @ kh.T
            if table is not None:
                b = table.double()[where, h]
                s = s + torch.where(b < MASKED, -math.inf, b)
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            any_ = top > -math.inf
            p = torch.where(any_, (s - torch.where(any_, top, 0.0)).exp(), 0.0)
            total = p.sum(-1, keepdim=True)
            p = torch.where(any_, p / torch.where(any_, total, 1.0), 0.0)
            o = p @ vh
            r["out"][q0:q1, h] = o
            r["lse"][h, q0:q1] = ((top + total.log()) / math.log(2.0))[:, 0]
            # numerator and denominator from rounded P, then one rounding
            met = seen.double() * step
            o_err = (2 * u + tiny) * (p @ vh.abs()) + met @ vh.abs()
            r["out_err"][q0:q1, h] = o_err + u * o.abs()
            if do is None:
                continue
            doh = do[q0:q1, h]
            dp = doh @ vh.T
            ds = p * (dp - (doh * o).sum(-1, keepdim=True))
            r["dq"][q0:q1, h] = scale * ds @ kh
            r["dk"][k0:k1, h // g] += scale * ds.T @ qh
            r["dv"][k0:k1, h // g] += p.T @ doh
            # P is off by the LSE's error (u) and a rounding; the row sum of
            # dO O by the error of the rounded O
            spread = tiny * (doh.abs() @ vh.abs().T) + \
                (doh.abs() * (o_err + u * o.abs())).sum(-1, keepdim=True)
            ds_err = (2 * u + tiny) * ds.abs() + p * spread + met
            r["dq_err"][q0:q1, h] = scale * ds_err @ kh.abs()
            r["dk_err"][k0:k1, h // g] += scale * ds_err.T @ qh.abs()
            r["dv_err"][k0:k1, h // g] += (2 * u + tiny) * (p.T @ doh.abs()) + \
                met.T @ doh.abs()
            if table is not None:
                r["dtable"][:, h].index_add_(0, where.reshape(-1), ds.reshape(-1))
                r["dtable_err"][:, h].index_add_(0, where.reshape(-1), ds_err.reshape(-1))
    if do is not None:
        for n in ("dq", "dk", "dv", "dtable"):
            if n in r:
                r[n + "_err"] = 1.01 * r[n + "_err"] + u * r[n].abs()
    r["out_err"] *= 1.01
    return r
