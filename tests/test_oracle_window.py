"""Pins of oracle.window: visibility against the rule spelt out pair by pair,
gradients against torch autograd and against differences, the bucket map of
sparse.ops.relative_position_buckets against the logarithm's formula."""

import math

import pytest
import torch

import sparse.ops as ops
from oracle.window import bias_map, visible, window_attn_ref


@pytest.mark.parametrize("lq,lk", [(1, 1), (5, 9), (9, 5), (7, 7)])
@pytest.mark.parametrize("left,right,sinks", [(0, 0, 0), (2, 0, 1), (3, 2, 2), (-1, 0, 0),
                                              (1, -1, 3), (-1, -1, 4)])
def test_visible_pair_by_pair(lq, lk, left, right, sinks):
    got = visible(lq, lk, left, right, sinks)
    for i in range(lq):
        for j in range(lk):
            p = i + lk - lq
            want = (right < 0 or j <= p + right) and (left < 0 or j >= p - left or j < sinks)
            assert bool(got[i, j]) == want, (i, j)


def _inputs(seed=0):
    g = torch.Generator().manual_seed(seed)
    cu_q, cu_k = torch.tensor([0, 6, 7, 12]), torch.tensor([0, 4, 9, 14])
    q, do = (torch.randn(13, 4, 8, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(15, 2, 8, generator=g, dtype=torch.float64) for _ in range(2))
    table = torch.randn(6, 4, generator=g, dtype=torch.float64)
    buckets = torch.randint(0, 6, (7,), generator=g)
    return q, k, v, do, cu_q, cu_k, table, buckets


def _dense(q, k, v, cu_q, cu_k, left, right, sinks, table, buckets):
    """One softmax over a block-diagonal mask, by torch."""
    nq, hq, d = q.shape
    nk, hkv, _ = k.shape
    seen = torch.zeros(nq, nk, dtype=torch.bool)
    where = torch.zeros(nq, nk, dtype=torch.long)
    for a, b, c, e in zip(cu_q[:-1], cu_q[1:], cu_k[:-1], cu_k[1:]):
        seen[a:b, c:e] = visible(int(b - a), int(e - c), left, right, sinks)
        where[a:b, c:e] = bias_map(int(b - a), int(e - c), buckets)
    kk, vv = (t.repeat_interleave(hq // hkv, 1) for t in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, kk) / math.sqrt(d) + table[where].permute(2, 0, 1)
    some = seen.any(-1)
    p = torch.softmax(s.masked_fill(~seen, -math.inf)[:, some], -1)
    out = torch.zeros(hq, nq, d, dtype=q.dtype).index_put(
        (torch.arange(hq)[:, None], some.nonzero()[:, 0][None]), p @ vv.transpose(0, 1))
    return out.transpose(0, 1)


@pytest.mark.parametrize("left,right,sinks", [(2, 0, 1), (1, 1, 0), (-1, 0, 0)])
def test_outputs_and_gradients_against_autograd(left, right, sinks):
    q, k, v, do, cu_q, cu_k, table, buckets = _inputs()
    ref = window_attn_ref(q, k, v, cu_q, cu_k, left, right, sinks, table, buckets, do=do)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    out = _dense(*leaves[:3], cu_q, cu_k, left, right, sinks, leaves[3], buckets)
    assert torch.allclose(out, ref["out"], rtol=1e-12, atol=1e-12)
    for name, grad in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, do)):
        assert torch.allclose(grad, ref[name], rtol=1e-11, atol=1e-11), name


def test_gradients_against_differences():
    q, k, v, do, cu_q, cu_k, table, buckets = _inputs(1)
    args = (cu_q, cu_k, 2, 1, 1)
    ref = window_attn_ref(q, k, v, *args, table, buckets, do=do)
    g = torch.Generator().manual_seed(3)
    step = 1e-6
    for name, at in (("dq", 0), ("dk", 1), ("dv", 2), ("dtable", 3)):
        tensors = [q, k, v, table]
        way = torch.randn(tensors[at].shape, generator=g, dtype=torch.float64)
        loss = []
        for sign in (1, -1):
            moved = list(tensors)
            moved[at] = tensors[at] + sign * step * way
            out = window_attn_ref(*moved[:3], *args, moved[3], buckets)["out"]
            loss.append(float((out * do).sum()))
        want = float((ref[name] * way).sum())
        assert abs((loss[0] - loss[1]) / (2 * step) - want) < 1e-6 * (1 + abs(want)), name


def test_empty_rows_and_masked_buckets():
    q, k, v, do, cu_q, cu_k, table, buckets = _inputs(2)
    table[:, 1] = -math.inf
    table[:, 2] = torch.finfo(torch.bfloat16).min
    ref = window_attn_ref(q, k, v, cu_q, cu_k, 2, 0, 1, table, buckets, do=do)
    for h in (1, 2):
        assert (ref["out"][:, h] == 0).all() and (ref["lse"][h] == -math.inf).all()
        assert (ref["dtable"][:, h] == 0).all()
    assert (ref["lse"][0, :2] == -math.inf).all()  # 6 queries over 4 keys
    assert (ref["out"][12:] == 0).all() and (ref["dk"][14:] == 0).all()


@pytest.mark.parametrize("n,distance,two_sided", [(32, 128, True), (32, 128, False),
                                                  (8, 20, False), (6, 3, True), (2, 3, False),
                                                  (64, 512, True), (4, 512, False)])
def test_bucket_map(n, distance, two_sided):
    got = ops.relative_position_buckets(n, distance, two_sided)
    assert got.dtype == torch.int32 and got.numel() == 2 * distance + 1
    side = n // 2 if two_sided else n
    near = side // 2
    for i, rel in enumerate(range(-distance, distance + 1)):
        d = abs(rel) if two_sided else max(0, -rel)
        b = int(got[i]) - (side if two_sided and rel > 0 else 0)
        if d < near:
            assert b == d
            continue
        x = math.log(d / near) / math.log(distance / near) * (side - near)
        # the whole number below, where 64 bits can tell
        if abs(x - round(x)) > 1e-9:
            assert b == near + min(side - near - 1, math.floor(x)), (rel, x)
        else:
            assert b == near + min(side - near - 1, round(x)), (rel, x)
    assert int(got.max()) <= n - 1 and int(got.min()) == 0


def test_bucket_map_refusals():
    for args in ((1, 10, False), (2, 10, True), (7, 10, True), (32, 8, False), (8, 600, False)):
        with pytest.raises(ValueError):
            ops.relative_position_buckets(*args)
