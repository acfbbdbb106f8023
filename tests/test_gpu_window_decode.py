"""Sliding-window attention of single tokens against a cache
(sparse.ops.sliding_window_decode, HIP lsrm_window_decode) against the 64-bit
definition, each element within the bound of the kernel's roundings."""

import math

import pytest
import torch

import sparse.ops as ops
from oracle.window import window_attn_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def _inputs(lens, capacity, hq, hkv, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    q = torch.randn(b, hq, d, generator=g).to(DT[dtype])
    k, v = (torch.randn(b, capacity, hkv, d, generator=g).to(DT[dtype]) for _ in range(2))
    return q, k, v, torch.tensor(lens, dtype=torch.int32)


def _reference(q, k, v, lens, left, sinks, table, buckets, unit, scale=None):
    """Every sequence as one query behind its tokens, packed."""
    n = lens.clamp(0, k.shape[1]).tolist()
    cu_k = torch.tensor([0] + n).cumsum(0)
    cu_q = torch.tensor([0] + [min(1, x) for x in n]).cumsum(0)
    some = lens > 0
    pick = lambda t: torch.cat([t[b, :x] for b, x in enumerate(n)])  # noqa: E731
    ref = window_attn_ref(q[some], pick(k), pick(v), cu_q, cu_k, left, 0, sinks, table, buckets,
                          scale, unit=unit)
    out = {}
    for name in ("out", "out_err"):
        out[name] = torch.zeros(q.shape, dtype=torch.float64)
        out[name][some] = ref[name]
    out["lse"] = torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64)
    out["lse"][:, some] = ref["lse"]
    return out


def _check(out, lse, ref, unit):
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(lse == -math.inf, ref["lse"] == -math.inf)
    seen = ref["lse"] > -math.inf
    bound = 1.45 * unit + 2.0 ** -18 * (1 + ref["lse"][seen].abs())
    assert ((lse[seen] - ref["lse"][seen]).abs() <= bound).all()
    assert torch.isfinite(out).all()
    over = (out - ref["out"]).abs() > ref["out_err"] + 2.0 ** -24
    assert not over.any(), over.nonzero()[:4].tolist()


def _compare(lens, capacity, hq, hkv, d, left, sinks, dtype="bf16", buckets=None, n_buckets=0,
             seed=0, scale=None):
    q, k, v, n = _inputs(lens, capacity, hq, hkv, d, dtype, seed)
    table = None
    if buckets is not None:
        table = torch.randn(n_buckets, hq, generator=torch.Generator().manual_seed(seed + 1)).to(
            DT[dtype])
    ref = _reference(q, k, v, n, left, sinks, table, buckets, UNIT[dtype], scale)
    # what is not seen holds NaN
    at = torch.arange(capacity)[None, :]
    last = n[:, None].clamp(0, capacity) - 1
    seen = (at <= last) & ((at >= last - left) | (at < sinks) | (left < 0))
    for t in (k, v):
        t[~seen] = math.nan
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    out, lse = ops.sliding_window_decode(dev(q), dev(k), dev(v), dev(n), left, sinks, dev(table),
                                         dev(buckets), scale, return_lse=True)
    _check(out, lse, ref, UNIT[dtype])


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2), (3, 1), (33, 1), (80, 2)])
def test_heads_and_types(d, dtype, hq, hkv):
    _compare([1, 0, 100, 33], 100, hq, hkv, d, 50, 3, dtype)


@pytest.mark.parametrize("left", [0, 1, 31, 32, 500, -1])
@pytest.mark.parametrize("sinks", [0, 1, 32, 33, 64])
def test_windows(left, sinks):
    _compare([1, 2, 31, 32, 33, 64, 65, 97, 200, 399, 400], 400, 2, 1, 64, left, sinks)


def test_lengths_beyond_the_cache_and_below_zero_are_clamped():
    _compare([500, 10, -3], 40, 4, 2, 64, 20, 2)


def test_no_sequences_and_no_capacity():
    e = torch.empty(0, 4, 64, device=DEV, dtype=torch.bfloat16)
    c = torch.empty(0, 10, 2, 64, device=DEV, dtype=torch.bfloat16)
    n = torch.empty(0, dtype=torch.int32, device=DEV)
    assert ops.sliding_window_decode(e, c, c, n, 5).shape == (0, 4, 64)
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    c = torch.empty(3, 0, 2, 64, device=DEV, dtype=torch.bfloat16)
    out, lse = ops.sliding_window_decode(q, c, c, torch.tensor([0, 1, 5], device=DEV), 5,
                                         return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("lens", [[4097], [3000, 4500, 17]])
@pytest.mark.parametrize("left,sinks", [(4000, 4), (-1, 0)])
def test_long_windows_split_between_workgroups(lens, left, sinks):
    for d, hq, hkv in ((64, 4, 1), (128, 8, 8)):
        _compare(lens, 4600, hq, hkv, d, left, sinks)


@pytest.mark.parametrize("n_buckets,distance", [(32, 128), (8, 20), (2, 3), (16, 512)])
def test_bias(n_buckets, distance):
    buckets = ops.relative_position_buckets(n_buckets, distance)
    _compare([1, 0, 40, 300, 700], 700, 8, 2, 64, 400, 5, "bf16", buckets, n_buckets, 2)
    _compare([1, 700], 700, 40, 1, 32, 690, 0, "fp16", buckets, n_buckets, 3, 0.2)


def test_strides_and_the_packed_operator():
    # a head-major cache, queries that are a slice of a projection, int64 lengths
    g = torch.Generator().manual_seed(4)
    b, cap, hq, hkv, d = 5, 300, 8, 2, 64
    qkv = torch.randn(b, hq + 2 * hkv, d, generator=g).bfloat16().to(DEV)
    store = torch.randn(2, b, hkv, cap, d, generator=g).bfloat16().to(DEV)
    k, v = store[0].transpose(1, 2), store[1].transpose(1, 2)
    lens = torch.tensor([300, 1, 77, 129, 256], device=DEV)
    out = ops.sliding_window_decode(qkv[:, :hq], k, v, lens, 100, 4)
    again = ops.sliding_window_decode(qkv[:, :hq].contiguous(), k.contiguous(), v.contiguous(),
                                      lens.int(), 100, 4)
    assert torch.equal(out, again)
    ref = _reference(qkv[:, :hq].cpu(), k.cpu(), v.cpu(), lens.cpu().int(), 100, 4, None, None,
                     UNIT["bf16"])
    over = (out.double().cpu() - ref["out"]).abs() > ref["out_err"]
    assert not over.any()


def test_refusals():
    q = torch.zeros(2, 4, 64, device=DEV, dtype=torch.bfloat16)
    c = torch.zeros(2, 16, 2, 64, device=DEV, dtype=torch.bfloat16)
    n = torch.ones(2, dtype=torch.int32, device=DEV)
    dec = ops.sliding_window_decode
    with pytest.raises(ValueError, match="window_left"):
        dec(q, c, c, n, -2)
    with pytest.raises(ValueError, match="num_sinks"):
        dec(q, c, c, n, 5, 65)
    with pytest.raises(ValueError, match="seqlens"):
        dec(q, c, c, n[:1], 5)
    with pytest.raises(ValueError, match="expected"):
        dec(q, c[:1], c[:1], n, 5)
    with pytest.raises(TypeError):
        dec(q.float(), c.float(), c.float(), n, 5)
    with pytest.raises(ValueError, match="multiple"):
        dec(q[:, :3], c, c, n, 5)
    with pytest.raises(ValueError, match="strides"):
        odd = torch.zeros(2, 16, 2, 65, device=DEV, dtype=torch.bfloat16)[..., :64]
        dec(q, odd, odd, n, 5)
    with pytest.raises(ValueError, match="go together"):
        dec(q, c, c, n, 5, bias_table=torch.zeros(4, 4, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="no_grad"):
        dec(q.clone().requires_grad_(), c, c, n, 5)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dec(q.cpu(), c.cpu(), c.cpu(), n.cpu(), 5)


@pytest.mark.parametrize("lens,capacity", [([40000], 40005), ([50], 40005), ([639], 639),
                                           ([640], 640), ([9000, 641, 0], 9000)])
def test_parts_that_are_many_or_empty(lens, capacity):
    for d, hq, hkv in ((64, 4, 1), (32, 2, 2)):
        _compare(lens, capacity, hq, hkv, d, -1, 0)
