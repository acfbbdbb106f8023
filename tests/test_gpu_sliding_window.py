"""Sliding-window attention (sparse.ops.sliding_window_attention, HIP
lsrm_window_attn_fwd / _bwd) against its definition in 64 bits: outputs, LSE
and all gradients, each element within the bound that the kernel's roundings
allow (oracle.window: P and dS rounded once, outputs once)."""

import math

import pytest
import torch

import lsrm_hip as H
import sparse.ops as ops
from oracle.window import window_attn_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def _case(lens_q, lens_k, hq, hkv, d, dtype, seed=0, buckets=None, n_buckets=0, tail_q=0,
          tail_k=0):
    """Inputs on the CPU, already of the kernel's type."""
    g = torch.Generator().manual_seed(seed)
    cu = [torch.tensor([0] + list(torch.tensor(x).cumsum(0)), dtype=torch.int32)
          for x in (lens_q, lens_k)]
    nq, nk = int(cu[0][-1]) + tail_q, int(cu[1][-1]) + tail_k
    q, k, v, do = (torch.randn(n, h, d, generator=g).to(DT[dtype])
                   for n, h in ((nq, hq), (nk, hkv), (nk, hkv), (nq, hq)))
    table = None
    if buckets is not None:
        table = torch.randn(n_buckets, hq, generator=g).to(DT[dtype])
    return q, k, v, do, cu[0], cu[1], table


def _run(q, k, v, do, cu_q, cu_k, window, sinks, table, buckets, scale=None):
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    t = None if table is None else table.to(DEV).requires_grad_()
    b = None if buckets is None else buckets.to(DEV)
    out, lse = ops.sliding_window_attention(*leaves, cu_q.to(DEV), cu_k.to(DEV), window, sinks,
                                            t, b, scale, return_lse=True)
    grads = torch.autograd.grad(out, leaves + ([] if t is None else [t]), do.to(DEV))
    torch.cuda.synchronize()
    names = ["dq", "dk", "dv", "dtable"]
    got = {"out": out.detach(), "lse": lse, **dict(zip(names, grads))}
    return {n: x.double().cpu() for n, x in got.items()}


def _check(got, ref, unit):
    lse, want = got["lse"], ref["lse"]
    assert torch.equal(lse == -math.inf, want == -math.inf)
    seen = want > -math.inf
    # the sum of rounded P: a relative error of `unit`, and 32-bit scores
    bound = 1.45 * unit + 2.0 ** -18 * (1 + want[seen].abs())
    assert ((lse[seen] - want[seen]).abs() <= bound).all(), "lse"
    for n in ("out", "dq", "dk", "dv", "dtable"):
        if n not in got:
            continue
        err, bound = (got[n] - ref[n]).abs(), ref[n + "_err"] + 2.0 ** -24
        assert torch.isfinite(got[n]).all(), n
        assert (err <= bound).all(), (n, float((err / bound).max()),
                                      (err > bound).nonzero()[:4].tolist())


def _compare(dtype, lens_q, lens_k, hq, hkv, d, window, sinks, buckets=None, n_buckets=0, seed=0,
             scale=None, tail_q=0, tail_k=0):
    q, k, v, do, cu_q, cu_k, table = _case(lens_q, lens_k, hq, hkv, d, dtype, seed, buckets,
                                           n_buckets, tail_q, tail_k)
    ref = window_attn_ref(q, k, v, cu_q, cu_k, *window, sinks, table, buckets, scale, do,
                          UNIT[dtype])
    got = _run(q, k, v, do, cu_q, cu_k, window, sinks, table, buckets, scale)
    _check(got, ref, UNIT[dtype])


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 2), (8, 2), (3, 1)])
def test_heads_and_types(d, dtype, hq, hkv):
    _compare(dtype, [130, 1, 77], [130, 1, 77], hq, hkv, d, (40, 0), 3)


@pytest.mark.parametrize("window", [(0, 0), (1, 0), (63, 0), (64, 64), (0, 5), (200, 31),
                                    (-1, 0), (-1, -1), (7, -1), (1000, 1000)])
@pytest.mark.parametrize("sinks", [0, 1, 64])
def test_windows_and_first_tokens(window, sinks):
    _compare("bf16", [333, 5, 64], [333, 5, 64], 2, 1, 64, window, sinks)


@pytest.mark.parametrize("lens_q,lens_k", [
    ([1], [1]), ([1], [300]), ([129], [400]), ([3, 0, 2], [100, 7, 2]), ([0], [5]), ([4], [0]),
    ([200], [100]), ([10, 1, 64], [3, 1, 65]), ([1] * 40, list(range(40)))])
@pytest.mark.parametrize("sinks", [0, 4])
def test_lengths(lens_q, lens_k, sinks):
    # more queries than keys leave rows that see nothing; so do empty sequences
    _compare("bf16", lens_q, lens_k, 4, 2, 64, (30, 0), sinks)


@pytest.mark.parametrize("d,hq,hkv", [(64, 2, 2), (32, 8, 1), (128, 2, 1)])
@pytest.mark.parametrize("n_buckets,distance,two_sided", [
    (32, 128, True), (8, 20, False), (2, 3, False), (16, 512, True)])
def test_bias(d, hq, hkv, n_buckets, distance, two_sided):
    buckets = ops.relative_position_buckets(n_buckets, distance, two_sided)
    _compare("bf16", [260, 1, 75], [260, 1, 75], hq, hkv, d, (150, 90 if two_sided else 0), 5,
             buckets, n_buckets)


def test_bias_of_a_single_position_and_any_map():
    _compare("fp16", [100], [100], 2, 2, 64, (20, 3), 2, torch.tensor([1], dtype=torch.int32), 3)
    g = torch.Generator().manual_seed(5)
    buckets = torch.randint(0, 7, (41,), generator=g).to(torch.int32)
    _compare("bf16", [150, 90], [200, 90], 4, 4, 32, (60, 60), 4, buckets, 7)


def test_scale_and_rows_behind_the_last_sequence():
    _compare("bf16", [100, 30], [90, 60], 2, 2, 64, (25, 2), 2, scale=0.31, tail_q=150,
             tail_k=140)


def test_first_tokens_of_long_sequences():
    # several partial sums per sequence for the gradients of the first tokens
    _compare("bf16", [1700, 600], [1700, 600], 2, 1, 32, (64, 0), 7)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("left", [0, 1, 2])
@pytest.mark.parametrize("few_bits", [True, False])
def test_bits_behind_the_rounding(d, dtype, left, few_bits):
    # with q = 0 a row is the mean of its keys' values: P = 1 exactly, so the
    # sum and the division are 32-bit; of two values it often lies half way
    # between two numbers of 16 bits
    _, k, v, _, cu, _, _ = _case([150], [150], 4, 2, d, dtype)
    if few_bits:  # sums that are exact in 16 bits, zeros of equal and opposite values
        v.mul_(8).round_()
    out, _, low = torch.ops.lsrm_hip.window_attn_fwd(
        torch.zeros(150, 4, d, dtype=DT[dtype], device=DEV), k.to(DEV), v.to(DEV), cu.to(DEV),
        cu.to(DEV), left, 0, 0, None, None, 0.125, True)
    # bytes of a row: eight columns of every sixteen, then the other eight
    low = low.cpu().view(150, 4, 2, d // 16, 8).transpose(2, 3).reshape(150, 4, d)
    bits = out.cpu().float().view(torch.int32)
    got = (bits + low.int() * (256 if dtype == "bf16" else 32)).view(torch.float32).double()
    x = v.double().repeat_interleave(2, 1)
    ref = torch.stack([x[max(0, p - left):p + 1].mean(0) for p in range(150)])
    # the bits below the byte (256 or 32 steps of 2^-23 of the value), the 32-bit
    # sum, division and product (a half step each), and in fp16 the step of its
    # subnormal numbers, which the byte does not divide
    bound = (ref.abs() * (2.0 ** -15 if dtype == "bf16" else 2.0 ** -18)
             + torch.stack([x[max(0, p - left):p + 1].abs().mean(0) for p in range(150)])
             * 2.0 ** -22 + (2.0 ** -25 if dtype == "fp16" else 0.0))
    assert ((got - ref).abs() <= bound).all()
    assert (low != 0).any() == (left == 2 or (left == 1 and not few_bits))
