"""The window and norm operators as a model uses them: strided inputs, other
streams, captured graphs, tracing, refused metadata, values that are not finite
in masked places, offsets beyond 32 bits, and a block's window branch run
whole, in training and token by token."""

import math

import pytest
import torch

import lsrm_hip as H
import sparse.ops as ops
from oracle.norm import dropout_mask
from oracle.window import window_attn_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -8  # one rounding to bf16


def _cu(*lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)


def _rand(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _reference(q, k, v, cu_q, cu_k, window, sinks, table=None, buckets=None, do=None, unit=U):
    cpu = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    return window_attn_ref(cpu(q), cpu(k), cpu(v), cpu(cu_q), cpu(cu_k), *window, sinks,
                           cpu(table), cpu(buckets), None, cpu(do), unit)


def _within(got, ref, name):
    err = (got.detach().double().cpu() - ref[name]).abs()
    assert (err <= ref[name + "_err"] + 2.0 ** -24).all(), (name, float(err.max()))


# ------------------------------------------------------------ memory layouts --

def test_slices_of_a_fused_projection_and_broadcast_inputs():
    n, hq, hkv, d = 200, 4, 2, 64
    cu = _cu(120, 80)
    qkv = _rand(n, hq + 2 * hkv, d, seed=1).requires_grad_()
    do = _rand(n, hq, d, seed=2)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    out = ops.sliding_window_attention(q, k, v, cu, cu, (50, 0), 2)
    (grad,) = torch.autograd.grad(out, [qkv], do)
    dense = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
    out2 = ops.sliding_window_attention(*dense, cu, cu, (50, 0), 2)
    assert torch.equal(out, out2)
    assert torch.equal(grad, torch.cat(torch.autograd.grad(out2, dense, do), 1))
    # one key head for all tokens' heads, an output gradient of one number
    one = _rand(n, 1, d, seed=3).requires_grad_()
    k1 = one.expand(n, hkv, d)
    (g1,) = torch.autograd.grad(
        ops.sliding_window_attention(q.detach(), k1, k1, cu, cu, (50, 0)).sum(), [one])
    kd = k1.detach().contiguous()
    ref = _reference(q, kd, kd, cu, cu, (50, 0), 0, do=torch.ones_like(out))
    want = (ref["dk"] + ref["dv"]).sum(1, keepdim=True)
    # two gradients per head, each rounded and within its bound, and sums of four
    bound = (ref["dk_err"] + ref["dv_err"] + U * 4 * (ref["dk"].abs() + ref["dv"].abs())).sum(
        1, keepdim=True) + 2 * U * want.abs()
    assert ((g1.double().cpu() - want).abs() <= bound).all()


def test_odd_strides_and_unaligned_starts_are_copied():
    n, h, d = 90, 2, 64
    cu = _cu(n)
    wide = _rand(n, h * d + 3, seed=4)
    q = wide[:, 1:1 + h * d].unflatten(1, (h, d))
    k, v = _rand(h, n, d, seed=5).transpose(0, 1), _rand(n, d, h, seed=6).transpose(1, 2)
    out = ops.sliding_window_attention(q, k, v, cu, cu, (20, 3), 1)
    again = ops.sliding_window_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, cu,
                                         (20, 3), 1)
    assert torch.equal(out, again)


def test_offsets_beyond_32_bits():
    # 40000 tokens 2^18 bytes apart: the last ones lie 10 GB into the tensor
    n, h, d = 40000, 1, 64
    store = torch.empty(n, 1 << 17, dtype=torch.bfloat16, device=DEV)
    q, k, v = (store[:, i * d:(i + 1) * d].unflatten(1, (h, d)) for i in range(3))
    for i, t in enumerate((q, k, v)):
        t.copy_(_rand(n, h, d, seed=i))
    do = _rand(n, h, d, seed=9)
    cu = _cu(100, n - 100)
    dense = [t.contiguous().requires_grad_() for t in (q, k, v)]
    far = [t.requires_grad_() for t in (q, k, v)]
    results = []
    for leaves in (dense, far):
        out = ops.sliding_window_attention(*leaves, cu, cu, (30, 0), 2)
        results.append([out] + list(torch.autograd.grad(out, leaves, do)))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    # a cache of one long sequence, token by token
    cache = store.detach()[None, :, :2 * d]
    lens = torch.tensor([n], device=DEV)
    with torch.no_grad():
        got = ops.sliding_window_decode(q[-1:], cache[..., None, :d], cache[..., None, d:], lens,
                                        30, 2)
        want = ops.sliding_window_decode(q[-1:].contiguous(), cache[..., None, :d].contiguous(),
                                         cache[..., None, d:].contiguous(), lens, 30, 2)
    assert torch.equal(got, want)


# ------------------------------------------------------------------- values --

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_that_grow_by_hundreds(dtype):
    # keys that grow along the sequence: every block outgrows the softmax
    # reference of the first, and others fall hundreds of powers below it
    n, d = 300, 64
    cu = _cu(n)
    unit = torch.finfo(dtype).eps / 2
    q, k, v, do = (_rand(n, 2, d, seed=i, dtype=dtype) for i in range(4))
    rise = torch.linspace(0.1, 30.0, n, device=DEV).view(n, 1, 1)
    for kk in (k * rise, k * rise.flip(0)):
        kk = kk.to(dtype)
        leaves = [t.clone().requires_grad_() for t in (q, kk, v)]
        out = ops.sliding_window_attention(*leaves, cu, cu, (-1, 0))
        ref = _reference(q, kk, v, cu, cu, (-1, 0), 0, do=do, unit=unit)
        _within(out, ref, "out")
        # scores of some 400 in 32 bits (64 products each, and the LSE): P is
        # off by 400 * 64 * 2^-24 = 2^-9.4 more than the bound's 2^-18, twice
        more = 2.0 ** -8.4 / (2 * unit + 2.0 ** -18) + 1
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do)):
            err = (g.double().cpu() - ref[name]).abs()
            assert (err <= more * ref[name + "_err"] + 2.0 ** -24).all(), name


def test_values_that_are_not_finite_stay_with_the_rows_that_see_them():
    n, d, at = 200, 64, 100
    cu = _cu(n)
    q, k, v = (_rand(n, 2, d, seed=i) for i in range(3))
    clean = ops.sliding_window_attention(q, k, v, cu, cu, (30, 0), 0)
    for bad, where in ((math.nan, "v"), (math.inf, "v"), (math.nan, "k"), (math.inf, "k")):
        k2, v2 = k.clone(), v.clone()
        (v2 if where == "v" else k2)[at] = bad
        out = ops.sliding_window_attention(q, k2, v2, cu, cu, (30, 0), 0)
        rows = torch.arange(n, device=DEV)
        seen = (rows >= at) & (rows <= at + 30)
        # a row redone by definition keeps P unrounded: one rounding of P less
        far = (out[~seen].float() - clean[~seen].float()).abs()
        assert torch.isfinite(out[~seen]).all()
        assert (far <= 4 * U * v.float().abs().max()).all()
        if where == "v":
            assert not torch.isfinite(out[seen]).any()


def test_masked_buckets_leave_rows_empty():
    n, h, d = 150, 2, 32
    cu = _cu(n)
    buckets = ops.relative_position_buckets(8, 20, device=DEV)
    for low in (-math.inf, torch.finfo(torch.bfloat16).min):
        table = _rand(8, h, seed=3)
        table[:, 1] = low          # head 1 sees nothing
        table[0, 0] = low          # head 0 does not see its own token
        table = table.requires_grad_()
        leaves = [_rand(n, h, d, seed=i).requires_grad_() for i in range(3)]
        do = _rand(n, h, d, seed=7)
        out, lse = ops.sliding_window_attention(*leaves, cu, cu, (40, 0), 1, table, buckets,
                                                return_lse=True)
        grads = torch.autograd.grad(out, leaves + [table], do)
        ref = _reference(*leaves, cu, cu, (40, 0), 1, table, buckets, do)
        assert (out[:, 1] == 0).all() and (lse[1] == -math.inf).all()
        assert (out[0] == 0).all() and (lse[:, 0] == -math.inf).all()
        _within(out, ref, "out")
        for name, g in zip(("dq", "dk", "dv", "dtable"), grads):
            assert torch.isfinite(g).all(), name
            _within(g, ref, name)


def test_same_inputs_give_same_bits():
    n = 700
    cu = _cu(300, 1, n - 301)
    buckets = ops.relative_position_buckets(16, 64, True, device=DEV)
    do = _rand(n, 8, 64, seed=9)
    runs = []
    for _ in range(3):
        leaves = [_rand(n, h, 64, seed=i).requires_grad_() for i, h in enumerate((8, 2, 2))]
        table = _rand(16, 8, seed=5).requires_grad_()
        out = ops.sliding_window_attention(*leaves, cu, cu, (100, 50), 3, table, buckets)
        runs.append([out] + list(torch.autograd.grad(out, leaves + [table], do)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


# ----------------------------------------------------- checks, streams, graphs --

def test_bad_metadata_is_refused_and_clamped():
    n = 64
    q, k = _rand(n, 2, 64), _rand(n, 2, 64, seed=1)
    good = _cu(30, 34)
    att = ops.sliding_window_attention
    for bad in ([0, 40, 30], [5, 30, 64], [0, 30, 65], [0, -1, 64]):
        cu = torch.tensor(bad, dtype=torch.int32, device=DEV)
        for pair in ((cu, good), (good, cu)):
            with pytest.raises(ValueError, match="valid offsets"):
                att(q, k, k, *pair, (10, 0))
    table = _rand(4, 2)
    for entry in (-1, 4):
        buckets = torch.zeros(5, dtype=torch.int32, device=DEV)
        buckets[3] = entry
        with pytest.raises(ValueError, match="outside the table"):
            att(q, k, k, good, good, (10, 0), 0, table, buckets)
    assert torch.isfinite(att(q, k, k, good, good, (10, 0))).all()  # and the next call is fine


def test_refusals():
    q, k, cu = _rand(8, 4, 64), _rand(8, 2, 64), _cu(8)
    att = ops.sliding_window_attention
    table, buckets = _rand(4, 4), torch.zeros(5, dtype=torch.int32, device=DEV)
    for error, args, kw in (
            (ValueError, (q, k, k, cu, cu, (-2, 0)), {}),
            (ValueError, (q, k, k, cu, cu, (5, 0), 65), {}),
            (ValueError, (q, k, k, cu, cu, (5, 0)), {"softmax_scale": 0.0}),
            (ValueError, (q, k, k, cu, cu, (5, 0)), {"softmax_scale": math.inf}),
            (ValueError, (q[:, :3], k, k, cu, cu, (5, 0)), {}),
            (ValueError, (q, k, k[:7], cu, cu, (5, 0)), {}),
            (ValueError, (q, k[..., :32], k[..., :32], cu, cu, (5, 0)), {}),
            (ValueError, (q, k, k, cu, _cu(4, 4), (5, 0)), {}),
            (ValueError, (q, k, k, cu, cu, (5, 0)), {"bias_table": table}),
            (ValueError, (q, k, k, cu, cu, (5, 0)),
             {"bias_table": table[:, :2], "bias_buckets": buckets}),
            (ValueError, (q, k, k, cu, cu, (5, 0)),
             {"bias_table": table, "bias_buckets": buckets[:4]}),
            (TypeError, (q, k, k, cu, cu, (5, 0)),
             {"bias_table": table.float(), "bias_buckets": buckets}),
            (TypeError, (q.float(), k.float(), k.float(), cu, cu, (5, 0)), {}),
            (TypeError, (q, k.half(), k.half(), cu, cu, (5, 0)), {}),
            (RuntimeError, (q[..., :48].contiguous(), k[..., :48].contiguous(),
                            k[..., :48].contiguous(), cu, cu, (5, 0)), {}),
            (RuntimeError, (q.cpu(), k.cpu(), k.cpu(), cu.cpu(), cu.cpu(), (5, 0)), {}),
            (RuntimeError, (q, k, k, cu.cpu(), cu, (5, 0)), {})):
        with pytest.raises(error):
            att(*args, **kw)
    far = torch.zeros(2 * 513 + 1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="status 2"):
        att(q, k, k, cu, cu, (5, 0), 0, table, far)
    leaf = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(att(leaf, k, k, cu, cu, (5, 0)).sum(), [leaf], create_graph=True)


def test_another_stream():
    n = 500
    cu = _cu(n)
    q, k, v = (_rand(n, 4, 64, seed=i) for i in range(3))
    x, w = _rand(n, 256, seed=4), _rand(256, seed=5)
    state = torch.tensor([3, 4], device=DEV)

    def work():
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = ops.sliding_window_attention(*leaves, cu, cu, (60, 0), 2)
        grads = torch.autograd.grad(out, leaves, out.detach())
        y, h = ops.residual_rms_norm(x, out.detach().view(n, 256), w, 1e-6, 0.2, state)
        return [out.detach(), *grads, y, h]

    torch.cuda.synchronize()
    want = work()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = work()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_backward_and_decode_replay_in_graphs():
    # lengths, offsets, inputs and the generator's state change between replays
    n, hq, hkv, d = 400, 4, 2, 64
    q, k, v, do = (_rand(n, h, d, seed=i) for i, h in enumerate((hq, hkv, hkv, hq)))
    cu = _cu(150, 250)
    buckets = ops.relative_position_buckets(8, 40, device=DEV)
    table = _rand(8, hq, seed=8)
    x, w = _rand(n, 256, seed=4), _rand(256, seed=5)
    state = torch.tensor([3, 4], device=DEV)
    cache = _rand(2, 3, 300, hkv, d, seed=6)
    lens = torch.tensor([300, 1, 120], dtype=torch.int32, device=DEV)

    def work():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
        out = ops.sliding_window_attention(*leaves[:3], cu, cu, (70, 0), 3, leaves[3], buckets)
        grads = torch.autograd.grad(out, leaves, do)
        rows = [t.detach().requires_grad_() for t in (x, out.detach().view(n, 256), w)]
        y, h = ops.residual_rms_norm(*rows, 1e-6, 0.3, state)
        more = torch.autograd.grad([y, h], rows, [x, x])
        step = ops.sliding_window_decode(q[:3], cache[0], cache[1], lens, 100, 2, table, buckets)
        q8, scales, _ = ops.residual_rms_norm_fp8(x, None, w, 1e-6, 64)
        return [out.detach(), *grads, y.detach(), h.detach(), *more, step, q8.float(), scales]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for rep in range(4):
        q.copy_(_rand(n, hq, d, seed=20 + rep))
        cu.copy_(_cu(100 + 37 * rep, 300 - 37 * rep))
        lens.copy_(torch.tensor([300 - rep, rep, 120 + 50 * rep], device=DEV))
        state += 1
        want = [t.clone() for t in work()]
        torch.cuda.synchronize()
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(captured, want)):
            assert torch.equal(a, b), (rep, i)


def test_registered_operators_and_compilation():
    n, hq, hkv, d = 300, 4, 2, 64
    cu = _cu(100, 200)
    leaves = [_rand(n, h, d, seed=i).requires_grad_() for i, h in enumerate((hq, hkv, hkv))]
    table = _rand(8, hq, seed=8).requires_grad_()
    buckets = ops.relative_position_buckets(8, 40, device=DEV)
    x, w = _rand(n, hq * d, seed=4).requires_grad_(), _rand(hq * d, seed=5).requires_grad_()
    state = torch.tensor([3, 4], device=DEV)
    torch.library.opcheck(torch.ops.lsrm_hip.window_attn_fwd.default,
                          (*leaves, cu, cu, 50, 0, 2, table, buckets, 0.125, True))
    torch.library.opcheck(torch.ops.lsrm_hip.window_attn_fwd.default,
                          (*leaves, cu, cu, 50, 7, 0, None, None, 0.125))
    torch.library.opcheck(torch.ops.lsrm_hip.residual_norm_fwd.default,
                          (x, x.detach(), w, 1e-6, 9000, state))
    torch.library.opcheck(torch.ops.lsrm_hip.residual_norm_fwd.default,
                          (x, None, w, 1e-6, 0, None))
    torch.library.opcheck(torch.ops.lsrm_hip.residual_norm_fp8.default,
                          (x.detach(), None, w.detach(), 1e-6, 64))
    cache = _rand(2, 3, 90, hkv, d, seed=6)
    lens = torch.tensor([90, 0, 7], dtype=torch.int32, device=DEV)
    torch.library.opcheck(torch.ops.lsrm_hip.window_decode.default,
                          (leaves[0].detach()[:3], cache[0], cache[1], lens, 40, 2, None, None,
                           0.125))

    def block(q, k, v, table, x, w):
        o = ops.sliding_window_attention(q, k, v, cu, cu, (50, 0), 2, table, buckets)
        y, h = ops.residual_rms_norm(o.reshape(n, hq * d), x, w, 1e-6, 0.25, state)
        step = ops.sliding_window_decode(q[:3].detach(), cache[0], cache[1], lens, 40, 2)
        return y * 2 + h, step

    results = []
    for fn in (block, torch.compile(block, backend="aot_eager", fullgraph=True)):
        ins = [t.detach().clone().requires_grad_() for t in (*leaves, table, x, w)]
        out, step = fn(*ins)
        out.backward(torch.ones_like(out))
        results.append([out.detach(), step.detach()] + [t.grad for t in ins])
    for a, b in zip(*results):
        assert torch.equal(a, b)


# ------------------------------------------------------------- used together --

def test_window_branch_of_a_training_step():
    # window attention with a learned bias -> gated merge with another branch
    # -> dropout, residual and norm, forward and backward, against the same
    # block in 64 bits
    n, hq, hkv, d = 260, 4, 2, 32
    hid = hq * d
    cu = _cu(100, 1, 159)
    buckets = ops.relative_position_buckets(8, 40, True, device=DEV)
    names = ["q", "k", "v", "table", "gate", "other", "residual", "weight"]
    shapes = [(n, hq, d), (n, hkv, d), (n, hkv, d), (8, hq), (n, 2 * hid), (n, hid), (n, hid),
              (hid,)]
    data = {a: _rand(*s, seed=i) for i, (a, s) in enumerate(zip(names, shapes))}
    data["gate"] = torch.sigmoid(data["gate"].float()).bfloat16()
    dy, dh = _rand(n, hid, seed=21), _rand(n, hid, seed=22)
    state = torch.tensor([11, 12], device=DEV)
    ins = {a: t.clone().requires_grad_() for a, t in data.items()}
    win = ops.sliding_window_attention(ins["q"], ins["k"], ins["v"], cu, cu, (30, 10), 2,
                                       ins["table"], buckets)
    merged = ops.gate_merge(ins["gate"], ins["other"], win.reshape(n, hid))
    y, h = ops.residual_rms_norm(merged, ins["residual"], ins["weight"], 1e-5, 0.25, state)
    got = torch.autograd.grad([y, h], list(ins.values()), [dy, dh])

    ref = {a: t.double().cpu().requires_grad_() for a, t in data.items()}
    mask = dropout_mask(n, hid, 16384, 11, 12).double() / 0.75
    seen = torch.zeros(n, n, dtype=torch.bool)
    rel = torch.arange(n)[None, :] - torch.arange(n)[:, None]
    first = torch.zeros(n, dtype=torch.bool)
    for a, b in ((0, 100), (100, 101), (101, 260)):
        seen[a:b, a:b] = True
        first[a:min(b, a + 2)] = True
    seen &= (rel <= 10) & ((rel >= -30) | first[None, :])
    kk, vv = (ref[a].repeat_interleave(2, 1) for a in "kv")
    bias = ref["table"][buckets.cpu().long()[rel.clamp(-40, 40) + 40]].permute(2, 0, 1)
    s = torch.matmul(ref["q"].transpose(0, 1), kk.permute(1, 2, 0)) / math.sqrt(d) + bias
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    w64 = torch.matmul(p, vv.transpose(0, 1)).transpose(0, 1).reshape(n, hid)
    m64 = ref["gate"][:, :hid] * ref["other"] + ref["gate"][:, hid:] * w64
    h64 = ref["residual"] + m64 * mask
    y64 = h64 * torch.rsqrt(h64.pow(2).mean(-1, keepdim=True) + 1e-5) * ref["weight"]
    want = torch.autograd.grad([y64, h64], list(ref.values()), [dy.double().cpu(),
                                                                dh.double().cpu()])
    # Each value passes at most eight roundings to bf16 on its way (P, the
    # branch, two products and their sum, h, y; the gradients as many), each at
    # most 2^-8 of an intermediate of the result's size, independent of each
    # other: in the 2-norm within 8 * 2^-8 = 2^-5.
    for name, a, b in [("y", y, y64), ("h", h, h64)] + list(zip(names, got, want)):
        rel_err = float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm())
        assert rel_err <= 2.0 ** -5, (name, rel_err)


def test_tokens_one_by_one_follow_the_packed_prompt():
    # a prompt through the packed operator, then steps through the cache: the
    # steps are the rows that the packed operator gives for the longer prompt
    b, prompt, steps, hq, hkv, d = 3, (40, 1, 97), 6, 8, 2, 64
    cap = 128
    buckets = ops.relative_position_buckets(16, 48, device=DEV)
    table = _rand(16, hq, seed=9)
    k, v = (_rand(b, cap, hkv, d, seed=i) for i in (1, 2))
    q = _rand(b, cap, hq, d, seed=3)
    rows = {}
    for extra in range(steps + 1):
        total = [p + extra for p in prompt]
        pick = lambda t: torch.cat([t[i, :m] for i, m in enumerate(total)])  # noqa: E731
        cu = _cu(*total)
        out = ops.sliding_window_attention(pick(q), pick(k), pick(v), cu, cu, (33, 0), 4, table,
                                           buckets)
        rows[extra] = out[cu[1:].long() - 1]
        ref = _reference(pick(q), pick(k), pick(v), cu, cu, (33, 0), 4, table, buckets)
        lens = torch.tensor(total, dtype=torch.int32, device=DEV)
        step = ops.sliding_window_decode(q[torch.arange(b), lens.long() - 1], k, v, lens, 33, 4,
                                         table, buckets)
        at = (cu[1:].long() - 1).cpu()
        for got in (step, rows[extra]):
            err = (got.double().cpu() - ref["out"][at]).abs()
            assert (err <= ref["out_err"][at] + 2.0 ** -24).all()
        # and the projection's input in 8 bits, from the same rows
        q8, scale, h = ops.residual_rms_norm_fp8(step.view(b, hq * d), None,
                                                 torch.ones(hq * d, device=DEV).bfloat16(), 1e-6,
                                                 128)
        assert torch.equal(h, step.view(b, hq * d))
        f = h.float()
        y = f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + 1e-6)
        back = q8.float() * scale.repeat_interleave(128, 1)
        # half a step of e4m3 of the value, or of the group's smallest normal
        assert ((back - y).abs() <= 2.0 ** -4 * torch.maximum(
            y.abs(), scale.repeat_interleave(128, 1) * 2.0 ** -6) * 1.001 + 1e-6).all()


def _block(x, residual, weight, table, cu, buckets, rng):
    """Attention of the normed rows with themselves, its output back into them."""
    y, h = ops.residual_rms_norm(x, residual, weight, 1e-6, 0.1, rng)
    a = y.view(-1, 4, 64)
    out = ops.sliding_window_attention(a, a[:, :2], a[:, 2:], cu, cu, (40, 0), 2, table, buckets)
    return out.reshape(x.shape) + h


def test_recomputed_and_offloaded_activations():
    from torch.utils.checkpoint import checkpoint
    leaves = [_rand(*s, seed=i).requires_grad_()
              for i, s in enumerate(((150, 256), (150, 256), (256,), (8, 4)))]
    rest = (_cu(100, 50), ops.relative_position_buckets(8, 20, device=DEV),
            torch.tensor([3, 4], device=DEV))
    do = _rand(150, 256, seed=9)
    want = torch.autograd.grad(_block(*leaves, *rest), leaves, do)
    kept = checkpoint(_block, *leaves, *rest, use_reentrant=False)
    for g, w in zip(torch.autograd.grad(kept, leaves, do), want):
        assert torch.equal(g, w)
    with torch.autograd.graph.save_on_cpu():
        kept = _block(*leaves, *rest)
    for g, w in zip(torch.autograd.grad(kept, leaves, do), want):
        assert torch.equal(g, w)


def test_two_threads_at_once():
    import threading
    rest = (_cu(100, 50), ops.relative_position_buckets(8, 20, device=DEV))
    do = _rand(150, 256, seed=9)
    cases = [[_rand(*s, seed=10 * n + i).requires_grad_()
              for i, s in enumerate(((150, 256), (150, 256), (256,), (8, 4)))] +
             [torch.tensor([n, 4], device=DEV)] for n in range(2)]

    def once(case):
        *leaves, rng = case
        return torch.autograd.grad(_block(*leaves, *rest, rng), leaves, do)

    want = [once(c) for c in cases]
    torch.cuda.synchronize()
    got = [None, None]

    def work(n):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[n] = [once(cases[n]) for _ in range(20)]
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for n in range(2):
        for run in got[n]:
            assert all(torch.equal(g, w) for g, w in zip(run, want[n]))


def test_derivatives_that_are_not_there_are_refused():
    cu = _cu(10)
    q, w, x = _rand(10, 2, 64), _rand(64, seed=1), _rand(10, 64, seed=2)
    attend = lambda t: ops.sliding_window_attention(t, q, q, cu, cu, (5, 0))  # noqa: E731
    norm = lambda t: ops.residual_rms_norm(t, None, w)[0]  # noqa: E731
    for f, t in ((attend, q), (norm, x)):
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(dual)
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda u: f(u).float().sum())(t)
        with pytest.raises(RuntimeError):
            torch.vmap(f)(torch.stack([t, t]))
        leaf = t.detach().requires_grad_()
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(f(leaf).float().sum(), leaf, create_graph=True)


def test_binding_is_loaded_from_the_tree():
    assert H.native().__file__ == str(H.LIB_PATH.with_name("_native.so"))
