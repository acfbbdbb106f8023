"""CPU checks of the window and norm operators: sizes and refusals of their C
entry points (before any device work), fake implementations, and host tensors
refused by every path."""

import pytest
import torch

import lsrm_hip as H
import sparse.ops as ops

META = "meta"
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3


@pytest.fixture()
def lib():
    if not H.LIB_PATH.exists():
        pytest.skip("liblsrm_hip.so not built")
    return H.lib()


def _fwd(lib, q=16, k=16, v=16, dtype=2, qs=256, ks=128, vs=128, nq=10, nk=10, hq=4, hkv=2, d=64,
         cu_q=16, cu_k=16, batch=1, left=5, right=0, sinks=0, table=None, nb=0, buckets=None, r=-1,
         scale=0.1, out=16, low=None, lse=16):
    return lib.lsrm_window_attn_fwd(q, k, v, dtype, qs, ks, vs, nq, nk, hq, hkv, d, cu_q, cu_k,
                                    batch, left, right, sinks, table, nb, buckets, r, scale, out,
                                    low, lse, None)


def test_attention_refusals(lib):
    # addresses are made up: every call below is refused before any is used
    for want, kw in ((UNSUPPORTED, {"dtype": 0}), (UNSUPPORTED, {"d": 48}),
                     (INVALID, {"hq": 3}), (INVALID, {"nq": -1}), (INVALID, {"left": -2}),
                     (INVALID, {"right": -2}), (INVALID, {"sinks": -1}),
                     (UNSUPPORTED, {"sinks": 65}), (INVALID, {"scale": 0.0}),
                     (INVALID, {"scale": float("nan")}), (INVALID, {"scale": float("inf")}),
                     (INVALID, {"q": None}), (INVALID, {"k": None}), (INVALID, {"cu_q": None}),
                     (INVALID, {"out": None}), (INVALID, {"qs": 128}),
                     (UNSUPPORTED, {"qs": 260}), (UNSUPPORTED, {"ks": (1 << 22) + 8}),
                     (UNSUPPORTED, {"q": 24}), (UNSUPPORTED, {"out": 8}),
                     (UNSUPPORTED, {"low": 8}),
                     (UNSUPPORTED, {"nk": (1 << 29) + 1}),
                     (INVALID, {"table": 16}), (INVALID, {"buckets": 16}),
                     (INVALID, {"table": 16, "buckets": 16, "nb": 0, "r": 4}),
                     (INVALID, {"table": 16, "buckets": 16, "nb": 4, "r": -1}),
                     (UNSUPPORTED, {"table": 16, "buckets": 16, "nb": 4, "r": 513})):
        assert _fwd(lib, **kw) == want, kw
    assert _fwd(lib, nq=0, nk=0, q=None, k=None, v=None, cu_q=None, cu_k=None, out=None,
                lse=None) == 0


def test_backward_workspace(lib):
    size = lib.lsrm_window_attn_bwd_workspace_size
    plain = size(1000, 1000, 4, 4, 64, 1, 100, 0, -1)
    assert plain >= 2 * 4 * 1000 * 4
    assert size(1000, 1000, 4, 4, 64, 1, 100, 4, -1) > plain
    assert size(1000, 1000, 4, 4, 64, 1, 1000, 4, -1) == plain  # no query leaves them behind
    assert size(1000, 1000, 4, 4, 64, 1, 100, 0, 128) > plain
    assert size(10, 10, 3, 2, 64, 1, 5, 0, -1) == 0
    args = [16, 16, 16, 16, 16, None, 16, 2, 256, 128, 128, 10, 10, 4, 2, 64, 16, 16, 1, 5, 0, 0, None,
            0, None, -1, 0.1, 16, 16, 16, None, 256, 100, None]
    assert lib.lsrm_window_attn_bwd(*args) == WORKSPACE
    args[31] = None
    assert lib.lsrm_window_attn_bwd(*args) == WORKSPACE
    args[31], args[30] = 256, 16  # a table's gradient without a table
    assert lib.lsrm_window_attn_bwd(*args) == INVALID


def test_decode_sizes_and_refusals(lib):
    size = lib.lsrm_window_decode_workspace_size
    assert size(1, 131072, 32, 2, 64, 4095, 4) > 0       # split between workgroups
    assert size(4096, 4096, 32, 8, 128, 4095, 4) == 0    # enough sequences
    assert size(1, 64, 32, 2, 64, 63, 0) == 0            # too few keys to split
    base = dict(q=16, k=16, v=16, dt=2, qs=256, kb=6400, kt=128, kh=64, vb=6400, vt=128, vh=64,
                lens=16, b=2, cap=50, hq=4, hkv=2, d=64, left=9, sinks=0, table=None, nb=0,
                buckets=None, r=-1, scale=0.1, out=16, lse=16, ws=None, wsn=0, st=None)
    for want, kw in ((UNSUPPORTED, {"dt": 0}), (UNSUPPORTED, {"d": 96}), (INVALID, {"hq": 5}),
                     (INVALID, {"left": -2}), (UNSUPPORTED, {"sinks": 100}),
                     (UNSUPPORTED, {"kt": 129}), (INVALID, {"vb": -8}),
                     (UNSUPPORTED, {"vt": (1 << 22) + 8}), (UNSUPPORTED, {"k": 8}),
                     (INVALID, {"lens": None}), (INVALID, {"scale": -1.0}),
                     (WORKSPACE, {"b": 1, "cap": 131072, "left": 4095})):
        assert lib.lsrm_window_decode(*{**base, **kw}.values()) == want, kw
    assert lib.lsrm_window_decode(*{**base, "b": 0, "q": None}.values()) == 0


def test_norm_sizes_and_refusals(lib):
    fwd = dict(x=16, r=None, w=16, dt=2, n=4, c=64, eps=1e-6, least=0, rng=None, used=None, y=16,
               h=16, rstd=16, st=None)
    for want, kw in ((UNSUPPORTED, {"dt": 7}), (UNSUPPORTED, {"c": 16385}), (INVALID, {"c": 0}),
                     (INVALID, {"n": -1}), (INVALID, {"least": 65536}), (INVALID, {"least": 5}),
                     (INVALID, {"eps": -1.0}), (INVALID, {"eps": float("nan")}),
                     (INVALID, {"x": None}), (INVALID, {"x": 17}), (INVALID, {"rstd": None})):
        assert lib.lsrm_residual_norm_fwd(*{**fwd, **kw}.values()) == want, kw
    assert lib.lsrm_residual_norm_fwd(*{**fwd, "n": 0}.values()) == 0
    fp8 = dict(x=16, r=None, w=16, dt=2, n=4, c=96, eps=1e-6, group=32, y8=16, s=16, h=16, st=None)
    for want, kw in ((INVALID, {"group": 64}), (UNSUPPORTED, {"group": 48}),
                     (INVALID, {"group": -32}), (INVALID, {"y8": None}), (INVALID, {"s": None})):
        assert lib.lsrm_residual_norm_fp8(*{**fp8, **kw}.values()) == want, kw
    assert lib.lsrm_residual_norm_bwd_workspace_size(100000, 1024) >= 1024 * 4
    assert lib.lsrm_residual_norm_bwd_workspace_size(10, 20000) == 0
    bwd = dict(dy=16, dh=16, h=16, w=16, rstd=16, dt=2, n=4, c=64, least=0, rng=None, dx=None,
               dr=16, dw=16, ws=256, wsn=10, st=None)
    for want, kw in ((WORKSPACE, {}), (INVALID, {"dx": 16}), (INVALID, {"least": 9}),
                     (INVALID, {"dw": None}), (WORKSPACE, {"ws": None, "wsn": 1 << 20})):
        assert lib.lsrm_residual_norm_bwd(*{**bwd, **kw}.values()) == want, kw


def test_fake_shapes():
    q = torch.empty(30, 4, 64, dtype=torch.bfloat16, device=META, requires_grad=True)
    k = torch.empty(50, 2, 64, dtype=torch.bfloat16, device=META, requires_grad=True)
    cu = torch.empty(3, dtype=torch.int32, device=META)
    t = torch.empty(8, 4, dtype=torch.bfloat16, device=META, requires_grad=True)
    b = torch.empty(41, dtype=torch.int32, device=META)
    o, lse, low = torch.ops.lsrm_hip.window_attn_fwd(q, k, k, cu, cu, 5, 0, 1, t, b, 0.1, True)
    assert low.shape == q.shape and low.dtype == torch.int8
    o, lse, low = torch.ops.lsrm_hip.window_attn_fwd(q, k, k, cu, cu, 5, 0, 1, t, b, 0.1)
    assert low.numel() == 0
    assert o.shape == q.shape and lse.shape == (4, 30) and lse.dtype == torch.float32
    grads = torch.autograd.grad(o.sum(), [q, k, t])
    assert [g.shape for g in grads] == [q.shape, k.shape, t.shape]
    cache = torch.empty(3, 9, 2, 64, dtype=torch.bfloat16, device=META)
    o, lse = torch.ops.lsrm_hip.window_decode(q.detach()[:3], cache, cache, cu, 5, 0, None, None,
                                              0.1)
    assert o.shape == (3, 4, 64) and lse.shape == (4, 3)
    x = torch.empty(5, 96, dtype=torch.float16, device=META, requires_grad=True)
    w = torch.empty(96, dtype=torch.float16, device=META, requires_grad=True)
    rng = torch.empty(2, dtype=torch.int64, device=META)
    for least, state in ((0, None), (100, rng)):
        y, h, rstd, used = torch.ops.lsrm_hip.residual_norm_fwd(x, x.detach(), w, 1e-6, least,
                                                                state)
        assert y.shape == h.shape == x.shape and rstd.shape == (5,)
        gx, gw = torch.autograd.grad(y.sum() + h.sum(), [x, w])
        assert gx.shape == x.shape and gw.shape == w.shape
    q8, s, h = torch.ops.lsrm_hip.residual_norm_fp8(x.detach(), None, w.detach(), 1e-6, 32)
    assert q8.dtype == torch.float8_e4m3fn and s.shape == (5, 3) and h.shape == x.shape


def test_host_tensors_are_refused(lib):
    q = torch.zeros(8, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    x, w = torch.zeros(4, 64), torch.ones(64)
    c = torch.zeros(8, 4, 2, 64, dtype=torch.bfloat16)
    lens = torch.ones(8, dtype=torch.int32)
    for call in (lambda: ops.sliding_window_attention(q, q, q, cu, cu, (5, 0)),
                 lambda: torch.ops.lsrm_hip.window_attn_fwd(q, q, q, cu, cu, 5, 0, 0, None, None,
                                                            0.1),
                 lambda: H.window_attn_bwd(q, q, q, q, q, torch.zeros(0, dtype=torch.int8),
                                           torch.zeros(2, 8), cu, cu, 5, 0, 0, None,
                                           None, 0.1),
                 lambda: ops.sliding_window_decode(q, c, c, lens, 5),
                 lambda: torch.ops.lsrm_hip.window_decode(q, c, c, lens, 5, 0, None, None, 0.1),
                 lambda: H.window_validate(8, 8, cu, cu),
                 lambda: ops.residual_rms_norm(x, x, w),
                 lambda: ops.residual_rms_norm_fp8(x, x, w),
                 lambda: torch.ops.lsrm_hip.residual_norm_fwd(x, x, w, 1e-6, 0, None),
                 lambda: torch.ops.lsrm_hip.residual_norm_fp8(x, x, w, 1e-6, 0)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
