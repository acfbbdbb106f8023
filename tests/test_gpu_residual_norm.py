"""The residual norm (sparse.ops.residual_rms_norm and its 8-bit form, HIP
lsrm_residual_norm_*) against its definition in 64 bits, each element within
the bound of its roundings; the dropout mask bit for bit."""

import pytest
import torch

import sparse.ops as ops
from oracle.norm import dropout_mask, residual_norm_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
UNIT = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def _inputs(n, hidden, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, res, dy, dh = (torch.randn(n, hidden, generator=g).to(DT[dtype]) for _ in range(4))
    w = (1 + 0.3 * torch.randn(hidden, generator=g)).to(DT[dtype])
    return x, res, w, dy, dh


def _near(got, want, err, what):
    # values below the type's smallest normal (2^-14 in fp16) are a whole number
    # of its smallest subnormals (2^-24): a rounding there is off by at most half
    # a step, whatever the value
    info = torch.finfo(got.dtype)
    least = info.smallest_normal * info.eps / 2
    got = got.detach().double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    over = (got - want).abs() > err + least * 1.01 + 2.0 ** -40
    assert not over.any(), (what, over.nonzero()[:4].tolist())


def _compare(n, hidden, dtype, p, residual=True, seed=0):
    x, res, w, dy, dh = _inputs(n, hidden, dtype, seed)
    res = res if residual else None
    least = min(65535, round(p * 65536))
    state = torch.tensor([77 - seed, 2 ** 40 + seed], dtype=torch.int64)
    mask = dropout_mask(n, hidden, least, *state.tolist()) if least else None
    leaves = [None if t is None else t.to(DEV).requires_grad_() for t in (x, res, w)]
    y, h = ops.residual_rms_norm(*leaves, 1e-5, p, state.to(DEV))
    used = [t for t in leaves if t is not None]
    grads = torch.autograd.grad([y, h], used, [dy.to(DEV), dh.to(DEV)])
    ref = residual_norm_ref(x, res, w, 1e-5, mask, least, dy, dh, UNIT[dtype], h.detach().cpu())
    _near(h, ref["h"], ref["h_err"], "h")
    _near(y, ref["y"], ref["y_err"], "y")
    for name, got in zip(["dx"] + ["dres"] * residual + ["dw"], grads):
        _near(got, ref[name], ref[name + "_err"], name)
    if mask is not None:  # a gradient that is not 0 in exactly the kept places
        kept = grads[0].cpu() != 0
        assert torch.equal(kept & (ref["dx"].abs() > 1e-4), mask & (ref["dx"].abs() > 1e-4))
        assert not (kept & ~mask).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,hidden", [(1, 1), (3, 7), (2, 8), (5, 513), (7, 1536), (1, 4096),
                                      (2, 8200), (3, 16384), (1030, 24), (1025, 1001),
                                      (1030, 2049)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_sizes_and_types(n, hidden, dtype, p):
    if n * hidden > 300000 and p > 0:
        hidden = hidden // 4 + 1  # the oracle's mask is slow
    _compare(n, hidden, dtype, p)


@pytest.mark.parametrize("n,hidden", [(1900, 1800), (1500, 1500), (8200, 24), (2100, 1000)])
def test_many_rows(n, hidden):
    _compare(n, hidden, "bf16", 0.0)


@pytest.mark.parametrize("p", [0.0, 0.5, 0.99, 0.999999])
def test_without_residual_and_probabilities(p):
    _compare(40, 136, "bf16", p, residual=False)
    _compare(40, 136, "fp32", p, seed=3)


def test_one_output_used():
    x, res, w, dy, dh = _inputs(9, 64, "fp32")
    for use in ("y", "h"):
        leaves = [t.to(DEV).requires_grad_() for t in (x, res, w)]
        y, h = ops.residual_rms_norm(*leaves, 1e-5)
        out, d = (y, dy) if use == "y" else (h, dh)
        grads = torch.autograd.grad(out, leaves, d.to(DEV))
        ref = residual_norm_ref(x, res, w, 1e-5, dy=dy if use == "y" else None,
                                dh=dh if use == "h" else None, unit=UNIT["fp32"])
        for name, got in zip(("dx", "dres", "dw"), grads):
            _near(got, ref[name], ref[name + "_err"], (use, name))


def test_no_rows_and_more_dimensions():
    w = torch.ones(32, device=DEV, requires_grad=True)
    x = torch.empty(0, 32, device=DEV, requires_grad=True)
    y, h = ops.residual_rms_norm(x, x.detach(), w)
    (dw,) = torch.autograd.grad(y.sum() + h.sum(), [w])
    assert y.shape == (0, 32) and (dw == 0).all()
    z = torch.randn(2, 3, 32, device=DEV)
    y3, h3 = ops.residual_rms_norm(z, z, w.detach())
    y2, h2 = ops.residual_rms_norm(z.view(6, 32), z.view(6, 32), w.detach())
    assert torch.equal(y3.view(6, 32), y2) and torch.equal(h3.view(6, 32), h2)
    q, s, _ = ops.residual_rms_norm_fp8(z, None, w.detach())
    assert q.shape == (2, 3, 32) and s.shape == (2, 3, 1)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,hidden,group", [(1, 1, 0), (3, 100, 0), (5, 1536, 128), (4, 96, 32),
                                            (2, 16384, 64), (1100, 256, 128), (1100, 333, 0),
                                            (2, 5003, 0)])
def test_rows_in_8_bits(n, hidden, group, dtype):
    x, res, w, _, _ = _inputs(n, hidden, dtype, 5)
    x[0] = 0
    res[0] = 0  # a row of zeros: scale 1
    q, s, h = ops.residual_rms_norm_fp8(x.to(DEV), res.to(DEV), w.to(DEV), 1e-5, group)
    ref = residual_norm_ref(x, res, w, 1e-5, unit=UNIT[dtype], h=h.cpu())
    _near(h, ref["h"], ref["h_err"], "h")
    y = ref["y"].view(n, -1, group or hidden)
    top = y.abs().amax(-1)
    want = torch.where(top > 0, top / 448.0, 1.0)
    _near(s, want, 2.0 ** -18 * want, "scales")
    # half a step of e4m3: 2^-4 of the value, or of its smallest normal 2^-6
    exact = y / want[..., None]
    got = q.float().double().cpu().view_as(exact)
    bound = 2.0 ** -4 * exact.abs().clamp_min(2.0 ** -6) * (1 + 2.0 ** -12) + 2.0 ** -12
    assert ((got - exact).abs() <= bound).all()
    assert float(got.abs().max()) <= 448.0


def test_state_is_read_at_the_forward():
    # the state moves on before the backward, which draws the forward's mask
    x, res, w, dy, _ = _inputs(30, 200, "fp32", 8)
    state = torch.tensor([5, 6], dtype=torch.int64, device=DEV)
    leaves = [t.to(DEV).requires_grad_() for t in (x, res, w)]
    y, _ = ops.residual_rms_norm(*leaves, 1e-5, 0.4, state)
    state += 11
    dx = torch.autograd.grad(y, leaves, dy.to(DEV))[0]
    assert not ((dx.cpu() != 0) & ~dropout_mask(30, 200, round(0.4 * 65536), 5, 6)).any()
    again, _ = ops.residual_rms_norm(*[t.detach() for t in leaves], 1e-5, 0.4,
                                     torch.tensor([5, 6], device=DEV))
    assert torch.equal(again, y)


def test_refusals():
    x = torch.zeros(4, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    with pytest.raises(ValueError, match="rng_state"):
        ops.residual_rms_norm(x, x, w, dropout_p=0.5)
    with pytest.raises(ValueError, match="rng_state"):
        ops.residual_rms_norm(x, x, w, dropout_p=0.5, rng_state=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError, match="probability"):
        ops.residual_rms_norm(x, x, w, dropout_p=1.0, rng_state=torch.zeros(2, device=DEV).long())
    with pytest.raises(ValueError, match="group_size"):
        ops.residual_rms_norm_fp8(x, x, w, group_size=48)
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.residual_rms_norm_fp8(x.clone().requires_grad_(), x, w)
    with pytest.raises(TypeError):
        ops.residual_rms_norm(x, x.half(), w)
    with pytest.raises(ValueError):
        ops.residual_rms_norm(x, x[:3], w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.residual_rms_norm(x.cpu(), x.cpu(), w.cpu())
