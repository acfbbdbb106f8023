"""Dropout, residual addition and root-mean-square norm by definition in 64
bits, with the gradients, the counter-based mask (Philox4x32-10, written with
Python's whole numbers) and error bounds."""

from __future__ import annotations

import numpy as np
import torch


def philox4x32(counter, key, rounds: int = 10):
    """One block of Salmon et al. (2011), four 32-bit words."""
    c, (k0, k1) = list(counter), key
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k0, b & 0xffffffff, (a >> 32) ^ c[3] ^ k1, a & 0xffffffff]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return c


def dropout_mask(n: int, hidden: int, least: int, seed: int, offset: int) -> torch.Tensor:
    """[n, hidden] truth values: element stays."""
    seed, offset = seed & (2 ** 64 - 1), offset & (2 ** 64 - 1)
    key = (seed & 0xffffffff, seed >> 32)
    out = np.zeros((n, (hidden + 7) // 8 * 8), dtype=bool)
    for row in range(n):
        for g in range((hidden + 7) // 8):
            words = philox4x32((g, row, offset & 0xffffffff, offset >> 32), key)
            for e in range(8):
                out[row, g * 8 + e] = ((words[e // 2] >> (16 * (e % 2))) & 0xffff) >= least
    return torch.from_numpy(out[:, :hidden])


def residual_norm_ref(x, residual, weight, eps, mask=None, least=0, dy=None, dh=None, unit=0.0,
                      h=None):
    """Rows of any float type -> dict in 64 bits of h, y (of h rounded to x's
    type, or of the `h` given), rstd and, with dy or dh, dx, dres, dw; for unit
    > 0 (one rounding to the kernel's type, relative) bounds "<name>_err"."""
    dtype, w = x.dtype, weight.double()
    factor = 65536.0 / (65536 - least)
    d = x.double() if mask is None else x.double() * mask * factor
    s = d if residual is None else d + residual.double()
    tiny = 2.0 ** -18
    r = {"h": s, "h_err": unit * s.abs() + 2.0 ** -22 * d.abs()}
    stored = (s.to(dtype) if h is None else h).double()
    hidden = x.shape[-1]
    rstd = (stored.pow(2).mean(-1, keepdim=True) + eps) ** -0.5
    n = stored * rstd
    r["y"] = n * w
    r["rstd"] = rstd[..., 0]
    r["y_err"] = (unit + tiny) * r["y"].abs()
    if dy is None and dh is None:
        return r
    dy = torch.zeros_like(stored) if dy is None else dy.double()
    dh = torch.zeros_like(stored) if dh is None else dh.double()
    g = dy * w
    mean = (g * n).mean(-1, keepdim=True)
    r["dres"] = dh + rstd * (g - n * mean)
    spread = dh.abs() + rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    r["dres_err"] = unit * r["dres"].abs() + tiny * spread
    keep = 1.0 if mask is None else mask.double() * factor
    r["dx"] = r["dres"] * keep
    r["dx_err"] = unit * r["dx"].abs() + tiny * spread * keep
    rows = (-1, hidden)
    r["dw"] = (dy * n).reshape(rows).sum(0)
    r["dw_err"] = unit * r["dw"].abs() + tiny * (dy * n).abs().reshape(rows).sum(0)
    return r
