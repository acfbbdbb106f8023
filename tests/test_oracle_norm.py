"""Pins of oracle.norm: the generator against the published known answers,
gradients against torch autograd and against differences."""

import pytest
import torch

from oracle.norm import dropout_mask, philox4x32, residual_norm_ref


def test_philox_known_answers():
    # Philox4x32-10 of the paper's reference vectors: all zeros, all ones, and
    # the digits of pi
    assert philox4x32((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    ones = 0xffffffff
    assert philox4x32((ones,) * 4, (ones,) * 2) == \
        [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert philox4x32((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344),
                      (0xa4093822, 0x299f31d0)) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def test_mask_rate_and_columns():
    m = dropout_mask(64, 101, 16384, 1234, 5)
    assert m.shape == (64, 101) and abs(float(m.double().mean()) - 0.75) < 0.03
    assert torch.equal(dropout_mask(64, 33, 16384, 1234, 5), m[:, :33])
    assert not torch.equal(dropout_mask(64, 101, 16384, 1234, 6), m)
    assert dropout_mask(3, 9, 0, 1, 1).all()
    assert torch.equal(dropout_mask(4, 20, 9000, -1, -2),
                       dropout_mask(4, 20, 9000, 2 ** 64 - 1, 2 ** 64 - 2))


@pytest.mark.parametrize("least", [0, 20000])
def test_gradients_against_autograd_and_differences(least):
    g = torch.Generator().manual_seed(1)
    x, res, dy, dh = (torch.randn(5, 12, generator=g, dtype=torch.float64) for _ in range(4))
    w = torch.randn(12, generator=g, dtype=torch.float64)
    mask = dropout_mask(5, 12, least, 9, 9) if least else None
    factor = 65536.0 / (65536 - least)
    ref = residual_norm_ref(x, res, w, 1e-3, mask, least, dy, dh)
    leaves = [t.clone().requires_grad_() for t in (x, res, w)]
    h = leaves[1] + (leaves[0] if mask is None else leaves[0] * mask * factor)
    y = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + 1e-3) * leaves[2]
    assert torch.allclose(y, ref["y"]) and torch.allclose(h, ref["h"])
    for name, grad in zip(("dx", "dres", "dw"), torch.autograd.grad([y, h], leaves, [dy, dh])):
        assert torch.allclose(grad, ref[name], rtol=1e-11, atol=1e-12), name

    def loss(x, res, w):
        r = residual_norm_ref(x, res, w, 1e-3, mask, least)
        return float((r["y"] * dy + r["h"] * dh).sum())

    tensors, step = [x, res, w], 1e-6
    for at, name in enumerate(("dx", "dres", "dw")):
        way = torch.randn(tensors[at].shape, generator=g, dtype=torch.float64)
        moved = [[t + s * step * way if i == at else t for i, t in enumerate(tensors)]
                 for s in (1, -1)]
        want = float((ref[name] * way).sum())
        got = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        assert abs(got - want) < 1e-6 * (1 + abs(want)), name
