"""Digits of the norm and of the rotation one by one, where the bound of the whole pass would hide a step's own.

Tolerance of the norm: a channel of 12 bits alone in its row has an exact square and mean; the reciprocal root is off by half a
unit of its last place and next to nothing more (2^-24 of it), its product with the channel is rounded once (2^-24): 2 units of
2^-24. Rows whose squares are subnormal: a square is off by 2^-150, and so is the mean after the sum, which is exact there; the
root halves what the mean is off by. The weight is 1.

Of the rotation: a pair of 16 and 0 in a row whose mean square is 1 becomes 16 times cosine and sine. Position times frequency is
exact in 64 bits below 2^53, turns are then off by fewer than 3 * 2^-53 of themselves. Cosine and sine are two units of their
last place off (2^-22 of them at most), the term for what float32 rounds off the turns is added with one rounding (2^-24), and
what it neglects is the square of 2^-26 turns.
"""

import numpy as np
import pytest
import torch

from moespresso_amd.runtime.qwen import paged

pytestmark = pytest.mark.gpu

F32 = torch.float32


def _call(q, pos=None, eps=0.0, inv=None):
    T = q.shape[0]
    ones = torch.ones(256, device="cuda")
    pos = torch.zeros(T, dtype=torch.int32, device="cuda") if pos is None else pos
    inv = torch.ones(32, device="cuda") if inv is None else inv
    return paged.qk_norm_rope(q, q.clone(), ones, ones, pos, inv, eps=eps)


def test_the_root_of_the_mean_square_keeps_its_digits():
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.zeros(65536, 1, 256, device="cuda")
    q[:, 0, 100] = torch.randint(2048, 4096, (65536,), device="cuda", generator=gen).float()
    q *= torch.exp2(torch.randint(-20, 20, (65536, 1, 1), device="cuda", generator=gen).float())
    for got in _call(q):
        assert ((got[:, 0, 100].double() - 16).abs() <= 16 * 2.01 * 2.0 ** -24).all()


@pytest.mark.parametrize("eps", [0.0, 1e-42, 1e-38])
@pytest.mark.parametrize("size", [1e-20, 3e-20, 1e-19, 1e-17])
def test_rows_whose_mean_square_is_hardly_a_number(size, eps):
    """Below 2^-126 a mean is subnormal, not zero."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = (1 + torch.rand(64, 3, 256, device="cuda", generator=gen)) * size
    eps = float(np.float32(eps))
    mean = q.double().square().mean(-1, keepdim=True) + eps
    want = q.double() / mean.sqrt()
    bound = want * (32 * 2.0 ** -24 + 2.0 ** -150 / mean)
    for got in _call(q, eps=eps):
        assert ((got.double() - want).abs() <= bound).all()


def test_rows_of_zeros_and_of_what_cannot_be_squared():
    q = torch.zeros(4, 1, 256, device="cuda")
    q[1], q[2, 0, 7], q[3, 0, 7] = 1e30, float("nan"), float("inf")
    got = _call(q, eps=1e-6)[0]
    assert (got[:2] == 0).all()  # (nothing over the root of eps; a mean beyond float32 is infinite, and its root's reciprocal zero)
    assert got[2].isnan().all()
    pair = torch.zeros(256, dtype=torch.bool, device="cuda")
    pair[[7, 39]] = True  # (infinity times that zero, and the channel that it rotates with)
    assert got[3, 0].isnan().equal(pair) and (got[3, 0][~pair] == 0).all()


def test_cosines_and_sines_keep_their_digits_near_their_zeros():
    gen = torch.Generator(device="cuda").manual_seed(3)
    T = 20000
    q = torch.zeros(T, 1, 256, device="cuda")
    q[torch.arange(T), 0, torch.randint(0, 32, (T,), device="cuda", generator=gen)] = 16
    channel = q[:, 0].argmax(-1)
    pos = torch.randint(-120000, 120000, (T,), device="cuda", generator=gen, dtype=torch.int32)
    inv = (1e7 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float().cuda()
    got = _call(q, pos, 0.0, inv)[0][:, 0].double()
    angle = pos.double() * inv[channel].double()
    slack = angle.abs() * 4 * 2.0 ** -53 + 2 * torch.pi ** 2 * 2.0 ** -52
    for want, at in ((angle.cos(), channel), (angle.sin(), channel + 32)):
        err = (got[torch.arange(T), at] / 16 - want).abs()
        assert (err <= (2.0 ** -22 + 2.0 ** -24) * want.abs() + slack).all()
