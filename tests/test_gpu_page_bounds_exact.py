"""Bounds of pages against rational arithmetic: no key lies outside what they say, by however little.

A key of 8-bit rows is code * scale + bias as a rational number, one of 16-bit rows the number itself; the exponent is the smallest with
max |k| <= 127 * 2^e (within +-50), the codes are the floor of the smallest key and the ceiling of the largest in steps of 2^e, within +-127."""

import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from paged_reference import BF16, F16, F32, i32
from moespresso_amd.runtime.qwen import paged

pytestmark = pytest.mark.gpu

PAGE = 16


def _keys(side):
    """Rows [n_pages, Hkv, page, 256] as rational numbers."""
    if torch.is_tensor(side):
        x = side.double().cpu().numpy()
        return np.array([Fraction(v) for v in x.reshape(-1).tolist()], dtype=object).reshape(x.shape)
    codes, scales, biases = side
    c = codes.view(torch.uint8).cpu().numpy()
    s, z = (np.array([Fraction(v) for v in t.double().cpu().reshape(-1).tolist()], dtype=object).reshape(t.shape).repeat(64, -1)
            for t in (scales, biases))
    return c.astype(object) * s + z


def _bounds(rows):
    """(lower codes, upper codes, exponent) of rows [n, 256]."""
    low, high = rows.min(0), rows.max(0)
    top, e = max(-low.min(), high.max()), -50
    while top > 127 * Fraction(2) ** e and e < 50:
        e += 1
    step = Fraction(2) ** e
    low, high = ([min(max(f(x / step), -127), 127) for x in xs] for f, xs in ((math.floor, low), (math.ceil, high)))
    return low, high, e


def _check(side, steps):
    """Rows of every page appended in so many at a time; after every step the bounds are those of all rows."""
    n_pages, n_kv = (side if torch.is_tensor(side) else side[0]).shape[:2]
    codes = torch.zeros(n_pages, n_kv, 2, 256, dtype=torch.int8, device="cuda")
    scales = torch.zeros(n_pages, n_kv, device="cuda")
    keys, held = _keys(side), 0
    for n in steps:
        paged.page_bounds(i32([p * PAGE + i for p in range(n_pages) for i in range(held, held + n)]), side, codes, scales)
        held += n
        for p in range(n_pages):
            for g in range(n_kv):
                low, high, e = _bounds(keys[p, g, :held])
                assert scales[p, g] == 2.0 ** e, (p, g, held)
                assert codes[p, g, 0].tolist() == low and codes[p, g, 1].tolist() == high, (p, g, held)


def _triplet(n_pages, n_kv, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n_pages, n_kv, PAGE, 256), device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8)
    scales, biases = (torch.zeros(n_pages, n_kv, PAGE, 4, dtype=dtype, device="cuda") for _ in range(2))
    return codes, scales, biases


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_biases_on_whole_steps_beside_tiny_scales(dtype):
    """127 and a little more needs the next step; a little more or less than any other whole step counts too."""
    codes, scales, biases = _triplet(6, 2, dtype, 1)
    scales[0], biases[0] = 1e-20, 127
    scales[1], biases[1] = -1e-20, -127
    scales[2], biases[2, ..., 0], biases[2, ..., 1:] = -1e-25, 127, 64
    scales[3], biases[3] = 1e-30, 3
    biases[3, ..., 0], codes[3, ..., ::3] = 100, 0
    scales[4], biases[4, ..., 1], biases[4, ..., 2] = 1e-38, 2.0 ** 40, -2.0 ** 40
    scales[5], biases[5] = -2.0 ** -40, 1.0
    _check((codes.view(torch.int32).view(torch.uint32), scales, biases), [16])
    _check((codes.view(torch.int32).view(torch.uint32), scales, biases), [1, 2, 5, 8])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scales_and_biases_of_any_size(dtype):
    rng = np.random.default_rng(2)
    codes, scales, biases = _triplet(12, 2, dtype, 2)
    most = 12 if dtype == F16 else 60
    for t, low in ((scales, -24 if dtype == F16 else -120), (biases, -24 if dtype == F16 else -100)):
        x = (1 + rng.integers(0, 4, t.shape) / 4) * 2.0 ** rng.integers(low, most - 8, t.shape) * rng.choice([-1, 1], t.shape)
        t.copy_(torch.tensor(x))
    biases[:4] = biases[:4].float().clamp(-127, 127).round().to(dtype)
    _check((codes.view(torch.int32).view(torch.uint32), scales, biases), [3, 13])


def test_rows_of_16_bits_far_below_the_step():
    """Negative keys lie below zero, positive ones above it, however small they are beside the largest."""
    keys = torch.zeros(3, 1, PAGE, 256, dtype=BF16, device="cuda")
    for p, top in enumerate((2.0 ** 100, 2.0 ** 57, 1.0)):
        keys[p, 0, :, 0] = top
        for c, x in enumerate((1e-30, -1e-30, 2.0 ** -126, -2.0 ** -126, 2.0 ** -133, -2.0 ** -133), 1):
            keys[p, 0, 5, c], keys[p, 0, 9, 10 + c] = x, -x
            keys[p, 0, :, 20 + c] = x
    _check(keys, [16])
    _check(keys, [2, 7, 7])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_groups_beside_one_that_is_no_number(dtype):
    """An infinite or missing bias takes the page's step to its largest; the other groups' codes are their own bounds in such steps."""
    codes, scales, biases = _triplet(3, 1, dtype, 4)
    scales[:], biases[:] = 1e-20, 3
    biases[..., 2] = -127 * 2.0 ** 50
    scales[..., 2], biases[..., 3] = -1.0, 2.0 ** 50
    for p, bad in enumerate((float("inf"), float("-inf"), float("nan"))):
        biases[p, 0, 7, 0] = bad
        if p < 2:
            scales[p, 0, 9, 0] = bad
    side = codes.view(torch.int32).view(torch.uint32), scales, biases
    got, of = torch.zeros(3, 1, 2, 256, dtype=torch.int8, device="cuda"), torch.zeros(3, 1, device="cuda")
    paged.page_bounds(i32(range(3 * PAGE)), side, got, of)
    biases[..., 0] = scales[..., 0] = 0
    keys = _keys(side)
    for p in range(3):
        low, high, e = _bounds(keys[p, 0])
        assert e == 50 and of[p, 0] == 2.0 ** 50
        assert got[p, 0, 0, 64:].tolist() == low[64:] and got[p, 0, 1, 64:].tolist() == high[64:], p
        assert (got[p, 0, 0, :64].long() <= got[p, 0, 1, :64].long()).all()
