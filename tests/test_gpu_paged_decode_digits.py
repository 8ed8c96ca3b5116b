"""Decode attention over 8-bit pages whose rows or groups differ in size by orders of magnitude, against float64.

Tolerance, from the arithmetic, by channel. A score is off by at most 260 * 2^-24 of the sum of its products' magnitudes, which
moves the result by twice that of the values' sum. A weight times a scale is two float16 terms, each off by half a step: 2^-22 of
it; taken 2^11 times as large in multiples of a power of two that is less than twice the largest scale, a term ends at 2^-25 of
that, so that n weights lose n * 2^-36 of twice the largest scale and 128 codes. Codes (from 128 on) and biases are
summed apart, in float32: over n / 8 additions where four waves share the keys, n / 4 where one has them, of the weights' and of
the values' sums. The result is rounded once more, to eps / 2 of its type (beyond float16's largest number it is infinite).
"""

import pytest
import torch

from moespresso_amd.runtime.qwen import paged

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAGE, HOT = 64, 7 * 64 + 11  # a key that takes most of the weight of some queries


def _wide(side):
    codes, scale, bias = side
    scale, bias = (t.double().repeat_interleave(64, -1) for t in (scale, bias))
    codes = codes.double() - 128
    return tuple(t.reshape(-1, 256) for t in (codes * scale + (bias + 128 * scale), (codes * scale).abs() + (bias + 128 * scale).abs(), scale))


def _check(dtype, n, queries, seed, change):
    """`queries` of four heads over n keys of equal scores but one, of values whose scales `change` has changed."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pages = -(-n // PAGE)
    shape = (pages, 1, PAGE)
    k = [torch.full(shape + (256,), 128, device="cuda", dtype=torch.uint8), torch.ones(shape + (4,), device="cuda")]
    k[0].view(-1, 256)[HOT, 0] = 138
    k.append(-128 * k[1])
    v = [torch.randint(0, 256, shape + (256,), device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8),
         0.03 * (0.5 + torch.rand(shape + (4,), device="cuda", generator=gen))]
    change(v[1].view(-1, 4))
    v.append(v[1] * -(96 + 64 * torch.rand(v[1].shape, device="cuda", generator=gen)))
    q = torch.zeros(queries, 4, 256, device="cuda")
    q[:, :, 0] = torch.tensor([0.0, 0.5, 1.0, 1.375], device="cuda")  # (whole in every type)
    tables = torch.arange(pages, device="cuda", dtype=torch.int32)[None]
    pack = lambda side: (side[0].view(torch.int32).view(torch.uint32), *side[1:])
    lens, requests = torch.full((queries,), n, device="cuda", dtype=torch.int32), torch.zeros(queries, device="cuda", dtype=torch.int32)
    got = paged.sdpa_decode_paged_q8(q.to(dtype), *pack(k), *pack(v), tables, lens, 1.0, requests=requests)
    keys, most, _ = (t[:n] for t in _wide(k))
    values, size, scale = (t[:n] for t in _wide(v))
    w = torch.softmax(q[0].double() @ keys.t(), -1)
    want = w @ values
    most = (q[0].double().abs() @ most.t()).amax(-1, keepdim=True)
    adds = n / (8 if queries < 128 else 4) + 8
    bound = (w @ size) * (2 * 260 * 2.0 ** -24 * most + 2.0 ** -22 + 2 * adds * 2.0 ** -24)
    bound += n * 2.0 ** -36 * 2 * 128 * scale.amax(0) + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).tiny
    # (a result beyond the type's largest number, by more than it may be off, is infinite; one that may lie on either side is either)
    top = torch.finfo(dtype).max
    over = want.abs() - bound > top
    assert got.double()[over.expand_as(got)].equal((want.sign() * torch.inf).expand_as(got)[over.expand_as(got)])
    err = torch.where(want.abs() + bound > top, 0.0, (got.double() - want).abs())
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("queries", [1, 130])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [500, 5000])
def test_a_key_whose_scales_are_far_above_the_others(n, dtype, queries):
    """Where its value is a small difference of its code's and its bias's parts, an error of its weight is many times that value."""
    for ratio in (1.0, 1e2, 1e4):
        def change(scales):
            scales[HOT] *= ratio

        _check(dtype, n, queries, 1, change)


@pytest.mark.parametrize("queries", [1, 130])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [500, 5000, 37000])
def test_groups_of_channels_of_different_size(n, dtype, queries):
    """No group loses digits to another's scales, whichever is met first."""
    for ratio in (1e2, 1e4, 1e6):
        def change(scales):
            scales[:, 1] *= ratio
            scales[:, 3] /= ratio
            scales[n // 2:, 2] *= ratio
            scales[:n // 3, 0] *= ratio

        _check(dtype, n, queries, 2, change)
