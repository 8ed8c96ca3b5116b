"""GPU parity of the norm-and-rope pass and its append with the float64 formula.

Tolerance: the result is rounded once, to eps/2 of its type relative to the value. In front of that lie float32 steps, each off
by half a unit of the last place (2^-24): 21 additions on the longest path of a sum of 256 squares (eight a lane, five lane
exchanges; the sum counts half, under the root), division, root and two products of the norm, cosine and sine (two units each,
and 2^-24 * pi of the angle's turn), two products and a sum: fewer than 32 units of the pair's magnitude together.
"""

import numpy as np
import pytest
import torch

from moespresso_amd.runtime.qwen import kquant, paged
from oracle import paged as oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SECTIONS = {32: (11, 11, 10), 64: (22, 21, 21), 128: (44, 42, 42), 8: (4, 2, 2), 24: (8, 8, 8)}


def _inputs(T, H, G, dtype, rotary, axes, seed, layout="gated", far=120000):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen).to(dtype)

    if layout == "gated":  # a query beside its output gate
        q, k, v = randn(T, H, 512)[:, :, :256], randn(T, G, 256), randn(T, G, 256)
    elif layout == "fused":  # heads of one projection
        row = randn(T, H + 2 * G, 256)
        q, k, v = row[:, :H], row[:, H:H + G], row[:, H + G:]
    elif layout == "heads_first":
        q, k, v = (randn(n, T, 256).transpose(0, 1) for n in (H, G, G))
    else:  # rows that no 16-byte load can read: copied first
        q, k, v = (randn(T, n, 257)[:, :, 1:] for n in (H, G, G))
    inv = (1e7 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float().cuda()
    shape = (T,) if axes == 1 else (3, T)
    pos = torch.randint(0, far, shape, device="cuda", generator=gen, dtype=torch.int32)
    return q, k, v, (1 + 0.2 * randn(256)).to(dtype), (1 + 0.2 * randn(256)).to(dtype), pos, inv


def _wide(t):
    return t.double().cpu().numpy()


def _check(got, x, w, pos, inv, sections, eps=1e-6):
    y = oracle.norm_rope(_wide(x), _wide(w), pos.cpu().numpy(), inv.cpu().numpy(), eps, sections)
    flat = _wide(x) / np.sqrt((_wide(x) ** 2).mean(-1, keepdims=True) + eps) * _wide(w)
    half = inv.numel()
    size = np.abs(flat)
    pair = np.abs(flat[..., :half]) + np.abs(flat[..., half:2 * half])
    size[..., :half] = size[..., half:2 * half] = pair
    bound = torch.finfo(got.dtype).eps / 2 * np.abs(y) + 32 * 2.0 ** -24 * size + torch.finfo(got.dtype).tiny
    err = np.abs(_wide(got) - y)
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,H,G,rotary,axes,layout", [
    (1, 16, 2, 64, 1, "gated"), (1, 1, 1, 16, 1, "gated"), (7, 16, 2, 64, 3, "fused"), (33, 3, 3, 128, 3, "heads_first"),
    (255, 16, 2, 64, 1, "gated"), (256, 5, 1, 256, 1, "fused"), (300, 8, 8, 48, 3, "unaligned"), (2047, 2, 1, 256, 3, "gated"),
    (2051, 4, 2, 64, 3, "fused"),
])
def test_norm_and_rope(T, H, G, rotary, axes, layout, dtype):
    q, k, _, qw, kw, pos, inv = _inputs(T, H, G, dtype, rotary, axes, T + H, layout)
    sections = SECTIONS[rotary // 2] if axes == 3 else None
    got = paged.qk_norm_rope(q, k, qw, kw, pos, inv, sections=sections)
    assert all(t.is_contiguous() and t.dtype == dtype for t in got)
    _check(got[0], q, qw, pos, inv, sections)
    _check(got[1], k, kw, pos, inv, sections)


def test_far_and_negative_positions_and_eps():
    q, k, _, qw, kw, pos, inv = _inputs(40, 4, 2, F32, 64, 1, 1, far=2 ** 31 - 1)
    pos[::2] *= -1
    pos[0], pos[1] = 0, 2 ** 31 - 1
    got = paged.qk_norm_rope(q, k, qw, kw, pos, inv, eps=0.25)
    _check(got[0], q, qw, pos, inv, None, eps=0.25)
    _check(got[1], k, kw, pos, inv, None, eps=0.25)


def test_rows_of_zeros_small_and_large_values():
    q, k, _, qw, kw, pos, inv = _inputs(12, 4, 2, F32, 64, 1, 2)
    q[0], q[1], q[2], q[3] = 0, q[1] * 1e-12, q[2] * 1e15, q[3] * 2.0 ** -140
    _check(paged.qk_norm_rope(q, k, qw, kw, pos, inv)[0], q, qw, pos, inv, None)


def test_a_row_with_nan_stays_alone():
    q, k, _, qw, kw, pos, inv = _inputs(5, 4, 2, BF16, 64, 1, 2)
    want = paged.qk_norm_rope(q, k, qw, kw, pos, inv)[0]
    q[2, 1, 7], q[3, 0, 0] = float("nan"), float("inf")
    got = paged.qk_norm_rope(q, k, qw, kw, pos, inv)[0]
    assert got[2, 1].isnan().all() and got[3, 0].isnan().any()
    hurt = torch.zeros(5, 4, dtype=torch.bool)
    hurt[2, 1] = hurt[3, 0] = True
    assert got[~hurt.cuda()].equal(want[~hurt.cuda()])


def test_no_rows():
    q, k, v, qw, kw, pos, inv = _inputs(3, 4, 2, F16, 64, 1, 2)
    out = paged.qk_norm_rope(q[:0], k[:0], qw, kw, pos[:0], inv)
    assert tuple(out[0].shape) == (0, 4, 256) and tuple(out[1].shape) == (0, 2, 256)
    pages = torch.zeros(2, 2, 16, 256, dtype=F16, device="cuda")
    assert paged.qk_norm_rope_append(q[:0], k[:0], v[:0], qw, kw, pos[:0], inv, pos[:0], pages, pages.clone()).numel() == 0


def _slots(rng, T, n_pages, page):
    slots = rng.permutation(n_pages * page)[:T].astype(np.int32)
    slots[rng.random(T) < 0.2] = -1
    if T > 4:  # beyond the pool, by one and by much
        slots[1], slots[3] = n_pages * page, 2 ** 31 - 1
    return slots


def _fill(pages, rows, slots):
    """What the pages hold after the append of dense rows [T, Hkv, W]."""
    n, _, page, _ = pages.shape
    want = pages.clone()
    ok = (slots >= 0) & (slots < n * page)
    want[slots[ok].long() // page, :, slots[ok].long() % page] = rows[ok]
    return want


@pytest.mark.parametrize("dtype,kind", [(F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)])
@pytest.mark.parametrize("T,H,G,page,axes,layout", [(1, 16, 2, 16, 1, "gated"), (17, 3, 3, 64, 3, "fused"), (300, 16, 2, 16, 1, "gated"),
                                                    (2050, 4, 1, 256, 3, "heads_first"), (40, 8, 2, 32, 1, "unaligned")])
def test_append_of_16_bit_rows(T, H, G, page, axes, layout, dtype, kind):
    q, k, v, qw, kw, pos, inv = _inputs(T, H, G, dtype, 64, axes, T, layout)
    sections = SECTIONS[32] if axes == 3 else None
    n_pages = T // page + 3
    slots = torch.from_numpy(_slots(np.random.default_rng(T), T, n_pages, page)).cuda()
    pages = [torch.randn(n_pages, G, page, 256, device="cuda").to(kind) for _ in range(2)]
    dense = paged.qk_norm_rope(q, k, qw, kw, pos, inv, sections=sections)
    want = [_fill(p, x.to(kind), slots) for p, x in zip(pages, (dense[1], v))]
    got = paged.qk_norm_rope_append(q, k, v, qw, kw, pos, inv, slots, *pages, sections=sections)
    assert got.equal(dense[0]) and pages[0].equal(want[0]) and pages[1].equal(want[1])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,H,G,page,axes", [(1, 16, 2, 16, 1), (19, 5, 1, 64, 3), (517, 16, 2, 64, 1), (2050, 2, 1, 256, 1)])
def test_append_of_8_bit_rows_is_what_the_separate_calls_write(T, H, G, page, axes, dtype):
    q, k, v, qw, kw, pos, inv = _inputs(T, H, G, dtype, 64, axes, T)
    v[0, 0, :64], v[0, 0, 64:128] = 0, 1.5  # groups of one value
    sections = SECTIONS[32] if axes == 3 else None
    n_pages = T // page + 3
    slots = torch.from_numpy(_slots(np.random.default_rng(T), T, n_pages, page)).cuda()
    cache = paged.PagedKVCache(n_pages, G, page_size=page, dtype=dtype, quantized=True)
    for t in cache.keys + cache.values:
        t.view(torch.int32 if t.dtype == torch.uint32 else t.dtype).fill_(7)
    dense = paged.qk_norm_rope(q, k, qw, kw, pos, inv, sections=sections)
    want = []
    for side, x in ((cache.keys, dense[1]), (cache.values, v)):
        parts = kquant.quantize(x)
        want += [_fill(p.view(torch.int32) if p.dtype == torch.uint32 else p, c.view(torch.int32) if c.dtype == torch.uint32 else c, slots)
                 for p, c in zip(side, parts)]
    got = cache.append(q, k, v, qw, kw, pos, inv, slots, sections=sections)
    assert got.equal(dense[0])
    for t, w in zip(cache.keys + cache.values, want):
        assert (t.view(torch.int32) if t.dtype == torch.uint32 else t).equal(w)


def test_append_beyond_4_gb_of_pages():
    """Row offsets of 33 bits: the last pages of a pool of 5 GB a side."""
    q, k, v, qw, kw, pos, inv = _inputs(3, 4, 2, BF16, 64, 1, 5)
    n_pages, page = 20000, 256
    keys, values = (torch.empty(n_pages, 2, page, 256, dtype=BF16, device="cuda") for _ in range(2))
    for side in (keys, values):
        side[-2:], side[0] = 0, 0
    slots = torch.tensor([n_pages * page - 1, n_pages * page - page - 3, 2], dtype=torch.int32, device="cuda")
    paged.qk_norm_rope_append(q, k, v, qw, kw, pos, inv, slots, keys, values)
    want = paged.qk_norm_rope(q, k, qw, kw, pos, inv)[1]
    for side, x in ((keys, want), (values, v)):
        assert side[-1, :, -1].equal(x[0]) and side[-2, :, -3].equal(x[1]) and side[0, :, 2].equal(x[2])
        assert int((side[-2:] != 0).any(-1).sum()) == 4 and int((side[0] != 0).any(-1).sum()) == 2
