"""Attention behind shared prefixes over values whose channels are of very different size: every channel keeps the digits it would have
alone, whichever form of the kernels takes the call (tables of few entries, and of so many that prefixes are a kernel's own).

Bound: that of paged_reference.py, which for bfloat16 rows is of each channel by itself (float32 sums: no term of another channel's
values). An infinite value makes its own channel no number of those that see it, and leaves all other channels as they are."""

import numpy as np
import pytest
import torch

import paged_reference as ref
from paged_reference import BF16, i32
from moespresso_amd.runtime.qwen import paged

pytestmark = pytest.mark.gpu

SCALE = 256 ** -0.5
PAGE, HEADS, KV_HEADS = 16, 16, 2
PREFIXES, GROUPS = [300, 40, 1000], [0] * 9 + [1] * 4 + [2] * 6 + [-1]
LENS = [50, 1, 0, 70, 16] * 4


def _case(seed, prefix_lens, long):
    rng = np.random.default_rng(seed)
    n_pages = sum(-(-n // PAGE) for n in [*prefix_lens, *LENS])
    order = list(rng.permutation(n_pages))
    prefixes = ref.tables(rng, prefix_lens, PAGE, -(-max(prefix_lens) // PAGE), n_pages, order)
    tables = ref.tables(rng, LENS, PAGE, -(-max(LENS) // PAGE), n_pages, order)
    columns = len(LENS) * HEADS // KV_HEADS
    if long:
        prefixes = np.pad(prefixes, ((0, 0), (0, (5 << 19) // (columns * PAGE) + 1)), constant_values=-1)
    assert (columns * prefixes.shape[1] * PAGE >= 5 << 19) == long
    keys, values = ref.cache(rng, (n_pages, KV_HEADS, PAGE, 256), BF16, "rows")
    return ref.rows(rng, (len(LENS), HEADS, 256), BF16) * 2, keys, values, prefixes, tables


def _places(prefixes, prefix_lens, tables, n_pages):
    return [[(ref.places(prefixes[g], prefix_lens[g], PAGE, n_pages) if g >= 0 else []) + ref.places(tables[r], LENS[r], PAGE, n_pages)] * KV_HEADS
            for r, g in enumerate(GROUPS)]


def _check(q, keys, values, prefixes, prefix_lens, tables, but=()):
    """Every channel within its own bound; those of ``but`` are not looked at."""
    got = paged.sdpa_decode_paged_shared(q, keys, values, i32(prefixes), i32(prefix_lens), i32(GROUPS), i32(tables), i32(LENS), SCALE)
    held = values.clone()
    held[..., list(but)] = 0
    want, bound = ref.attention(q, keys, held, _places(prefixes, prefix_lens, tables, keys.shape[0]), SCALE)
    bound = bound + torch.finfo(BF16).eps / 2 * want.abs() + torch.finfo(BF16).tiny
    some = [c for c in range(256) if c not in but]
    err = (got.double() - want).abs()[..., some]
    assert (err <= bound[..., some]).all(), (err / bound[..., some]).nan_to_num(9e9).amax((0, 1)).max()
    return got


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("outliers", [{7: 2.0 ** 20}, {0: 2.0 ** 12, 100: 2.0 ** -20, 255: 2.0 ** 28}, {3: 1e30, 64: 1e-30}])
def test_channels_beside_outliers_keep_their_digits(outliers, long):
    q, keys, values, prefixes, tables = _case(1, PREFIXES, long)
    for channel, by in outliers.items():
        values[..., channel] *= by
    _check(q, keys, values, prefixes, PREFIXES, tables)


@pytest.mark.parametrize("long", [False, True])
def test_channels_beside_an_infinite_one_keep_theirs(long):
    """Also where weights are nearly alike and sums, before they are divided by the weights', lie beyond float16. (Not quite alike: the rest
    of a weight of 1 is 0, which makes NaN of an infinite value.)"""
    prefix_lens = [4096, 40, 1000]
    q, keys, values, prefixes, tables = _case(2, prefix_lens, long)
    q[:, ::3] *= 2.0 ** -10
    values = values.abs() * 1000
    values[int(prefixes[0][5]), :, 3, 17] = float("inf")
    values[int(prefixes[2][9]), :, 0, 200] = float("-inf")
    got = _check(q, keys, values, prefixes, prefix_lens, tables, but=(17, 200))
    group = torch.tensor(GROUPS)
    assert not got[group == 0][..., 17].isfinite().any() and got[group != 0][..., 17].isfinite().all()
    assert not got[group == 2][..., 200].isfinite().any() and got[group != 2][..., 200].isfinite().all()
