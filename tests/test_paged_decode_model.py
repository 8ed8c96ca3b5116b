"""CPU model of how the paged decode kernel deals out its work and forms its addresses: every row of every request is
attended once, every address lies in its buffer, and no lengths need more ranges than the grid and the workspace have."""

import numpy as np
import pytest

from moespresso_amd import _lib

TILE, WAVES, RANGES, MIN_TILES = 32, 4, 256, 4


def _tiles(n, cap):
    return -(-min(max(n, 0), cap) // TILE)


def _ranges(batch, n_kv, cap):
    rows = batch * n_kv
    return min(rows * -(-(-(-cap // TILE)) // MIN_TILES), rows + RANGES)


def _find(wg, lens, n_kv, cap):
    """(request, KV head, first tile, end tile, its first range, its ranges) of a workgroup, or None."""
    tiles = [_tiles(n, cap) for n in lens]
    per = max(MIN_TILES, (sum(tiles) * n_kv + RANGES - 1) // RANGES)
    before = 0
    for b, t in enumerate(tiles):
        n = max(1, -(-t // per))
        if wg < before + n * n_kv:
            index, kvh = divmod(wg - before, n_kv)
            return b, kvh, index * per, min((index + 1) * per, t), before, n
        before += n * n_kv
    return None


def _lens(rng, batch, cap, kind):
    if kind == "all":
        return [cap] * batch
    if kind == "one":
        return [cap] + [1] * (batch - 1)
    if kind == "empty":
        return [0] * batch
    return [int(n) for n in rng.integers(0, cap + 1, size=batch)]


@pytest.mark.parametrize("kind", ["all", "one", "empty", "any"])
@pytest.mark.parametrize("batch,n_kv,page,width", [(1, 1, 16, 1), (1, 2, 16, 9), (1, 2, 64, 128), (3, 2, 16, 100), (65, 1, 32, 7),
                                                   (130, 8, 16, 3), (16, 2, 256, 40), (64, 4, 128, 2)])
def test_every_row_is_attended_once_and_every_address_lies_in_its_buffer(kind, batch, n_kv, page, width):
    rng = np.random.default_rng(batch * 1000 + width)
    cap = page * width
    lens = _lens(rng, batch, cap, kind)
    held = [-(-n // page) for n in lens]
    n_pages = sum(held) + 1
    order = rng.permutation(n_pages)
    tables, used = np.full((batch, width), -7), 0
    for b, h in enumerate(held):
        tables[b, :h] = order[used:used + h]
        used += h
    seen = np.zeros((batch, n_kv, cap), dtype=np.int64)
    plan = {}
    grid = _ranges(batch, n_kv, cap)
    for wg in range(grid):
        r = _find(wg, lens, n_kv, cap)
        if r is None:
            continue
        b, kvh, tile0, tile1, first, count = r
        assert plan.setdefault(b, (first, count)) == (first, count)
        assert first <= wg < first + count * n_kv <= grid  # partials of a request lie at first + index * n_kv + kvh
        for wave in range(WAVES):
            mine = (tile1 - tile0 - wave + WAVES - 1) // WAVES if lens[b] > 0 and tile1 - tile0 > wave else 0
            for it in range(mine):
                for u in range(2):
                    key = (tile0 + wave + WAVES * it) * TILE + 16 * u
                    p = tables[b, key // page] if key < lens[b] else -1
                    good = 0 <= p < n_pages
                    row = ((p if good else 0) * n_kv + kvh) * page + key % page
                    assert 0 <= row and row + 16 <= n_pages * n_kv * page and key % page + 16 <= page
                    n = min(16, max(0, lens[b] - key)) if good else 0
                    seen[b, kvh, key:key + n] += 1
    for b, n in enumerate(lens):
        assert (seen[b, :, :n] == 1).all() and not seen[b, :, n:].any()
        assert b in plan  # a workgroup of its own, also without rows: the output is written
    assert _find(grid, lens, n_kv, cap) is None  # none is left over


@pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")
@pytest.mark.parametrize("batch,heads,n_kv,page,width", [(1, 16, 2, 64, 1), (1, 16, 2, 64, 2048), (256, 64, 8, 16, 100), (65535, 1, 1, 16, 1)])
def test_the_workspace_holds_every_range(batch, heads, n_kv, page, width):
    need = _ranges(batch, n_kv, page * width) * (heads // n_kv * 256 + 32) * 4 + 8 * batch
    assert need <= _lib.lib().mspr_sdpa_decode_paged_workspace_bytes(batch, heads, n_kv, page, width) <= need + 64
