"""CPU model of how the paged decode kernel deals out its work and forms its addresses: every row of every request is
attended once, every address lies in its buffer, every output is written once, from the partials that its parts left."""

import numpy as np
import pytest

from moespresso_amd import _lib

TILE, WAVES, GROUPS, MIN_TILES, MANY_ROWS = 32, 4, 256, 2, 128
GROUP_COST, WAVE_COST = 8, 2


def _row_tiles(n):
    """Tiles that a row of n keys counts for."""
    return max(MIN_TILES, -(-n // TILE))


def _most(batch, n_kv):
    """Shares at most, and waves that take a share's tiles in turn: of few rows workgroups have shares, of many waves."""
    return (GROUPS * WAVES, 1) if batch * n_kv >= MANY_ROWS else (GROUPS, WAVES)


def _shares(batch, n_kv, cap):
    return min(_most(batch, n_kv)[0], -(-batch * n_kv * (_row_tiles(cap) + MIN_TILES) // MIN_TILES))


def _line(lens, n_kv, cap):
    """Length of the line of all rows, what a row counts for beside its tiles, and the shares' length."""
    most, waves = _most(len(lens), n_kv)
    tiles = sum(_row_tiles(n) for n in lens) * n_kv
    cost = 0 if cap <= MIN_TILES * TILE else min(GROUP_COST if waves == WAVES else WAVE_COST, -(-tiles // most))
    total = tiles + cost * n_kv * len(lens)
    return total, cost, max(MIN_TILES, -(-total // most))


def _numbers(batch, n_kv, cap, lens):
    """The share of every wave (of few rows: of every workgroup) that is launched."""
    most, waves = _most(batch, n_kv)
    groups = min(GROUPS, _shares(batch, n_kv, cap))
    if waves == WAVES:
        return list(range(groups))
    spread = _line(lens, n_kv, cap)[0] <= MIN_TILES * GROUPS * (WAVES // 2)
    return [g + groups * w if spread else g * WAVES + w for g in range(groups) for w in range(WAVES)]


def _parts(wg, lens, n_kv, cap):
    """The parts of rows that share wg holds: (request, KV head, first tile, end tile, tiles of the row), and its share."""
    total, cost, share = _line(lens, n_kv, cap)
    pos, end = wg * share, min((wg + 1) * share, total)
    parts, before = [], 0
    for b, n in enumerate(lens):
        for kvh in range(n_kv):
            t = _row_tiles(n)
            lo, hi = max(pos, before), min(end, before + t)
            if lo < hi:
                parts.append((b, kvh, lo - before, hi - before, t))
            before += t + cost
    return parts, share


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
                                                   (130, 8, 16, 3), (16, 2, 256, 40), (64, 4, 128, 2), (127, 1, 16, 9),
                                                   (300, 2, 16, 1), (70, 8, 32, 4), (600, 1, 64, 2)])
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
    most, waves = _most(batch, n_kv)
    slots = {}  # partials by row: the slots that the shares write, in the order of the row's tiles
    cuts, written = {}, set()
    grid = _shares(batch, n_kv, cap)
    for wg in range(grid):
        parts, share = _parts(wg, lens, n_kv, cap)
        for b, kvh, tile0, tile1, row_tiles in parts:
            assert (b, kvh) not in written
            if tile0 == 0 and tile1 == row_tiles:
                written.add((b, kvh))
            else:
                slots.setdefault((b, kvh), []).append(2 * wg + (tile0 == 0))
                if tile0 == 0:
                    assert wg not in cuts  # only a share's last part begins a row that it does not end
                    cuts[wg] = (b, kvh), wg + -(-(row_tiles - tile1) // share)
            last = min(tile1, -(-lens[b] // TILE))
            for wave in range(waves):
                mine = -(-(last - tile0 - wave) // waves) if last - tile0 > wave else 0
                for it in range(mine):
                    for u in range(2):
                        key = (tile0 + wave + waves * it) * TILE + 16 * u
                        p = tables[b, key // page] if key < lens[b] else -1
                        good = 0 <= p < n_pages
                        row = ((p if good else 0) * n_kv + kvh) * page + key % page
                        rows = min(16, max(0, lens[b] - key)) if good else 0
                        assert 0 <= row and row + rows <= n_pages * n_kv * page and key % page + rows <= page
                        seen[b, kvh, key:key + rows] += 1
    for b, n in enumerate(lens):
        assert (seen[b, :, :n] == 1).all() and not seen[b, :, n:].any()
    # every row is written once: whole, or by the merge of exactly the slots that its parts went to
    merged = {row: [2 * w + (w == first) for w in range(first, last + 1)] for first, (row, last) in cuts.items()}
    assert merged == slots and not written & set(merged) and len(written) + len(merged) == batch * n_kv
    assert all(0 <= s < 2 * grid for part in slots.values() for s in part)
    assert len({s for part in slots.values() for s in part}) == sum(len(part) for part in slots.values())
    # every share with work has one wave, and nothing is left over; waves without work stay in the table of cuts
    numbers = _numbers(batch, n_kv, cap, lens)
    assert len(set(numbers)) == len(numbers) and set(range(grid)) <= set(numbers) and max(numbers) < most
    assert not any(_parts(n, lens, n_kv, cap)[0] for n in set(numbers) - set(range(grid)))
    assert not _parts(grid, lens, n_kv, cap)[0]
    if _row_tiles(cap) == MIN_TILES and batch * n_kv <= most:
        assert not merged  # the merge is not launched


@pytest.mark.parametrize("n_kv", [1, 2, 8])
def test_no_share_with_work_is_behind_those_that_are_launched(n_kv):
    rng = np.random.default_rng(n_kv)
    for batch in (1, 2, 3, 7, 8, 31, 32, 63, 64, 65, 100, 127, 128, 129, 255, 256, 300, 600, 1000):
        for cap in (16, 32, 48, 64, 80, 96, 112, 128, 160, 256, 272, 512, 1040, 4096, 70000):
            for kind in ("all", "one", "empty", "any"):
                total, _, share = _line(_lens(rng, batch, cap, kind), n_kv, cap)
                assert -(-total // share) <= _shares(batch, n_kv, cap), (batch, cap, kind)


@pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")
@pytest.mark.parametrize("batch,heads,n_kv,page,width", [(1, 16, 2, 64, 1), (1, 16, 2, 64, 2048), (256, 64, 8, 16, 100), (65535, 1, 1, 16, 1),
                                                             (127, 4, 1, 16, 3), (128, 4, 1, 16, 3), (129, 4, 1, 16, 2)])
def test_the_workspace_holds_every_part(batch, heads, n_kv, page, width):
    need = _shares(batch, n_kv, page * width) * 2 * (heads // n_kv * 256 + 32) * 4 + 3 * 4 * GROUPS * WAVES
    assert need <= _lib.lib().mspr_sdpa_decode_paged_workspace_bytes(batch, heads, n_kv, page, width) <= need + 64
