"""CPU model of how the kernel of shared prefixes deals out its work: every tile of every prefix meets every member once, every
tile of own rows its query, every partial has a place of its own, and the second kernel finds them."""

import ctypes

import numpy as np
import pytest

from moespresso_amd import _lib

TILE, GROUPS, COLUMNS, MIN_SHARE, DIM = 32, 256, 32, 4, 256


def _ceil(a, b):
    return -(-a // b)


def _units(batch, n_prefixes, n_kv, rep):
    per = COLUMNS // rep
    return n_kv * ((batch + min(n_prefixes, batch) * (per - 1)) // per + batch)


def _slots(batch, n_prefixes, n_kv, rep):
    """Workgroups, and places for partials of prefix pieces and own ones."""
    pieces = max(GROUPS, GROUPS // 2 + _units(batch, n_prefixes, n_kv, rep))
    return pieces, pieces - batch * n_kv, max(GROUPS, GROUPS // 2 + batch * n_kv)


def _plan(prefix_lens, groups, lens, n_kv, rep):
    """Entries (prefixes, then queries): blocks, ranges, tiles, first piece; the number of pieces, and of those of prefixes."""
    per = COLUMNS // rep
    groups = [g if 0 <= g < len(prefix_lens) and prefix_lens[g] > 0 else -1 for g in groups]
    tiles = [_ceil(n, TILE) for n in list(prefix_lens) + list(lens)]
    blocks = [_ceil(groups.count(g), per) for g in range(len(prefix_lens))] + [1] * len(lens)
    total, units = n_kv * sum(b * t for b, t in zip(blocks, tiles)), n_kv * sum(blocks)
    share = max(MIN_SHARE, _ceil(total, max(GROUPS - units, GROUPS // 2)))
    entries, at, of_prefixes = [], 0, 0
    for e, (b, t) in enumerate(zip(blocks, tiles)):
        ranges = max(1, _ceil(t, share))
        entries.append((b, ranges, t, at))
        at += n_kv * b * ranges
        if e == len(prefix_lens) - 1:
            of_prefixes = at
    return groups, entries, at, of_prefixes


def _bundle_piece(bundle, block, bundles, blocks):
    q = bundle // 8
    return 8 * blocks * q + block * min(8, bundles - 8 * q) + bundle % 8


@pytest.mark.parametrize("batch,n_prefixes,n_kv,rep,most_prefix,most", [
    (1, 1, 1, 1, 40, 40), (2, 1, 2, 8, 137, 40), (16, 1, 2, 8, 32768, 512), (61, 5, 2, 8, 9001, 2000), (256, 1, 2, 8, 8192, 700),
    (33, 1, 2, 8, 20001, 300), (7, 20, 4, 5, 900, 90), (300, 300, 1, 16, 2000, 10), (2048, 3, 8, 1, 300, 60), (40, 2, 1, 3, 0, 500),
    (9, 2, 2, 7, 60000, 0), (100, 100, 8, 4, 70, 70)])
def test_every_tile_is_met_once_and_every_partial_has_a_place(batch, n_prefixes, n_kv, rep, most_prefix, most):
    rng = np.random.default_rng(batch + n_prefixes)
    prefix_lens = [int(n) for n in rng.integers(0, most_prefix + 1, n_prefixes)]
    prefix_lens[-1] = most_prefix
    raw = [int(g) for g in rng.integers(-1, n_prefixes + 1, batch)]
    lens = [int(n) for n in rng.integers(0, most + 1, batch)]
    groups, entries, pieces, of_prefixes = _plan(prefix_lens, raw, lens, n_kv, rep)
    grid, prefix_slots, own_slots = _slots(batch, n_prefixes, n_kv, rep)
    assert pieces <= grid and of_prefixes <= prefix_slots and pieces - of_prefixes <= own_slots
    met, places = {}, set()
    per = COLUMNS // rep
    for number in range(pieces):
        e = max(i for i, (b, r, t, at) in enumerate(entries) if at <= number and b)
        blocks, ranges, tiles, at = entries[e]
        i = number - at
        if e < n_prefixes:
            bundles = n_kv * ranges
            q = i // (8 * blocks)
            j, m = i - 8 * blocks * q, min(8, bundles - 8 * q)
            block, bundle = j // m, 8 * q + j % m
            assert _bundle_piece(bundle, block, bundles, blocks) == i
            members = [r for r in range(batch) if groups[r] == e][block * per:(block + 1) * per]
            assert members and len(members) * rep <= COLUMNS
        else:
            block, bundle, members = 0, i, [e - n_prefixes]
        kvh, part = divmod(bundle, ranges)
        assert 0 <= kvh < n_kv
        place = (e < n_prefixes, number if e < n_prefixes else number - of_prefixes)
        assert place not in places and place[1] < (prefix_slots if place[0] else own_slots)
        places.add(place)
        for tile in range(tiles * part // ranges, tiles * (part + 1) // ranges):
            for r in members:
                key = (e, kvh, tile, r)
                assert key not in met
                met[key] = place
    for r in range(batch):
        for e in ([groups[r]] if groups[r] >= 0 else []) + [n_prefixes + r]:
            for kvh in range(n_kv):
                blocks, ranges, tiles, at = entries[e]
                rank = [i for i in range(batch) if groups[i] == e].index(r) if e < n_prefixes else 0
                for tile in range(tiles):
                    part = next(p for p in range(ranges) if tile < tiles * (p + 1) // ranges)
                    i = _bundle_piece(kvh * ranges + part, rank // per, n_kv * ranges, blocks) if e < n_prefixes else kvh * ranges + part
                    place = (e < n_prefixes, at + i - (0 if e < n_prefixes else of_prefixes))
                    assert met.pop((e, kvh, tile, r)) == place
    assert not met


@pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")
@pytest.mark.parametrize("batch,hq,hkv,n_prefixes", [(1, 1, 1, 1), (16, 16, 2, 1), (2048, 64, 4, 2048), (100, 48, 3, 7), (5, 15, 3, 9)])
def test_the_workspace_holds_every_place(batch, hq, hkv, n_prefixes):
    rep = hq // hkv
    _, prefix_slots, own_slots = _slots(batch, n_prefixes, hkv, rep)
    words = prefix_slots * COLUMNS * (DIM + 2) + own_slots * (rep * DIM + 32) + batch * hkv * 8
    lib = _lib.lib()
    lib.mspr_sdpa_decode_paged_shared_workspace_bytes.restype = ctypes.c_size_t
    assert lib.mspr_sdpa_decode_paged_shared_workspace_bytes(batch, hq, hkv, n_prefixes) == 4 * words
