"""CPU model of how the kernel of shared prefixes deals out its work: every tile of every prefix meets every member once, every
tile of own rows its query, every partial has a place of its own, and the second kernel finds them."""

import numpy as np
import pytest

from moespresso_amd import _lib

TILE, GROUPS, MIN_SHARE, DIM, NARROW = 32, 256, 4, 256, 32
WIDE = 128  # columns of a block where prefixes are a kernel's own


def _ceil(a, b):
    return -(-a // b)


def _block(batch, n_prefixes, rep, wide):
    """Columns of a block of members, at most (wide: as many; 0: both kinds of rows in one launch)."""
    used = min(n_prefixes, batch)
    return min(wide, _ceil(_ceil((2 if used > 1 else 1) * batch * rep, used), 32) * 32) if wide else NARROW


def _pieces_of(units):
    return max(GROUPS, GROUPS // 2 + units)


def _slots(batch, n_prefixes, n_kv, rep, wide):
    """Workgroups, places for partials of prefixes, and of own rows."""
    per = _block(batch, n_prefixes, rep, wide) // rep
    own, blocks = batch * n_kv, n_kv * ((batch + min(n_prefixes, batch) * (per - 1)) // per)
    pieces = _pieces_of(blocks if wide else own + blocks)
    return pieces, pieces if wide else pieces - own, own * rep if wide else _pieces_of(own)


def _plan(tiles, blocks, n_kv, least, step=None):
    """Ranges and first piece of every entry of so many tiles and blocks, and the number of pieces. ``step``: of few prefixes lengths in
    such steps are tried."""
    total, units = n_kv * sum(b * t for b, t in zip(blocks, tiles)), n_kv * sum(blocks)
    share = max(MIN_SHARE, _ceil(total, max(GROUPS - units, GROUPS // 2)))
    if step and len(tiles) <= 16:
        first = _ceil(max(MIN_SHARE, _ceil(total, GROUPS)), step) * step
        tried = np.arange(first, first + 64 * step, step)
        pieces = np.zeros(64, dtype=int)
        for b, t in zip(blocks, tiles):  # (in float32, as the kernel's)
            q = (np.float32(t) + tried.astype(np.float32) - np.float32(0.5)) * (np.float32(1) / tried.astype(np.float32))
            assert (q.astype(int) == -(-t // tried)).all()
            pieces += b * q.astype(int)
        if (pieces * n_kv <= GROUPS).any():
            share = min(share, int(tried[np.argmax(pieces * n_kv <= GROUPS)]))
    entries, at = [], 0
    for b, t in zip(blocks, tiles):
        ranges = max(least, _ceil(t, share))
        entries.append((b, ranges, t, at))
        at += n_kv * b * ranges
    return entries, at


def _bundle_piece(bundle, block, bundles, blocks):
    q = bundle // 8
    return 8 * blocks * q + block * min(8, bundles - 8 * q) + bundle % 8


@pytest.mark.parametrize("wide,step", [(0, None), (WIDE, 1), (WIDE, 2)])
@pytest.mark.parametrize("batch,n_prefixes,n_kv,rep,most_prefix,most", [
    (1, 1, 1, 1, 40, 40), (2, 1, 2, 8, 137, 40), (16, 1, 2, 8, 32768, 512), (61, 5, 2, 8, 9001, 2000), (256, 1, 2, 8, 8192, 700),
    (33, 1, 2, 8, 20001, 300), (7, 20, 4, 5, 900, 90), (300, 300, 1, 16, 2000, 10), (2048, 3, 8, 1, 300, 60), (40, 2, 1, 3, 0, 500),
    (9, 2, 2, 7, 60000, 0), (100, 100, 8, 4, 70, 70)])
def test_every_tile_is_met_once_and_every_partial_has_a_place(batch, n_prefixes, n_kv, rep, most_prefix, most, wide, step):
    rng = np.random.default_rng(batch + n_prefixes)
    prefix_lens = [int(n) for n in rng.integers(0, most_prefix + 1, n_prefixes)]
    prefix_lens[-1] = most_prefix
    lens = [int(n) for n in rng.integers(0, most + 1, batch)]
    groups = [g if 0 <= g < n_prefixes and prefix_lens[g] > 0 else -1 for g in (int(g) for g in rng.integers(-1, n_prefixes + 1, batch))]
    block = _block(batch, n_prefixes, rep, wide)
    per = block // rep
    members = [[r for r in range(batch) if groups[r] == g] for g in range(n_prefixes)]
    blocks = [_ceil(len(m), per) for m in members]
    prefix_tiles, own_tiles = ([_ceil(n, TILE) for n in ns] for ns in (prefix_lens, lens))
    grid, prefix_slots, own_slots = _slots(batch, n_prefixes, n_kv, rep, wide)
    if not wide:  # one kernel: prefixes, then own rows
        entries, pieces = _plan(prefix_tiles + own_tiles, blocks + [1] * batch, n_kv, 1)
        prefixes, own = entries[:n_prefixes], entries[n_prefixes:]
        of_prefixes = own[0][3]
        own = [(b, r, t, at - of_prefixes) for b, r, t, at in own]
        assert pieces <= grid and of_prefixes <= prefix_slots and pieces - of_prefixes <= own_slots
    else:
        prefixes, of_prefixes = _plan(prefix_tiles, blocks, n_kv, 0, step)
        own = []  # (dealt out as test_paged_decode_model.py has it)
        assert of_prefixes <= grid and of_prefixes <= prefix_slots
    met, places = {}, set()
    for g, (n_blocks, ranges, tiles, at) in enumerate(prefixes):
        a_block = _ceil(len(members[g]), n_blocks) if n_blocks and wide else per  # (wide ones about equal)
        bundles = n_kv * ranges
        for i in range(n_blocks * bundles):
            q = i // (8 * n_blocks)
            j, m = i - 8 * n_blocks * q, min(8, bundles - 8 * q)
            b, bundle = j // m, 8 * q + j % m
            assert _bundle_piece(bundle, b, bundles, n_blocks) == i and at + i < prefix_slots and at + i not in places
            places.add(at + i)
            kvh, part = divmod(bundle, ranges)
            some = members[g][b * a_block:(b + 1) * a_block]
            assert some and len(some) * rep <= block and 0 <= kvh < n_kv
            for k, r in enumerate(some):
                column = b * block + k * rep  # where the last kernel looks for it
                assert (column // block, column % block + rep <= block) == (b, True)
                for tile in range(tiles * part // ranges, tiles * (part + 1) // ranges):
                    assert (g, kvh, tile, r) not in met
                    met[g, kvh, tile, r] = at + _bundle_piece(kvh * ranges + part, column // block, bundles, n_blocks)
                    assert met[g, kvh, tile, r] == at + i
    for g, m in enumerate(members):
        for r in m:
            for kvh in range(n_kv):
                for tile in range(prefix_tiles[g]):
                    met.pop((g, kvh, tile, r))
    assert not met
    taken = set()
    for _, ranges, tiles, at in own:
        for i in range(n_kv * ranges):
            assert at + i < own_slots and at + i not in taken
            taken.add(at + i)
        assert sum(tiles * (p + 1) // ranges - tiles * p // ranges for p in range(ranges)) == tiles


@pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")
@pytest.mark.parametrize("batch,hq,hkv,page,width,n_prefixes", [(1, 1, 1, 16, 1, 1), (16, 16, 2, 64, 8, 1), (2048, 64, 4, 16, 100, 2048),
                                                                (100, 48, 3, 256, 7, 7), (5, 15, 3, 16, 3, 9), (4, 16, 2, 64, 9, 1)])
def test_the_workspace_holds_every_place(batch, hq, hkv, page, width, n_prefixes):
    rep, lib = hq // hkv, _lib.lib()

    def bytes_of(wide):
        _, prefix_slots, own_slots = _slots(batch, n_prefixes, hkv, rep, wide)
        n = prefix_slots * _block(batch, n_prefixes, rep, wide) * (DIM + 4) + own_slots * (DIM if wide else rep * DIM)
        n = 4 * n + _ceil(own_slots * (8 if wide else 128), 16) * 16 + batch * hkv * 32
        return n + (lib.mspr_sdpa_decode_paged_workspace_bytes(batch, hq, hkv, page, width) if wide else 0)

    most = bytes_of(0) if batch * rep <= NARROW else max(bytes_of(0), bytes_of(WIDE))
    assert lib.mspr_sdpa_decode_paged_shared_workspace_bytes(batch, hq, hkv, page, width, n_prefixes) == most
