"""CPU model of what the kernels for shared prefixes share in LDS: asynchronous copies into a ring, what is made of them, and the reads of
eight waves, between barriers. Nothing may be read that has not landed, and nothing written that another wave may still read.

Waves run freely between two barriers, so that everything of one such epoch may happen in any order; a copy may land from when it
is issued to when a wait of the wave that issued it says that it has."""

import re

import pytest

from moespresso_amd import build

SOURCE = open(f"{build.CSRC}/paged_shared.hip").read()


def _constant(name):
    return int(re.search(rf"constexpr int {name} = (\d+);", SOURCE)[1])


class Memory:
    """Places that are written and read; conflicts within an epoch, and reads of what has not landed."""

    def __init__(self):
        self.epoch, self.content, self.read, self.written, self.flying = 0, {}, {}, {}, []

    def barrier(self):
        self.epoch += 1
        self.read, self.written = {}, {}

    def reads(self, wave, place, what):
        assert self.content.get(place) == what, f"{place} holds {self.content.get(place)}, not {what}"
        assert not any(p == place for p, *_ in self.flying), f"{place} is being copied to"
        others = self.written.get(place, set()) - {wave}
        assert not others, f"waves {others} write {place} in the epoch in which wave {wave} reads it"
        self.read.setdefault(place, set()).add(wave)

    def writes(self, wave, place, what):
        others = self.read.get(place, set()) - {wave}
        assert not others, f"wave {wave} writes {place} in the epoch in which waves {others} read it"
        self.written.setdefault(place, set()).add(wave)
        self.content[place] = what

    def copies(self, wave, place, what):
        """(every wave has a part of every place: `place` is the whole's name, the parts are the waves')"""
        others = self.read.get(place, set()) - {wave}
        assert not others, f"wave {wave} copies to {place} in the epoch in which waves {others} read it"
        assert not any(p == place and w != what for p, w, _ in self.flying), f"{place} has a copy under way"
        self.flying.append((place, what, wave))

    def waits(self, wave, left):
        """All but the last `left` copies of the wave have landed."""
        mine = [f for f in self.flying if f[2] == wave]
        for f in mine[:len(mine) - left] if left else mine:
            self.flying.remove(f)
            if not any(p == f[0] and w == f[1] for p, w, _ in self.flying):  # (the last wave's part)
                self.content[f[0]] = f[1]


WAVES = range(8)


def rows_kernel(n_tiles, stages, at_a_time):
    """paged_prefix_kernel: a step's tiles are copied while those of the step before are multiplied."""
    m, steps = Memory(), -(-n_tiles // at_a_time)

    def issue(step):
        for i in range(at_a_time):
            for w in WAVES:
                m.copies(w, ("stage", (step * at_a_time + i) % stages), ("tile", step * at_a_time + i))

    for w in WAVES:
        m.writes(w, ("plan",), "plan")
    m.barrier()
    issue(0)  # (the plan lies where the second half of the ring is: places 2 and 3)
    assert {(i % stages) for i in range(at_a_time)}.isdisjoint({2, 3})
    for w in WAVES:
        m.reads(w, ("plan",), "plan")
    m.barrier()
    for w in WAVES:  # the queries change lanes there, each wave in its own part
        m.writes(w, ("queries", w), "queries")
        m.reads(w, ("queries", w), "queries")
    for step in range(steps):
        for w in WAVES:
            m.waits(w, 0)
        m.barrier()
        issue(step + 1)
        for w in WAVES:
            tile = step * at_a_time + w // (8 // at_a_time)
            m.reads(w, ("stage", tile % stages), ("tile", tile))
    for w in WAVES:
        m.waits(w, 0)
    assert not m.flying


def codes_kernel(n_tiles, slots, ahead, columns, unpacked=2):
    """paged_prefix_codes_kernel: raw tiles three ahead, unpacked ones one ahead; waves without columns unpack for the others."""
    m, busy = Memory(), -(-columns // 16)
    idle, done = 8 - busy, []

    def issue(tile):
        for w in WAVES:
            m.copies(w, ("raw", tile % slots), ("tile", tile))

    def unpack(tile, everyone=False):
        parts = []
        for w in WAVES:
            for part in [w] if everyone or idle == 0 else range(w - busy, 8, idle) if w >= busy else []:
                m.reads(w, ("raw", tile % slots), ("tile", tile))
                m.writes(w, ("stage", tile % unpacked, part), ("tile", tile))
                parts.append(part)
        assert sorted(parts) == list(range(8))

    for tile in range(ahead):
        issue(tile)
    for w in WAVES:
        m.waits(w, ahead - 1)
    m.barrier()
    unpack(0, everyone=True)
    for tile in range(n_tiles):
        for w in WAVES:
            m.waits(w, 1)
        m.barrier()
        issue(tile + ahead)
        if tile + 1 < n_tiles:
            unpack(tile + 1)
        for w in range(busy):
            for part in WAVES:
                m.reads(w, ("stage", tile % unpacked, part), ("tile", tile))
            m.reads(w, ("raw", tile % slots), ("tile", tile))  # scales and biases, where the copies put them
        done.append(tile)
    for w in WAVES:
        m.waits(w, 0)
    assert done == list(range(n_tiles)) and not m.flying


@pytest.mark.parametrize("n_tiles", [1, 2, 3, 4, 7, 8, 31])
def test_nothing_is_read_too_soon_or_written_too_late(n_tiles):
    rows_kernel(n_tiles, _constant("kStages"), _constant("kAtATime"))
    for columns in (1, 16, 17, 88, 112, 113, 128):
        codes_kernel(n_tiles, _constant("kRawSlots"), 3, columns)


def test_the_model_finds_mistakes():
    for stages in (2, 3):
        with pytest.raises(AssertionError):
            rows_kernel(9, stages, 2)
    with pytest.raises(AssertionError):
        codes_kernel(9, 3, 3, 88)
    with pytest.raises(AssertionError):
        codes_kernel(9, 4, 4, 88)
    with pytest.raises(AssertionError):
        codes_kernel(9, 4, 2, 88)  # (a wait that leaves one tile under way does not reach the one that is unpacked)
    with pytest.raises(AssertionError):
        codes_kernel(9, 4, 3, 88, unpacked=1)
