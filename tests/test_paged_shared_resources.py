"""Registers, scratch, LDS and inline assembly of the kernels over shared prefixes and selected pages (CPU: hipcc compiles the
sources to assembly, nothing runs)."""
import os
import re
import shutil

import pytest

from moespresso_amd import build

pytestmark = pytest.mark.skipif(not (os.path.exists(build.HIPCC) or shutil.which(build.HIPCC)), reason="hipcc not installed")
SHARED = os.path.join(build.CSRC, "paged_shared.hip")


def _kernels(source, name):
    return {k: v for k, v in build.kernel_resources(os.path.join(build.CSRC, source)).items() if name in k}


def _loops(lines, multiplies):
    """The loops over tiles: the instructions from a label to the branch back to it, so many matrix instructions among them, that hold
    no other such."""
    code, labels, spans = [], {}, []
    for line in (l.split(";")[0].strip() for l in lines):
        if m := re.match(r"(\.?\w+):$", line):
            labels[m[1]] = len(code)
        elif line and not line.startswith("."):
            code.append(line)
            m = re.match(r"s_c?branch\w* (\.?\w+)$", line)
            if m and m[1] in labels:
                spans.append((labels[m[1]], len(code)))
    spans = [(a, b) for a, b in spans if sum("v_mfma" in l for l in code[a:b]) >= multiplies]
    inner = [s for s in spans if not any(t != s and s[0] <= t[0] and t[1] <= s[1] for t in spans)]
    return [code[a:b] for a, b in inner]


def test_the_tile_loops_of_the_prefix_kernels_use_no_scratch():
    """Registers that are put away (a few, where a wave has 256) are fetched again outside the loop over the tiles of keys."""
    bodies = build.kernel_bodies(build.device_assembly(SHARED))
    for kind, count in (("paged_prefix_kernel", 2), ("paged_prefix_codes_kernel", 9), ("paged_shared_kernel", 11)):
        kernels = {k: v for k, v in bodies.items() if kind in k}
        assert len(kernels) == count, sorted(kernels)
        for name, lines in kernels.items():
            tiles = _loops(lines, 48)
            assert tiles, name
            for loop in tiles:
                assert not [l for l in loop if l.startswith("scratch_")], name
    planted = [".L1:", "v_mfma_f32_16x16x32_f16 a, b, c", "scratch_load_dword v1, off, s0", "s_cbranch_scc1 .L1"]
    assert [l for loop in _loops(planted, 1) for l in loop if l.startswith("scratch_")]


def test_registers_put_away_by_the_kernels_are_few():
    for name, res in _kernels("paged_shared.hip", "paged_").items():
        most = 96 if "prefix_kernelILi1" in name else 32
        assert res["scratch_bytes"] <= most and res["vgpr_spills"] <= most // 4, (name, res)
        assert res["vgprs"] <= (256 if "prefix" in name else 512), (name, res)
        if "merge" in name or "codes" in name or "ILi1ELi1ELi1E" in name or "ILi2ELi2ELi2E" in name:
            assert res["scratch_bytes"] == 0, (name, res)


@pytest.mark.parametrize("source,name,count", [("page_bounds.hip", "page_bounds_kernel", 5), ("page_select.hip", "page_score_kernel", 6),
                                               ("page_select.hip", "page_choose_kernel", 8)])
def test_the_kernels_of_the_selection_use_no_scratch(source, name, count):
    kernels = _kernels(source, name)
    assert len(kernels) == count, sorted(kernels)
    for k, res in kernels.items():
        # (a thread of the choice from 32768 pages holds 32 worths at two waves a SIMD less, and puts one word away)
        most = 8 if "ILi1024ELi32E" in k else 0
        assert res["scratch_bytes"] <= most, (k, res)


def test_the_ring_of_the_prefix_kernels_is_aligned():
    """Places within it are addressed by exclusive or: its base, which all extern arrays of one name share, must be a multiple of 256."""
    text = build.device_assembly(SHARED)
    fixed = {}
    for record in re.split(r"\n  - \.", text[text.index("amdhsa.kernels:"):])[1:]:
        name, size = re.search(r"\.name:\s+(\S+)", record), re.search(r"\.group_segment_fixed_size:\s+(\d+)", record)
        if name and "paged_prefix" in name[1]:
            fixed[name[1]] = int(size[1])
    assert len(fixed) == 11 and all(n % 256 == 0 for n in fixed.values()), fixed


@pytest.mark.parametrize("source", ["paged_shared.hip", "paged_decode.hip", "page_bounds.hip", "page_select.hip"])
def test_inline_assembly_of_the_kernels(source):
    """No load into a register, no copy into LDS right behind the write of its address register, no scalar register read too soon."""
    bodies = build.kernel_bodies(build.device_assembly(os.path.join(build.CSRC, source)))
    assert bodies
    if source == "paged_shared.hip":
        assert sum("_load_lds_" in l for lines in bodies.values() for l in lines) > 0
    for name, lines in bodies.items():
        assert build.inline_asm_register_loads(lines) == [], name
        assert build.m0_hazards(lines) == [], name
        assert build.scalar_register_hazards(lines) == [], name
