"""Registers and scratch of the kernels of a paged cache (CPU: hipcc compiles the sources to assembly, nothing runs).

The decode kernel keeps a tile of keys, one of values and all results of sixteen heads in registers, with two tiles on their way:
a value put away to scratch and fetched again would wait for all of them, in every tile.
"""
import os
import re
import shutil

import pytest

from moespresso_amd import build

pytestmark = pytest.mark.skipif(not (os.path.exists(build.HIPCC) or shutil.which(build.HIPCC)), reason="hipcc not installed")


def _kernels(source, name):
    return {k: v for k, v in build.kernel_resources(os.path.join(build.CSRC, source)).items() if name in k}


def test_the_decode_kernels_use_no_scratch_and_fit_their_registers():
    kernels = _kernels("paged_decode.hip", "paged_decode_kernel")
    # 16-bit rows of two types; 8-bit rows: three types of queries, three of scales; shares of workgroups and of waves
    assert len(kernels) == 2 * (2 + 9), sorted(kernels)
    for name, res in kernels.items():
        query, form = re.search(r"paged_decode_kernelILi(\d)ELi(\d)E", name).groups()
        assert res["scratch_bytes"] == 0 and res["vgpr_spills"] == 0, (name, res)
        # a wave a SIMD has 512 registers; 8-bit rows and 16-bit queries are held to the 256 that need no accumulation registers
        assert res["vgprs"] <= (256 if form == "3" and query != "0" else 512), (name, res)


@pytest.mark.parametrize("source,name,count", [("paged_decode.hip", "paged_merge", 6), ("page_step.hip", "page_step_kernel", 4),
                                               ("qk_norm_rope.hip", "qk_norm_rope_kernel", 10)])
def test_the_other_kernels_of_a_paged_cache_use_no_scratch(source, name, count):
    kernels = _kernels(source, name)
    assert len(kernels) == count, sorted(kernels)
    for k, res in kernels.items():
        assert res["scratch_bytes"] == 0 and res["vgpr_spills"] == 0 and res["sgpr_spills"] == 0, (k, res)
