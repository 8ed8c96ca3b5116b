"""Steps of a layer over a paged cache that a server makes beside the ordinary ones."""

import pytest
import torch

from moespresso_amd.runtime.qwen import paged
from test_gpu_paged_attention import BF16, F16, F32, HEADS, HIDDEN, KV_HEADS, _Block, _ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,quantized", [(BF16, False), (F16, True), (F32, True), (F32, False)])
def test_a_step_without_rows(dtype, quantized):
    """Every request ends and nothing is padded; the layer goes on from there."""
    layer = paged.PagedAttention(_Block(1, dtype), paged.PagedKVCache(6, KV_HEADS, page_size=16, quantized=quantized,
                                                                      dtype=BF16 if dtype == F32 and not quantized else dtype))
    tables = paged.PageTables(3, 6, page_size=16, max_tokens=64)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(24, HIDDEN, device="cuda", generator=gen).to(dtype)
    want = layer(x, tables.step(_ints([20, 3, 1]), 24), tables)
    kept = [t.clone() for side in (layer.cache.keys, layer.cache.values) for t in (side if quantized else (side,))]
    step = tables.step(_ints([-1, -1, -1]), 0)
    out = layer(x[:0], step, tables)
    assert out.shape == (0, HIDDEN) and out.dtype == dtype and step.counts.tolist() == [0, 0, 0, 4]
    assert tables.lens.tolist() == [0, 0, 0] and int(tables.head) == 0
    for side, t in zip([t for side in (layer.cache.keys, layer.cache.values) for t in (side if quantized else (side,))], kept):
        assert side.view(torch.uint8).equal(t.view(torch.uint8))
    assert layer(x, tables.step(_ints([20, 3, 1]), 24), tables).equal(want)
