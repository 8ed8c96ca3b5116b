"""A prompt whose pages are selected from a table of the most pages there may be: its rows go in several calls, and each is what the
operator gives for its rows."""

import numpy as np
import pytest
import torch

from moespresso_amd.runtime.qwen import paged
from test_gpu_paged_shared_server import BF16, HEADS, HIDDEN, KV_HEADS, _Block, _cache, _ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quantized", [False, True])
def test_a_prompt_behind_a_table_of_32768_pages(quantized):
    layer = paged.PagedAttention(_Block(6, BF16), _cache(60, BF16, quantized, bounds=True), n_selected=9)
    tables = paged.PageTables(1, 60, page_size=16, max_tokens=16 * 32768)
    gen = torch.Generator(device="cuda").manual_seed(15)
    x = torch.randn(700, HIDDEN, device="cuda", generator=gen).to(BF16)
    step = tables.step(_ints([700]), 700)
    calls, attend = [], layer.cache.attend
    layer.cache.attend = lambda q, *a, **k: calls.append(len(q)) or attend(q, *a, **k)
    got = layer(x, step, tables)
    assert len(calls) > 1 and sum(calls) == 700 and max(calls) * 4 * HEADS * 32768 <= 256 << 20
    q, gate = layer.inner.q_proj(x).reshape(700, HEADS, 512).chunk(2, dim=-1)
    k = layer.inner.k_proj(x).reshape(700, KV_HEADS, 256)
    q, _ = paged.qk_norm_rope(q, k, layer.inner.q_norm.weight, layer.inner.k_norm.weight, step.positions, layer.inner.rope.inv_freq)
    keys, values = layer.cache.keys, layer.cache.values
    sides = (*keys, *values) if quantized else (keys, values)
    sparse = paged.sdpa_decode_paged_sparse_q8 if quantized else paged.sdpa_decode_paged_sparse
    parts, at = [], 0
    for n in calls:
        parts.append(sparse(q[at:at + n], *sides, layer.cache.codes, layer.cache.scales, tables.tables, step.visible[at:at + n],
                            layer.inner.scale, 9, requests=step.requests[at:at + n]))
        at += n
    assert got.equal(layer.inner.o_proj((torch.cat(parts) * torch.sigmoid(gate)).reshape(700, -1)))
    # the pages of a row do not depend on the call that it is in
    whole = paged.select_pages(q, layer.cache.codes, layer.cache.scales, tables.tables, step.visible, 9, page_size=16, requests=step.requests)
    few = paged.select_pages(q[690:], layer.cache.codes, layer.cache.scales, tables.tables, step.visible[690:], 9, page_size=16,
                             requests=step.requests[690:])
    assert all(np.array_equal(a[690:].cpu(), b.cpu()) for a, b in zip(whole, few))
