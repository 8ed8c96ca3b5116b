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


@pytest.mark.parametrize("requests,rows,max_tokens,quantized", [(2048, 33, 64, False), (2048, 33, 64, True), (600, 40, 1 << 20, False)])
def test_a_step_of_more_rows_than_one_decode_call_takes(requests, rows, max_tokens, quantized):
    """67584 rows, and 24000 over tables of 2^20 tokens: the limits are a decode call's, not a layer's.

    Both sides round the attention's result, the gate (its function twice that), their product and the projected result to
    bfloat16 and differ in the order of sums: 2 * 2.5 eps of the projection's products' magnitudes.
    """
    T = requests * rows
    layer = paged.PagedAttention(_Block(3, BF16), paged.PagedKVCache(requests * 3, KV_HEADS, page_size=16, quantized=quantized))
    tables = paged.PageTables(requests, requests * 3, page_size=16, max_tokens=max_tokens)
    x = torch.randn(T + 5, HIDDEN, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(BF16)
    step = tables.step(_ints([rows] * requests), T + 5)
    got = layer(x, step, tables)
    assert (got[T:] == 0).all() and tables.lens.tolist() == [rows] * requests
    inner = layer.inner
    q, gate = inner.q_proj(x).reshape(T + 5, HEADS, 512).chunk(2, dim=-1)
    k = inner.k_proj(x).reshape(T + 5, KV_HEADS, 256)
    q, _ = paged.qk_norm_rope(q, k, inner.q_norm.weight, inner.k_norm.weight, step.positions, inner.rope.inv_freq)
    for at in (slice(0, 5000), slice(T - 5000, T), slice(65000, 66000)):
        if at.start >= T:
            continue
        out = layer.cache.attend(q[at], tables.tables, step.visible[at], inner.scale, requests=step.requests[at])
        out = (out * torch.sigmoid(gate[at])).reshape(-1, HEADS * 256)
        size = out.double().abs() @ inner.o_proj.weight.double().abs().t()
        assert ((got[at].double() - out.double() @ inner.o_proj.weight.double().t()).abs() <= 5 * torch.finfo(BF16).eps * size).all()


def test_a_layer_refuses_what_its_attention_would_refuse_later():
    """Before any row is written."""
    for change in (dict(num_attention_heads=5), dict(num_attention_heads=34), dict(num_key_value_heads=1)):
        block = _Block(4, BF16)
        for name, value in change.items():
            setattr(block, name, value)
        with pytest.raises(ValueError, match="heads"):
            paged.PagedAttention(block, paged.PagedKVCache(6, KV_HEADS, page_size=16))
