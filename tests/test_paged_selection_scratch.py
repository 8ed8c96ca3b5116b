"""Scratch of a layer that selects its pages: a word for every query head and page of a table, whatever lengths are (CPU)."""

import pytest
import torch

from moespresso_amd import _lib
from moespresso_amd.runtime.qwen import paged

I32 = torch.int32


class _Norm(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.weight, self.eps = torch.nn.Parameter(torch.ones(256), requires_grad=False), 1e-6


class _Rope(torch.nn.Module):
    inv_freq = torch.ones(32)


class _Block(torch.nn.Module):
    def __init__(self, heads, kv_heads):
        super().__init__()
        self.q_proj, self.k_proj = torch.nn.Linear(2, heads * 512), torch.nn.Linear(2, kv_heads * 256)
        self.v_proj, self.o_proj = torch.nn.Linear(2, kv_heads * 256), torch.nn.Linear(heads * 256, 2)
        self.q_norm, self.k_norm, self.rope = _Norm(), _Norm(), _Rope()
        self.scale, self.num_attention_heads, self.num_key_value_heads = 0.0625, heads, kv_heads


def _layer(heads, kv_heads, n_selected=64):
    cache = paged.PagedKVCache(4, kv_heads, page_size=16, device="cpu", dtype=torch.float16, bounds=True)
    return paged.PagedAttention(_Block(heads, kv_heads), cache, n_selected=n_selected)


def _tables(width):
    return paged.PageTables(1, 4, page_size=16, max_tokens=16 * width, device="cpu")


def _calls(monkeypatch, layer, tables, rows):
    """Queries of every call of a step of so many rows."""
    asked = []
    monkeypatch.setattr(layer.cache, "append", lambda q, *a, **k: q)
    monkeypatch.setattr(layer.cache, "attend", lambda q, *a, **k: asked.append(len(q)) or q)
    n = torch.zeros(rows, dtype=I32)
    with torch.no_grad():
        layer(torch.zeros(rows, 2), paged.PageStep(n, n, n, n, n, n, n, n), tables)
    return asked


@pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")
@pytest.mark.parametrize("heads,kv_heads,width,n_selected", [(16, 2, 8192, 64), (16, 2, 32768, 64), (64, 8, 32768, 4096), (4, 4, 32767, 5), (16, 2, 512, 64)])
def test_the_calls_of_a_step_have_scratch_within_reach(monkeypatch, heads, kv_heads, width, n_selected):
    """2048 rows of a prompt; the attention over the selected pages has scratch of its own, which does not grow with the queries."""
    calls = _calls(monkeypatch, _layer(heads, kv_heads, n_selected), _tables(width), 2048)
    assert sum(calls) == 2048 and len(set(calls[:-1])) <= 1 and calls[-1] <= calls[0]
    lib = _lib.lib()

    def scratch(queries):
        return (lib.mspr_sdpa_decode_paged_sparse_workspace_bytes(queries, heads, kv_heads, 16, width, n_selected)
                - lib.mspr_sdpa_decode_paged_workspace_bytes(queries * kv_heads, heads // kv_heads, 1, 16, n_selected))

    assert scratch(calls[0]) <= (256 << 20) + 3 * 256 + 4 * calls[0] * kv_heads  # (three parts on whole 256 bytes, and lengths)
    if len(calls) > 1:  # (and no more calls than that takes)
        assert scratch(calls[0]) >= 128 << 20


def test_steps_over_short_tables_stay_one_call(monkeypatch):
    assert _calls(monkeypatch, _layer(16, 2), _tables(512), 2048) == [2048]
    assert _calls(monkeypatch, _layer(16, 2), _tables(32768), 64) == [64]
