"""What a layer over a paged cache does around its operators (CPU: the operators themselves are stood in for)."""

import pytest
import torch

from moespresso_amd.runtime.qwen import paged

HEADS, KV_HEADS, HIDDEN = 4, 2, 32


class _Norm(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.weight, self.eps = torch.nn.Parameter(1 + 0.1 * torch.randn(256)), 1e-6


class _Rope(torch.nn.Module):
    inv_freq, sections = torch.ones(32), (11, 11, 10)


class _Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.q_proj, self.k_proj = torch.nn.Linear(HIDDEN, HEADS * 512), torch.nn.Linear(HIDDEN, KV_HEADS * 256)
        self.v_proj, self.o_proj = torch.nn.Linear(HIDDEN, KV_HEADS * 256), torch.nn.Linear(HEADS * 256, HIDDEN)
        self.q_norm, self.k_norm, self.rope = _Norm(), _Norm(), _Rope()
        self.scale, self.num_attention_heads, self.num_key_value_heads = 256 ** -0.5, HEADS, KV_HEADS


def _layer(monkeypatch):
    layer = paged.PagedAttention(_Block(), paged.PagedKVCache(4, KV_HEADS, page_size=16, device="cpu", dtype=torch.float16))
    # (what the kernels return is in no graph)
    monkeypatch.setattr(layer.cache, "append", lambda q, k, v, *rest, **kw: q.detach().contiguous())
    monkeypatch.setattr(layer.cache, "attend", lambda q, *rest, **kw: torch.tanh(q.detach()))
    n = torch.zeros(5, dtype=torch.int32)
    step = paged.PageStep(n, n, n, n, n, n, n, n)
    return layer, step, paged.PageTables(2, 4, page_size=16, max_tokens=32, device="cpu")


def test_a_backward_pass_is_refused(monkeypatch):
    """Not cut off in silence: the gate and the projection alone would leave gradients that lack the attention's part."""
    layer, step, tables = _layer(monkeypatch)
    x = torch.randn(5, HIDDEN)
    with torch.no_grad():
        want = layer(x, step, tables)
    assert not want.requires_grad
    with torch.inference_mode():
        assert layer(x, step, tables).equal(want)
    out = layer(x, step, tables)
    assert out.detach().equal(want)
    with pytest.raises(RuntimeError, match="no backward pass"):
        out.sum().backward()
    assert layer.inner.q_proj.weight.grad is None
    # frozen weights, and a gradient asked for of what goes in
    layer.requires_grad_(False)
    assert not layer(x, step, tables).requires_grad
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        (x + layer(x, step, tables)).sum().backward()
    # what lies behind the attention may still learn
    layer.inner.o_proj.requires_grad_(True)
    x.requires_grad_(False)
    layer(x, step, tables).sum().backward()
    assert layer.inner.o_proj.weight.grad.abs().sum() > 0
