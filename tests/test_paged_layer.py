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


class _CalledNorm(_Norm):
    centre, power = 0.0, 0.5

    def forward(self, x):
        y = x.float()
        y = y * (y.square().mean(-1, keepdim=True) + self.eps) ** -self.power
        return (y * (self.centre + self.weight.float())).to(x.dtype)


class _CalledRope(_Rope):
    pairs, stretch = "halves", 1.0

    def __init__(self, rotary=64):
        super().__init__()
        self.inv_freq = (1e7 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float()

    def forward(self, x, offset=0):
        half = self.inv_freq.numel()
        angle = (offset + torch.arange(x.shape[-2]))[:, None] * self.inv_freq * self.stretch
        y = x.float().clone()
        i = torch.arange(half)
        first, second = (i, i + half) if self.pairs == "halves" else (2 * i, 2 * i + 1)
        a, b = y[..., first].clone(), y[..., second].clone()
        y[..., first], y[..., second] = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
        return y.to(x.dtype)


def _with(**modules):
    block = _Block()
    for name, module in modules.items():
        setattr(block, name, module)
    return paged.PagedAttention(block, paged.PagedKVCache(4, KV_HEADS, page_size=16, device="cpu", dtype=torch.float16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rotary", [16, 64, 256])
def test_modules_that_compute_what_the_operators_do_are_taken(dtype, rotary):
    _with(q_norm=_CalledNorm().to(dtype), k_norm=_CalledNorm().to(dtype), rope=_CalledRope(rotary))


@pytest.mark.parametrize("name", ["q_norm", "k_norm"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norms_that_compute_something_else_are_refused(name, dtype):
    """Else the layer would give wrong rows without a word."""
    from_one = _CalledNorm().to(dtype)
    from_one.centre = 1.0
    fresh = _CalledNorm().to(dtype)
    fresh.centre = 1.0
    torch.nn.init.zeros_(fresh.weight)
    other_eps = _CalledNorm().to(dtype)
    other_eps.forward = lambda x: (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-5) * other_eps.weight).to(x.dtype)
    no_root = _CalledNorm().to(dtype)
    no_root.power = 1.0
    for norm in (from_one, fresh, other_eps, no_root):
        with pytest.raises(ValueError, match=f"{name} is not weight"):
            _with(**{name: norm})
    narrow = _Norm()
    narrow.weight = torch.nn.Parameter(torch.ones(128))
    with pytest.raises(ValueError, match="256 channels"):
        _with(**{name: narrow})


def test_ropes_that_compute_something_else_are_refused():
    turned, stretched = _CalledRope(), _CalledRope()
    turned.pairs, stretched.stretch = "neighbours", 0.25
    for rope in (turned, stretched):
        with pytest.raises(ValueError, match="rope does not rotate"):
            _with(rope=rope)


def test_hooks_that_would_not_run_are_refused(monkeypatch):
    layer, step, tables = _layer(monkeypatch)
    x = torch.randn(5, HIDDEN)
    for module in (layer.inner.q_norm, layer.inner.k_norm, layer.inner.rope):
        for register in (module.register_forward_hook, module.register_forward_pre_hook):
            hook = register(lambda *a: None)
            with pytest.raises(RuntimeError, match="would not run"):
                layer(x, step, tables)
            hook.remove()
    layer(x, step, tables)


def test_modules_that_give_something_of_another_kind_are_not_compared():
    """A rope that makes cosines and sines, or takes positions: the layer needs its frequencies only."""
    class Tables(_Rope):
        def forward(self, x, offset=0):
            return torch.cos(self.inv_freq), torch.sin(self.inv_freq)

    class Positions(_Rope):
        def forward(self, x, position_ids):
            raise AssertionError("not called")

    class Residual(_Norm):
        def forward(self, x, **kwargs):
            return x, None

    _with(rope=Tables(), q_norm=Residual())
    _with(rope=Positions())


def test_tables_of_another_pool_are_refused(monkeypatch):
    """Slots of another page size are other rows, and pages beyond the pool would be left out without a word."""
    layer, step, tables = _layer(monkeypatch)
    x = torch.randn(5, HIDDEN)
    for n_pages, page_size in ((4, 32), (2, 64), (5, 16)):
        with pytest.raises(ValueError, match="than the cache has"):
            layer(x, step, paged.PageTables(2, n_pages, page_size=page_size, max_tokens=64, device="cpu"))
    layer(x, step, paged.PageTables(2, 3, page_size=16, max_tokens=64, device="cpu"))
