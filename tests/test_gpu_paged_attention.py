"""The operators of a paged cache together, as a server runs them: steps of prompts, single tokens, ended and padded rows
through a layer, against attention over each request's own history, and captured steps replayed against eager ones.

Tolerance of the histories: against float64 attention over the rows as the pages hold them, through the layer's own gate and
projection. The attention's result, the gate, their product and the projected result are each rounded to the type (eps / 2;
the gate's function eps): 2.5 eps of the sum of the projection's products' magnitudes, 4 with what the attention is off by
itself in 16 bits; in float32 that is the larger part, fewer than 2^-13 of the values' sum for some hundred keys.
"""

import numpy as np
import pytest
import torch

from moespresso_amd.runtime.qwen import paged
from oracle import paged as oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HEADS, KV_HEADS, HIDDEN = 4, 2, 96


class _Norm(torch.nn.Module):
    def __init__(self, gen, dtype):
        super().__init__()
        self.weight = torch.nn.Parameter((1 + 0.2 * torch.randn(256, device="cuda", generator=gen)).to(dtype), requires_grad=False)
        self.eps = 1e-6


class _Rope(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.inv_freq = (1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float().cuda()
        self.sections = (11, 11, 10)


class _Block(torch.nn.Module):
    """The modules of a full-attention block that the layer takes."""

    def __init__(self, seed, dtype):
        super().__init__()
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def linear(n, m):
            layer = torch.nn.Linear(n, m, bias=False, device="cuda", dtype=dtype)
            layer.weight = torch.nn.Parameter((torch.randn(m, n, device="cuda", generator=gen) * n ** -0.5).to(dtype), requires_grad=False)
            return layer

        self.q_proj, self.k_proj = linear(HIDDEN, HEADS * 512), linear(HIDDEN, KV_HEADS * 256)
        self.v_proj, self.o_proj = linear(HIDDEN, KV_HEADS * 256), linear(HEADS * 256, HIDDEN)
        self.q_norm, self.k_norm, self.rope = _Norm(gen, dtype), _Norm(gen, dtype), _Rope()
        self.scale, self.num_attention_heads, self.num_key_value_heads = 256 ** -0.5, HEADS, KV_HEADS


def _ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _stored(cache):
    def side(s):
        if torch.is_tensor(s):
            return s.double()
        codes, scale, bias = s
        return codes.view(torch.uint8).double() * scale.double().repeat_interleave(64, -1) + bias.double().repeat_interleave(64, -1)

    return (side(s).cpu().numpy() for s in (cache.keys, cache.values))


STEPS = [[40, 17, 0, 5], [1, 1, 33, 1], [1, -1, 1, 1], [1, 64, 1, -1], [0, 1, 1, 20], [1, 1, -1, 1], [1, 1, 1, 1]]


@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("dtype,quantized", [(F32, True), (BF16, False), (F16, False), (BF16, True), (F32, False)])
def test_a_server_of_four_requests(dtype, quantized, axes):
    gen = torch.Generator(device="cuda").manual_seed(5)
    layer = paged.PagedAttention(_Block(1, dtype), paged.PagedKVCache(14, KV_HEADS, page_size=16, quantized=quantized,
                                                                      dtype=BF16 if dtype == F32 and not quantized else dtype))
    tables = paged.PageTables(4, 14, page_size=16, max_tokens=128)
    inner, rope = layer.inner, layer.inner.rope
    for new in STEPS:
        rows = sum(max(n, 0) for n in new)
        x = torch.randn(rows + 3, HIDDEN, device="cuda", generator=gen).to(dtype)  # (a padded batch)
        step = tables.step(_ints(new), rows + 3)
        assert int(step.counts[1]) == 0
        positions = None if axes == 1 else torch.stack([step.positions, step.positions // 3, step.positions % 3])
        got = layer(x, step, tables, positions)
        # the same through the separate calls and the pages as they are now
        q, gate = inner.q_proj(x).reshape(rows + 3, HEADS, 512).chunk(2, dim=-1)
        k = inner.k_proj(x).reshape(rows + 3, KV_HEADS, 256)
        q, k = paged.qk_norm_rope(q, k, inner.q_norm.weight, inner.k_norm.weight, step.positions if axes == 1 else positions,
                                  rope.inv_freq, sections=None if axes == 1 else rope.sections)
        keys, values = _stored(layer.cache)
        for r in range(rows):
            slot = int(step.slots[r])
            stored = torch.from_numpy(keys[slot // 16, :, slot % 16]).cuda()
            if not quantized:
                assert stored.equal(k[r].to(layer.cache.keys.dtype).double())
        asked = q if quantized or dtype != F32 else q.to(BF16)
        want = oracle.paged_attention(asked.double().cpu().numpy(), keys, values, tables.tables.cpu().numpy(), step.visible.cpu().numpy(),
                                      inner.scale, step.requests.cpu().numpy())
        assert (want[rows:] == 0).all()
        out = torch.from_numpy(want).cuda() * torch.sigmoid(gate.double())
        want = out.reshape(rows + 3, -1) @ inner.o_proj.weight.double().t()
        bound = 4 * torch.finfo(BF16 if not quantized and dtype == F32 else dtype).eps
        bound = max(bound, 2.0 ** -13)
        assert (got.double() - want).abs().max() <= bound * (out.reshape(rows + 3, -1).abs() @ inner.o_proj.weight.double().abs().t()).max()


def test_rows_without_a_page_are_left_out_of_the_layer():
    """A pool that runs out: the rows that found no page see nothing and change nothing."""
    layer = paged.PagedAttention(_Block(2, BF16), paged.PagedKVCache(3, KV_HEADS, page_size=16))
    tables = paged.PageTables(2, 3, page_size=16, max_tokens=64)
    x = torch.randn(70, HIDDEN, device="cuda").to(BF16)
    step = tables.step(_ints([40, 30]), 70)
    got = layer(x, step, tables)
    assert step.lens.tolist() == [40, 0] and step.counts.tolist() == [70, 30, 3, 0]
    assert (got[40:] == 0).all() and got[:40].abs().sum() > 0 and not got.isnan().any()
    alone = paged.PagedAttention(layer.inner, paged.PagedKVCache(3, KV_HEADS, page_size=16))
    other = paged.PageTables(2, 3, page_size=16, max_tokens=64)
    want = alone(x, other.step(_ints([40, 0]), 70), other)
    assert got[:40].equal(want[:40]) and layer.cache.keys.equal(alone.cache.keys) and layer.cache.values.equal(alone.cache.values)


@pytest.mark.parametrize("quantized", [False, True])
def test_a_captured_step_follows_the_lengths(quantized):
    """One graph of a step and two layers, replayed with other rows and lengths, equals eager steps bit for bit; between the
    replays runs eager work of its own."""
    blocks = [_Block(3, BF16), _Block(4, BF16)]

    def server():
        return (paged.PageTables(5, 40, page_size=16, max_tokens=256),
                [paged.PagedAttention(b, paged.PagedKVCache(40, KV_HEADS, page_size=16, quantized=quantized)) for b in blocks])

    gen = torch.Generator(device="cuda").manual_seed(9)
    new, x = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(24, HIDDEN, device="cuda", dtype=BF16)

    def one(tables, layers, new, x):
        step = tables.step(new, 24)
        for layer in layers:
            x = x + layer(x, step, tables)
        return step, x

    graph_server, eager_server = server(), server()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # (allocations and handles of a first run, on a server that is thrown away)
        one(*server(), new, x)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out_step, out = one(*graph_server, new, x)
    for asked in ([5, 3, 0, 9, 1], [1, 1, 1, 1, 1], [1, -1, 20, 1, 1], [1, 8, 1, -1, 1], [-1, 1, 1, 1, 1], [4, 4, 4, 4, 4], [1, 1, 1, 1, 1]):
        new.copy_(_ints(asked))
        x.copy_(torch.randn(24, HIDDEN, device="cuda", generator=gen).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        step, want = one(*eager_server, new, x)
        torch.cuda.synchronize()
        assert all(a.equal(b) for a, b in zip(out_step, step)) and out.equal(want)
        assert graph_server[0].tables.equal(eager_server[0].tables) and graph_server[0].lens.equal(eager_server[0].lens)


def test_two_captured_graphs_share_a_workspace():
    gen = torch.Generator(device="cuda").manual_seed(10)
    keys, values = (torch.randn(60, 2, 64, 256, device="cuda", generator=gen).to(BF16) for _ in range(2))
    ws = torch.full((1 << 23,), float("nan"), device="cuda")
    calls = []
    for B, n in ((3, 1200), (20, 150)):
        q = torch.randn(B, 16, 256, device="cuda", generator=gen).to(BF16)
        tables = torch.randint(0, 60, (B, 20), device="cuda", generator=gen, dtype=torch.int32)
        lens = torch.randint(0, n, (B,), device="cuda", generator=gen, dtype=torch.int32)
        args = (q, keys, values, tables, lens, 0.0625)
        want = paged.sdpa_decode_paged(*args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged.sdpa_decode_paged(*args, workspace=ws)
        calls.append((graph, out, want, args))  # (a graph keeps no tensor alive)
    for _ in range(4):
        for graph, out, want, _ in calls:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert out.equal(want)


def test_calls_on_two_streams_at_once():
    gen = torch.Generator(device="cuda").manual_seed(11)
    keys, values = (torch.randn(300, 2, 64, 256, device="cuda", generator=gen).to(BF16) for _ in range(2))
    jobs = []
    for B in (1, 7):
        q = torch.randn(B, 16, 256, device="cuda", generator=gen).to(BF16)
        tables = torch.randint(0, 300, (B, 130), device="cuda", generator=gen, dtype=torch.int32)
        lens = torch.randint(4000, 8300, (B,), device="cuda", generator=gen, dtype=torch.int32)
        args = (q, keys, values, tables, lens, 0.0625)
        jobs.append((torch.cuda.Stream(), args, paged.sdpa_decode_paged(*args)))
    torch.cuda.synchronize()
    got = [[] for _ in jobs]
    for _ in range(10):
        for (stream, args, _), outs in zip(jobs, got):
            with torch.cuda.stream(stream):
                outs.append(paged.sdpa_decode_paged(*args))
    torch.cuda.synchronize()
    for (_, _, want), outs in zip(jobs, got):
        assert all(o.equal(want) for o in outs)
