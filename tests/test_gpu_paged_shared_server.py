"""The operators over shared prefixes and over selected pages together, as a server runs them: requests that join a prefix, go on and
end through a layer, and a layer that selects its pages, eager and captured.

Tolerance of the histories: against float64 attention over the rows as the pages hold them, through the layer's own gate and
projection. The attention's result, the gate, their product and the projected result are each rounded to the type (eps / 2; the
gate's function eps): 2.5 eps of the sum of the projection's products' magnitudes, 4 with what the attention is off by itself in
16 bits (partial sums in float16 are off by half an eps of bfloat16 at most); in float32 that is the larger part, fewer than 2^-13
of the values' sum for some hundred keys.
"""

import numpy as np
import pytest
import torch

from moespresso_amd.runtime.qwen import paged
from oracle import paged as oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HEADS, KV_HEADS, HIDDEN = 4, 2, 96
FORMS = [(F32, True), (BF16, False), (F16, False), (BF16, True), (F32, False)]


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


def _cache(n_pages, dtype, quantized, **kwargs):
    return paged.PagedKVCache(n_pages, KV_HEADS, page_size=16, quantized=quantized,
                              dtype=BF16 if dtype == F32 and not quantized else dtype, **kwargs)


def _rows(cache, table, n):
    """Keys and values [n, Hkv, 256] of a table's first rows in float64."""
    def side(s):
        at = [(int(table[i // 16]), i % 16) for i in range(n)]
        p, o = (torch.tensor([a[j] for a in at], dtype=torch.long, device="cuda") for j in range(2))
        if torch.is_tensor(s):
            return s[p, :, o].double()
        codes, scale, bias = (t.view(torch.int32)[p, :, o].contiguous() if t.dtype == torch.uint32 else t[p, :, o] for t in s)
        return codes.view(torch.uint8).double() * scale.double().repeat_interleave(64, -1) + bias.double().repeat_interleave(64, -1)

    return side(cache.keys), side(cache.values)


def _attended(q, keys, values, scale):
    """One query [Hq, 256] over rows [n, Hkv, 256] in float64."""
    if keys.shape[0] == 0:
        return torch.zeros(HEADS, 256, dtype=torch.float64, device="cuda")
    k, v = (t.transpose(0, 1).repeat_interleave(HEADS // KV_HEADS, 0) for t in (keys, values))
    w = ((k * q.double()[:, None]).sum(-1) * scale).softmax(-1)
    return (w[:, :, None] * v).sum(1)


def _projected(inner, out, gate):
    """(result, sum of magnitudes) of the layer's gate and projection of float64 attention."""
    out = (out * torch.sigmoid(gate.double())).reshape(out.shape[0], -1)
    w = inner.o_proj.weight.double().t()
    return out @ w, (out.abs() @ w.abs()).max()


def _bound(dtype, quantized):
    return max(4 * torch.finfo(BF16 if not quantized and dtype == F32 else dtype).eps, 2.0 ** -13)


# places 0 to 4 are requests, 5 and 6 prefixes; in front of the step: which request continues which prefix from now on
STEPS = [({}, [0, 0, 0, 0, 0, 40, 0]),
         ({}, [3, 0, 0, 0, 0, 7, 16]),
         ({1: 0, 2: 0, 3: 1}, [1, 20, 1, 5, 0, 0, 0]),
         ({4: 0}, [1, 1, 1, 1, 1, 0, 0]),
         ({}, [1, 1, -1, 1, 30, 0, 0]),
         ({2: 1}, [1, 1, 2, -1, 1, 0, 0]),
         ({3: None}, [-1, 1, 1, 4, 1, 0, 0]),
         ({1: None, 4: None}, [0, -1, 1, 1, -1, -1, 0]),
         ({0: 0, 1: 1}, [0, 1, 1, 1, 0, 33, 0])]


@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("dtype,quantized", FORMS)
def test_a_server_whose_requests_continue_prefixes(dtype, quantized, axes):
    gen = torch.Generator(device="cuda").manual_seed(5)
    layer = paged.PagedAttention(_Block(1, dtype), _cache(30, dtype, quantized))
    tables = paged.PageTables(5, 30, page_size=16, max_tokens=105, n_prefixes=2)
    inner = layer.inner
    for joins, new in STEPS:
        for request, prefix in joins.items():
            tables.continue_prefix(request, prefix)
        rows = sum(max(n, 0) for n in new)
        x = torch.randn(rows + 3, HIDDEN, device="cuda", generator=gen).to(dtype)
        step = tables.step(_ints(new), rows + 3)
        groups, lens = tables.groups.tolist(), tables.lens.tolist()
        assert int(step.counts[1]) == 0
        requests, visible = step.requests.tolist(), step.visible.tolist()
        assert requests == [b for b, n in enumerate(new) for _ in range(max(n, 0))] + [-1] * 3
        front = [lens[5 + groups[b]] if groups[b] >= 0 else 0 for b in requests[:rows]]
        assert step.positions[:rows].tolist() == [f + v - 1 for f, v in zip(front, visible)]
        positions = None if axes == 1 else torch.stack([step.positions, step.positions // 3, step.positions % 3])
        got = layer(x, step, tables, positions)
        q, gate = inner.q_proj(x).reshape(rows + 3, HEADS, 512).chunk(2, dim=-1)
        k = inner.k_proj(x).reshape(rows + 3, KV_HEADS, 256)
        q, k = paged.qk_norm_rope(q, k, inner.q_norm.weight, inner.k_norm.weight, step.positions if axes == 1 else positions,
                                  inner.rope.inv_freq, sections=None if axes == 1 else inner.rope.sections)
        asked = q if quantized or dtype != F32 else q.to(BF16)
        out = torch.zeros(rows + 3, HEADS, 256, dtype=torch.float64, device="cuda")
        held = tables.tables.tolist()
        for r in range(rows):
            own, before = _rows(layer.cache, held[requests[r]], visible[r]), ()
            if front[r]:
                before = _rows(layer.cache, held[5 + groups[requests[r]]], front[r])
                own = [torch.cat(pair) for pair in zip(before, own)]
            out[r] = _attended(asked[r], *own, inner.scale)
        want, most = _projected(inner, out, gate)
        assert (got.double() - want).abs().max() <= _bound(dtype, quantized) * most
        assert (got[rows:] == 0).all()


@pytest.mark.parametrize("max_tokens,max_prefix", [(320, None), (150000, None), (150000, 301)])
@pytest.mark.parametrize("dtype,quantized", FORMS)
def test_a_prefix_once_is_a_history_of_every_request(dtype, quantized, max_tokens, max_prefix):
    """Twenty requests behind a prefix of 300 rows, and the same where every request holds those rows itself: the same keys, and
    results that are each off by no more than the bound (tables of few and of many pages: both forms of the kernels)."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    block, n = _Block(2, dtype), 20
    shared = paged.PagedAttention(block, _cache(19 + 6 * n, dtype, quantized))
    apart = paged.PagedAttention(block, _cache(26 * n, dtype, quantized))
    tables = paged.PageTables(n, 19 + 6 * n, page_size=16, max_tokens=max_tokens, n_prefixes=1, max_prefix_tokens=max_prefix)
    others = paged.PageTables(n, 26 * n, page_size=16, max_tokens=416)
    x = torch.randn(300, HIDDEN, device="cuda", generator=gen).to(dtype)
    shared(x, tables.step(_ints([0] * n + [300]), 300), tables)
    for b in range(n):
        tables.continue_prefix(b, 0)
        apart(x, others.step(_ints([300 if i == b else 0 for i in range(n)]), 300), others)
    for new in ([2 + b % 5 for b in range(n)], [1] * n, [70] + [0] * (n - 1), [1] * n, [0] * (n - 3) + [1, 1, 1]):
        rows = sum(new)
        x = torch.randn(rows, HIDDEN, device="cuda", generator=gen).to(dtype)
        a, b = tables.step(_ints(new + [0]), rows), others.step(_ints(new), rows)
        assert a.positions.equal(b.positions) and a.requests.equal(b.requests)
        got, want = shared(x, a, tables), apart(x, b, others)
        inner = block
        gate = inner.q_proj(x).reshape(rows, HEADS, 512).chunk(2, dim=-1)[1]
        # (the sum of magnitudes is at most that of values as large as the largest of the pages)
        _, most = _projected(inner, _rows(apart.cache, others.tables[n - 1].tolist(), 300)[1].abs().amax((0, 1)).expand(rows, HEADS, 256), gate)
        assert (got.double() - want.double()).abs().max() <= 2 * _bound(dtype, quantized) * most
    for r in (0, 7, n - 1):
        own = _rows(shared.cache, tables.tables[r].tolist(), int(tables.lens[r]))
        all_rows = _rows(apart.cache, others.tables[r].tolist(), int(others.lens[r]))
        assert all(s.equal(t[300:]) for s, t in zip(own, all_rows))


def test_rows_without_a_page_see_no_prefix_either():
    layer = paged.PagedAttention(_Block(2, BF16), _cache(3, BF16, False))
    tables = paged.PageTables(2, 3, page_size=16, max_tokens=64, n_prefixes=1)
    x = torch.randn(50, HIDDEN, device="cuda").to(BF16)
    layer(x[:20], tables.step(_ints([0, 0, 20]), 20), tables)
    tables.continue_prefix(0, 0)
    tables.continue_prefix(1, 0)
    step = tables.step(_ints([10, 30, 0]), 50)
    got = layer(x, step, tables)
    assert step.lens.tolist() == [10, 0, 20] and step.counts[1] == 30
    assert (got[10:] == 0).all() and got[:10].abs().amin() > 0 and not got.isnan().any()


@pytest.mark.parametrize("dtype,quantized", FORMS)
def test_a_layer_that_selects_its_pages(dtype, quantized):
    """Steps through the layer equal the selection, and the paged decode over its tables, made from the layer's parts bit for bit; a
    step over all pages equals a layer that does not select."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    block = _Block(3, dtype)
    layer = paged.PagedAttention(block, _cache(60, dtype, quantized, bounds=True), n_selected=5)
    plain = paged.PagedAttention(block, _cache(60, dtype, quantized))
    tables, others = (paged.PageTables(3, 60, page_size=16, max_tokens=480) for _ in range(2))
    for new, dense in (([200, 30, 0], True), ([1, 1, 90], False), ([1, 1, 1], False), ([1, 60, -1], False), ([1, 1, 1], True), ([1, 1, 0], False)):
        rows = sum(max(n, 0) for n in new)
        x = torch.randn(rows + 2, HIDDEN, device="cuda", generator=gen).to(dtype)
        step, other = tables.step(_ints(new), rows + 2), others.step(_ints(new), rows + 2)
        got, whole = layer(x, step, tables, dense=dense), plain(x, other, others)
        cache, inner = layer.cache, layer.inner
        for p, g in [(int(p), g) for p in tables.tables[0][:3] for g in range(KV_HEADS)]:
            low, high, e = oracle.bounds(_rows(cache, [p], 16)[0][:, g].cpu().numpy())
            assert cache.scales[p, g] == 2.0 ** e and (cache.codes[p, g].cpu().numpy() == [low, high]).all()
        if dense:
            assert got.equal(whole)
            continue
        q, gate = inner.q_proj(x).reshape(rows + 2, HEADS, 512).chunk(2, dim=-1)
        k = inner.k_proj(x).reshape(rows + 2, KV_HEADS, 256)
        q, _ = paged.qk_norm_rope(q, k, inner.q_norm.weight, inner.k_norm.weight, step.positions, inner.rope.inv_freq)
        asked = q if quantized or dtype != F32 else q.to(BF16)
        of, n = paged.select_pages(asked, cache.codes, cache.scales, tables.tables, step.visible, 5, page_size=16, requests=step.requests)
        want_of, want_n = oracle.select_pages(asked.double().cpu().numpy(), cache.codes.cpu().numpy(), cache.scales.cpu().numpy(),
                                              tables.tables.cpu().numpy(), step.visible.cpu().numpy(), 16, 5, 1, 2, step.requests.cpu().numpy())
        assert (of.cpu().numpy() == want_of).all() and (n.cpu().numpy() == want_n).all()

        def heads(side):
            return side.reshape(60 * KV_HEADS, 1, 16, -1) if torch.is_tensor(side) else [t.reshape(60 * KV_HEADS, 1, 16, -1) for t in side]

        per_head = asked.reshape(-1, HEADS // KV_HEADS, 256), heads(cache.keys), heads(cache.values), of.reshape(-1, 5), n.reshape(-1)
        if quantized:
            a, k_, v_, t, m = per_head
            out = paged.sdpa_decode_paged_q8(a, *k_, *v_, t, m, inner.scale)
        else:
            out = paged.sdpa_decode_paged(*per_head, inner.scale)
        out = out.reshape(rows + 2, HEADS, 256).to(q.dtype)
        assert got.equal(inner.o_proj((out * torch.sigmoid(gate)).reshape(rows + 2, -1)))
        few = step.visible <= 5 * 16  # (requests of no more pages than are taken attend them all)
        want, most = _projected(inner, out.double(), gate)
        assert few.any() and (got[few].double() - whole[few].double()).abs().max() <= 2 * _bound(dtype, quantized) * most


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("selects", [False, True])
def test_a_captured_step_follows_prefixes_and_bounds(quantized, selects):
    """One graph of a step and two layers, replayed with other rows and prefixes, equals eager steps bit for bit; between the replays
    runs eager work of its own."""
    blocks = [_Block(3, BF16), _Block(4, BF16)]
    kwargs = dict(n_selected=4, recent=1) if selects else {}
    places = 7 if not selects else 5

    def server():
        return (paged.PageTables(5, 60, page_size=16, max_tokens=256, **({} if selects else dict(n_prefixes=2, max_prefix_tokens=40))),
                [paged.PagedAttention(b, _cache(60, BF16, quantized, bounds=selects), **kwargs) for b in blocks])

    gen = torch.Generator(device="cuda").manual_seed(9)
    new, x = torch.zeros(places, dtype=torch.int32, device="cuda"), torch.zeros(140, HIDDEN, device="cuda", dtype=BF16)

    def one(tables, layers, new, x):
        step = tables.step(new, 140)
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
    steps = (({}, [100, 3, 0, 9, 1, 20, 3]), ({1: 0, 2: 1}, [1, 1, 1, 1, 1, 0, 0]), ({4: 1}, [1, -1, 20, 1, 1, 0, 0]), ({1: 1}, [1, 8, 1, -1, 1, 0, 0]),
             ({0: None}, [-1, 1, 1, 1, 60, 0, 0]), ({2: None}, [4, 4, -1, 4, 4, -1, 0]), ({}, [1, 1, 1, 1, 1, 17, 0]))
    for joins, asked in steps:
        if not selects:
            for request, prefix in joins.items():
                for tables in (graph_server[0], eager_server[0]):
                    tables.continue_prefix(request, prefix)
        new.copy_(_ints(asked[:places]))
        x.copy_(torch.randn(140, HIDDEN, device="cuda", generator=gen).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        step, want = one(*eager_server, new, x)
        torch.cuda.synchronize()
        assert all(a.equal(b) for a, b in zip(out_step, step)) and out.equal(want)
        assert graph_server[0].tables.equal(eager_server[0].tables) and graph_server[0].lens.equal(eager_server[0].lens)
        if selects:
            for a, b in zip(graph_server[1], eager_server[1]):
                assert a.cache.codes.equal(b.cache.codes) and a.cache.scales.equal(b.cache.scales)


@pytest.mark.parametrize("selects", [False, True])
def test_a_step_of_more_rows_than_a_call_takes(selects):
    """2100 rows of a prompt behind a prefix, and of a prompt whose pages are selected: the rows of both calls against the operators
    called for each by itself."""
    layer = paged.PagedAttention(_Block(5, BF16), _cache(160, BF16, False, bounds=selects), **(dict(n_selected=9) if selects else {}))
    tables = paged.PageTables(1, 160, page_size=16, max_tokens=2304, n_prefixes=0 if selects else 1)
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(2100, HIDDEN, device="cuda", generator=gen).to(BF16)
    if not selects:
        layer(x[:50], tables.step(_ints([0, 50]), 50), tables)
        tables.continue_prefix(0, 0)
    step = tables.step(_ints([2100] if selects else [2100, 0]), 2100)
    got = layer(x, step, tables)
    q, gate = layer.inner.q_proj(x).reshape(2100, HEADS, 512).chunk(2, dim=-1)
    k = layer.inner.k_proj(x).reshape(2100, KV_HEADS, 256)
    q, _ = paged.qk_norm_rope(q, k, layer.inner.q_norm.weight, layer.inner.k_norm.weight, step.positions, layer.inner.rope.inv_freq)
    parts = []
    for at in (slice(0, 2048), slice(2048, 2100)):
        args = (tables.tables, step.visible[at], layer.inner.scale)
        if selects:
            parts.append(paged.sdpa_decode_paged_sparse(q[at], layer.cache.keys, layer.cache.values, layer.cache.codes, layer.cache.scales,
                                                        *args, 9, requests=step.requests[at]))
        else:
            parts.append(paged.sdpa_decode_paged_shared(q[at], layer.cache.keys, layer.cache.values, *tables.prefixes, *args,
                                                        requests=step.requests[at]))
    assert got.equal(layer.inner.o_proj((torch.cat(parts) * torch.sigmoid(gate)).reshape(2100, -1)))


def _calls(gen, quantized=False):
    """Calls of every operator, small and large: (function of a workspace, floats of it that are enough)."""
    n_kv, rep, page, pool = 2, 8, 64, 160
    if quantized:
        def side():
            scales = 0.02 * torch.rand(pool, n_kv, page, 4, device="cuda", generator=gen)
            return (torch.randint(-2 ** 31, 2 ** 31 - 1, (pool, n_kv, page, 64), device="cuda", generator=gen, dtype=torch.int32).view(torch.uint32),
                    scales.to(BF16), (-128 * scales).to(BF16))
        keys, values = side(), side()
        pages = (*keys, *values)
        shared, sparse = paged.sdpa_decode_paged_shared_q8, paged.sdpa_decode_paged_sparse_q8
    else:
        keys, values = (torch.randn(pool, n_kv, page, 256, device="cuda", generator=gen).to(BF16) for _ in range(2))
        pages = (keys, values)
        shared, sparse = paged.sdpa_decode_paged_shared, paged.sdpa_decode_paged_sparse
    codes, scales = torch.zeros(pool, n_kv, 2, 256, dtype=torch.int8, device="cuda"), torch.ones(pool, n_kv, device="cuda")
    paged.page_bounds(torch.arange(pool * page, dtype=torch.int32, device="cuda"), keys, codes, scales)

    def ints(high, *shape):
        return torch.randint(0, high, shape, device="cuda", generator=gen, dtype=torch.int32)

    calls = []
    for R in (2, 37):
        q = torch.randn(R, n_kv * rep, 256, device="cuda", generator=gen).to(BF16)
        own = ints(pool, R, 30), ints(1900, R)
        prefixes = ints(pool, 3, 40 if R == 2 else 300), ints(2500, 3), ints(4, R)  # (one launch, and prefixes by themselves)
        calls += [lambda ws, a=(q, *pages, *prefixes, *own, 0.0625): (shared(*a, workspace=ws),),
                  lambda ws, a=(q, *pages, codes, scales, *own, 0.0625, 6): (sparse(*a, workspace=ws),),
                  lambda ws, a=(q, codes, scales, *own, 6): paged.select_pages(*a, page_size=page, workspace=ws)]
    return calls


@pytest.mark.parametrize("quantized", [False, True])
def test_captured_graphs_share_a_workspace(quantized):
    """One after the other, of different operators and sizes, over memory that holds what the last one left (at first: not a number)."""
    calls, graphs = _calls(torch.Generator(device="cuda").manual_seed(12), quantized), []
    ws = torch.full((1 << 24,), float("nan"), device="cuda")
    for call in calls:
        want = call(None)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(ws)
        graphs.append((graph, out, want))
    for _ in range(3):
        for graph, out, want in graphs:
            for o in out:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(o.equal(w) for o, w in zip(out, want))


def test_calls_of_several_operators_on_streams_of_their_own():
    calls = _calls(torch.Generator(device="cuda").manual_seed(13))
    wants = [call(None) for call in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[] for _ in calls]
    for _ in range(10):
        for call, stream, outs in zip(calls, streams, got):
            with torch.cuda.stream(stream):
                outs.append(call(None))
    torch.cuda.synchronize()
    for want, outs in zip(wants, got):
        assert all(o.equal(w) for out in outs for o, w in zip(out, want))


def test_a_workspace_that_is_too_small_is_refused():
    for call in _calls(torch.Generator(device="cuda").manual_seed(14)):
        with pytest.raises((RuntimeError, ValueError), match="workspace"):
            call(torch.empty(4, device="cuda"))


@pytest.mark.parametrize("quantized", [False, True])
def test_calls_and_steps_without_rows(quantized):
    cache = _cache(8, BF16, quantized, bounds=True)
    sides = (*cache.keys, *cache.values) if quantized else (cache.keys, cache.values)
    shared, sparse = ((paged.sdpa_decode_paged_shared_q8, paged.sdpa_decode_paged_sparse_q8) if quantized else
                      (paged.sdpa_decode_paged_shared, paged.sdpa_decode_paged_sparse))
    q, none, t = torch.empty(0, HEADS, 256, device="cuda", dtype=BF16), _ints([]), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    two, bounds = _ints([0, 0]), (cache.codes, cache.scales)
    assert shared(q, *sides, t, two, two, t, none, 0.1, requests=none).shape == q.shape
    assert sparse(q, *sides, *bounds, t, none, 0.1, 4, requests=none).shape == q.shape
    of, n = paged.select_pages(q, *bounds, t, none, 4, page_size=16, requests=none)
    assert of.shape == (0, KV_HEADS, 4) and n.shape == (0, KV_HEADS)
    before = cache.codes.clone()
    paged.page_bounds(none, cache.keys, *bounds)
    assert cache.codes.equal(before)
    block, x = _Block(8, BF16), torch.empty(0, HIDDEN, device="cuda", dtype=BF16)
    for tables, kwargs in ((paged.PageTables(2, 8, page_size=16, max_tokens=48, n_prefixes=1), {}),
                           (paged.PageTables(2, 8, page_size=16, max_tokens=48), dict(n_selected=4))):
        layer = paged.PagedAttention(block, cache, **kwargs)
        step = tables.step(_ints([0] * (2 + tables.n_prefixes)), 0)
        assert layer(x, step, tables).shape == (0, HIDDEN)
