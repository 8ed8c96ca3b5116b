"""GPU parity of decode attention behind shared prefixes with float64 attention over the rows as stored (bound: paged_reference.py).

Every test runs twice: with prefixes' tables as they are, and with so many entries behind them that prefixes are a kernel's own (of more
than 32 query heads a KV head; which form a call takes goes by these and by the rows that the tables hold)."""

import numpy as np
import pytest
import torch

import paged_reference as ref
from paged_reference import BF16, F16, F32, i32
from moespresso_amd.runtime.qwen import paged

pytestmark = pytest.mark.gpu

SCALE = 256 ** -0.5
FORMS = [(F16, "rows"), (BF16, "rows"), (F32, F32), (F32, BF16), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (BF16, F16), (F32, F16),
         (F16, BF16)]
FEW = [(BF16, "rows"), (F16, "rows"), (F32, F32), (BF16, BF16)]


@pytest.fixture(params=["tables", "long_tables"], autouse=True)
def long_tables(request):
    global LONG
    LONG = request.param == "long_tables"
    return LONG


def _wide(prefix_tables, columns, page, codes):
    return columns > 1024 or columns > 32 and columns * np.shape(prefix_tables)[1] * page >= (4 << 20 if codes else 5 << 19)


def _tables_of(prefix_tables, columns, page):
    """The tables, or with so many entries that name no page behind them that the form of many columns takes them."""
    prefix_tables = np.asarray(prefix_tables)
    if LONG and columns > 32:
        width = -(-(4 << 20) // (columns * page))
        prefix_tables = np.pad(prefix_tables, ((0, 0), (0, max(0, width - prefix_tables.shape[1]))), constant_values=-1)
        assert _wide(prefix_tables, columns, page, True)
    return prefix_tables


def _shape_of(q, keys):
    """Query heads of all queries and one KV head, and the page size."""
    shape = (keys if torch.is_tensor(keys) else keys[0]).shape
    return q.shape[0] * (q.shape[1] // shape[1]), shape[2]


def _call(q, keys, values, prefix_tables, prefix_lens, groups, tables, lens, scale=SCALE, requests=None, **kw):
    prefix_tables = _tables_of(prefix_tables, *_shape_of(q, keys))
    rest = (i32(prefix_tables), i32(prefix_lens), i32(groups), i32(tables), i32(lens), scale)
    kw["requests"] = None if requests is None else i32(requests)
    if torch.is_tensor(keys):
        return paged.sdpa_decode_paged_shared(q, keys, values, *rest, **kw)
    return paged.sdpa_decode_paged_shared_q8(q, *keys, *values, *rest, **kw)


def _places(prefix_tables, prefix_lens, groups, tables, lens, requests, R, page, n_pages, G):
    out = []
    for r in range(R):
        b = r if requests is None else int(requests[r])
        at = []
        if 0 <= b < len(tables):
            if 0 <= groups[b] < len(prefix_tables):
                at += ref.places(prefix_tables[groups[b]], prefix_lens[groups[b]], page, n_pages)
            at += ref.places(tables[b], lens[r], page, n_pages)
        out.append([at] * G)
    return out


def _half_parts(q, keys, prefix_tables):
    """Where prefixes are a kernel's own, bfloat16 rows leave partial sums of eleven digits."""
    columns, page = _shape_of(q, keys)
    return torch.is_tensor(keys) and q.dtype == BF16 and _wide(_tables_of(prefix_tables, columns, page), columns, page, False)


def _check(q, keys, values, prefix_tables, prefix_lens, groups, tables, lens, scale=SCALE, requests=None):
    n_pages, G, page = (keys if torch.is_tensor(keys) else keys[0]).shape[:3]
    got = _call(q, keys, values, prefix_tables, prefix_lens, groups, tables, lens, scale, requests)
    at = _places(prefix_tables, prefix_lens, groups, tables, lens, requests, q.shape[0], page, n_pages, G)
    ref.check(got, q, keys, values, at, scale, _half_parts(q, keys, prefix_tables))
    return got


def _case(seed, heads, n_kv, page, prefix_lens, groups, lens, dtype, form):
    rng = np.random.default_rng(seed)
    n_pages = sum(-(-n // page) for n in [*prefix_lens, *lens]) + 2
    keys, values = ref.cache(rng, (n_pages, n_kv, page, 256), dtype, form)
    order = list(rng.permutation(n_pages))
    prefix_tables = ref.tables(rng, prefix_lens, page, -(-max(prefix_lens) // page) + 1, n_pages, order)
    tables = ref.tables(rng, lens, page, -(-max(lens) // page) + 1, n_pages, order)
    return ref.rows(rng, (len(lens), heads, 256), dtype) * 2, keys, values, prefix_tables, prefix_lens, groups, tables, lens


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("heads,n_kv,page,prefix_lens,groups,lens", [
    (16, 2, 16, [1], [0], [1]),
    (16, 2, 64, [137], [0, 0], [40, 3]),
    (16, 2, 64, [0, 31, 64, 200], [0, 1, 2, 3, 3, 3, 3, 3, -1, 4, 1, 2], [0, 1, 2, 15, 16, 17, 31, 0, 33, 63, 0, 65]),
    (1, 1, 32, [127, 128], [0, 1, 0, -7, 1] * 9, [127, 128, 129, 0, 160] * 9),
    (16, 1, 16, [300, 7], [0, 0, 1, 0, 0], [300, 1099, 5, 0, 1]),
    (15, 3, 128, [777], [0, 0, 0, 0, 0, 0, 0], [777, 1024, 64, 0, 1, 128, 129]),
    (8, 8, 256, [500], [0, -1], [500, 1]),
])
def test_lengths_heads_and_groups(heads, n_kv, page, prefix_lens, groups, lens, dtype, form):
    got = _check(*_case(heads * 100 + page, heads, n_kv, page, prefix_lens, groups, lens, dtype, form))
    for b, n in enumerate(lens):
        if n == 0 and not (0 <= groups[b] < len(prefix_lens) and prefix_lens[groups[b]]):
            assert (got[b] == 0).all()


@pytest.mark.parametrize("dtype,form", FEW)
def test_long_and_ragged_batches(dtype, form):
    rng = np.random.default_rng(8)
    for prefix_lens, n, most, n_kv, page in (([37000], 5, 300, 2, 64), ([9001, 300, 4000], 40, 900, 2, 16), ([700, 40], 200, 60, 1, 16),
                                             ([4000] * 9, 9, 1, 4, 256)):
        lens = [int(x) for x in rng.integers(0, most, n)]
        groups = [int(g) for g in rng.integers(-1, len(prefix_lens), n)]
        _check(*_case(n, 8 * n_kv, n_kv, page, prefix_lens, groups, lens, dtype, form))


def test_a_call_without_prefixes_is_the_plain_one_and_one_of_prefixes_alone_too():
    """Whole rows either way: the same sums up to the order of float32 additions, within the bound."""
    q, keys, values, prefix_tables, prefix_lens, groups, tables, lens = _case(3, 16, 2, 16, [100], [-1] * 5, [60, 1, 0, 700, 16], BF16, "rows")
    _check(q, keys, values, prefix_tables, prefix_lens, groups, tables, lens)
    _check(q, keys, values, prefix_tables, prefix_lens, [0] * 5, tables, [0] * 5)


@pytest.mark.parametrize("dtype,form", FEW)
def test_rows_that_do_not_count_may_hold_anything(dtype, form):
    """NaN and infinities behind the last row of a prefix and of a request, and in pages that no table names."""
    rng = np.random.default_rng(2)
    page, n_pages = 64, 9
    keys, values = ref.cache(rng, (n_pages, 2, page, 256), dtype, form)
    prefix_tables, prefix_lens, groups, tables, lens = [[1, 2]], [80], [0, 0, -1, 0], [[3], [4], [5], [6]], [1, 16, 40, 0]
    q = ref.rows(np.random.default_rng(1), (4, 16, 256), dtype)
    args = prefix_tables, prefix_lens, groups, tables, lens
    want = _call(q, keys, values, *args)
    held = {1: 64, 2: 16, 3: 1, 4: 16, 5: 40, 6: 0}
    for side in (keys, values):
        for t in (side,) if torch.is_tensor(side) else side[1:]:
            for bad, where in ((float("nan"), 0), (float("inf"), 1), (float("-inf"), 2)):
                t[0], t[7:] = bad, bad
                for p, n in held.items():
                    t[p, :, n + where::3] = bad
    assert _check(q, keys, values, *args).equal(want)


@pytest.mark.parametrize("dtype,form", [(BF16, "rows"), (F32, F32)])
def test_pages_that_are_not_in_the_pool_are_left_out(dtype, form):
    rng = np.random.default_rng(3)
    page, n_pages = 16, 30
    keys, values = ref.cache(rng, (n_pages, 2, page, 256), dtype, form)
    for t in (keys, values) if form == "rows" else keys[1:] + values[1:]:
        t[0] = float("nan")  # where a page that is not there would be read instead
    prefix_tables, tables = rng.integers(1, n_pages, (2, 13)), rng.integers(1, n_pages, (5, 6))
    prefix_tables[0, 3], prefix_tables[0, 12], prefix_tables[1] = -1, n_pages, 2 ** 31 - 1
    tables[0, 0], tables[1, 2], tables[4] = -2 ** 31, n_pages, -1
    got = _check(ref.rows(rng, (5, 16, 256), dtype), keys, values, prefix_tables, [200, 208], [0, 0, 1, 1, 1], tables, [50, 90, 33, 96, 96])
    assert (got[4] == 0).all()


def test_lengths_beyond_the_tables_and_below_zero():
    rng = np.random.default_rng(4)
    keys, values = ref.cache(rng, (13, 2, 16, 256), BF16, "rows")
    tables = np.arange(8).reshape(4, 2)
    got = _check(ref.rows(rng, (4, 16, 256), BF16), keys, values, [[8, 9], [10, 11]], [2 ** 31 - 1, -5], [0, 1, 1, 0], tables,
                 [32, 2 ** 31 - 1, -1, -2 ** 31])
    assert (got[2] == 0).all()


@pytest.mark.parametrize("dtype,form", [(F16, "rows"), (BF16, BF16)])
def test_queries_that_share_a_request(dtype, form):
    """Drafted rows, each with what it sees; queries of requests that no table has see nothing, prefixes neither."""
    rng = np.random.default_rng(6)
    keys, values = ref.cache(rng, (60, 2, 16, 256), dtype, form)
    order = rng.permutation(56)
    requests, lens = [2, 2, 2, 0, -1, 1, 3, 2 ** 31 - 1, 2], [100, 101, 102, 7, 50, 192, 50, 50, 103]
    got = _check(ref.rows(rng, (9, 16, 256), dtype), keys, values, order[36:].reshape(2, 10), [150, 9], [1, -1, 0], order[:36].reshape(3, 12),
                 lens, requests=requests)
    assert (got[4] == 0).all() and (got[6:8] == 0).all()


@pytest.mark.parametrize("R,n_prefixes", [(2048, 1), (2048, 2048), (257, 2000), (1300, 3)])
def test_as_many_queries_and_prefixes_as_a_call_takes(R, n_prefixes):
    rng = np.random.default_rng(R + n_prefixes)
    keys, values = ref.cache(rng, (40, 2, 16, 256), BF16, "rows")
    prefix_tables, prefix_lens = rng.integers(0, 40, (n_prefixes, 5)), rng.integers(0, 81, n_prefixes)
    groups, tables = rng.integers(-1, n_prefixes + 1, 9), rng.integers(0, 40, (9, 7))
    requests, lens = rng.integers(-1, 10, R), rng.integers(0, 113, R)
    q = ref.rows(rng, (R, 4, 256), BF16)
    got = _call(q, keys, values, prefix_tables, prefix_lens, groups, tables, lens, requests=requests)
    some = sorted({0, R - 1, *(int(i) for i in rng.choice(R, 40, replace=False))})
    at = _places(prefix_tables, prefix_lens, groups, tables, lens[some], requests[some], len(some), 16, 40, 2)
    ref.check(got[some], q[some], keys, values, at, SCALE, _half_parts(q, keys, prefix_tables))
    assert not got.isnan().any()


def test_sharp_and_flat_weights():
    """One key of a prefix far above all others, and keys whose weights are 2^-20 of its: none may be lost."""
    rng = np.random.default_rng(7)
    n, page = 40000, 64
    for dtype in (F16, BF16):
        keys, values = (torch.zeros(n // page + 2, 1, page, 256, dtype=dtype, device="cuda") for _ in range(2))
        table = rng.permutation(n // page + 1)[None, :n // page]
        values[:, 0, :, 0], values[:, 0, :, 1] = 1, -0.5
        hot = int(table[0, 300])
        keys[hot, 0, 11, 0], values[hot, 0, 11] = 1, 0
        q = torch.zeros(3, 4, 256, dtype=dtype, device="cuda")
        q[:, :, 0] = torch.tensor([0.0, 13.8629, 30.0, 80.0])
        _check(q, keys, values, table, [n], [0, 0, 0], [[n // page + 1]] * 3, [0, 1, 5], scale=1.0)


@pytest.mark.parametrize("dtype,form", [(F32, F32), (F32, BF16), (F16, F16), (BF16, BF16)])
def test_every_weight_keeps_its_digits(dtype, form):
    """Small queries over few keys: a weight of which a term is off by a step of its type shows."""
    rng = np.random.default_rng(17)
    lens = [int(n) for n in rng.integers(1, 12, 120)]
    prefix_lens = [int(n) for n in rng.integers(1, 12, 30)]
    q, *rest = _case(17, 16, 1, 16, prefix_lens, [int(g) for g in rng.integers(0, 30, 120)], lens, dtype, form)
    _check(q * 2.0 ** -10, *rest)


def test_large_queries_and_scales_of_very_different_size():
    rng = np.random.default_rng(9)
    keys, values = ref.codes(rng, (6, 1, 32, 256), F32, spread=1e-7), ref.codes(rng, (6, 1, 32, 256), F32, spread=1e-6)
    for part in values[1:]:
        part[2, 0, 5] *= 1e4
    q = ref.rows(rng, (3, 4, 256), F32) * torch.tensor([1e6, 1.0, 1e-6, 0.0], device="cuda")[None, :, None]
    args = keys, values, [[0, 1, 2, 3]], [120], [0, 0, 0], [[4], [5], [5]], [20, 32, 0]
    _check(q, *args)
    _check(q.bfloat16(), *args)


def test_values_of_any_size():
    """Beyond float16's range and below it, a prefix's and own rows' of very different size."""
    q, keys, values, prefix_tables, *rest = _case(22, 16, 2, 16, [300, 40], [0] * 9 + [1] * 5, [50, 1, 0, 70, 16, 17, 3] * 2, BF16, "rows")
    for of_prefixes, of_others in ((1e30, 1e30), (1e-30, 1e-30), (1e30, 1e-6), (1e-30, 1.0), (0.0, 1.0), (1.0, 0.0)):
        v = values * of_others
        for p in prefix_tables[0][:19].tolist() + prefix_tables[1][:3].tolist():
            v[p] = values[p] * of_prefixes
        _check(q, keys, v, prefix_tables, *rest)


def test_a_negative_scale_and_one_of_zero():
    case = _case(21, 16, 2, 16, [90], [0] * 6, [40, 1, 0, 70, 16, 17], BF16, "rows")
    for scale in (-0.05, 0.0):
        _check(*case, scale=scale)


def test_the_same_call_gives_the_same_bits():
    """Whatever the workspace held before, in eager calls and in replays of a captured one."""
    rng = np.random.default_rng(11)
    lens = [int(n) for n in rng.integers(0, 900, 20)]
    q, keys, values, *rest = _case(12, 16, 2, 16, [5000, 77], [int(g) for g in rng.integers(-1, 2, 20)], lens, BF16, "rows")
    want = _call(q, keys, values, *rest)
    ws = torch.full((1 << 24,), float("nan"), device="cuda")
    assert all(_call(q, keys, values, *rest, workspace=ws).equal(want) for _ in range(4))
    lens_dev = i32(rest[4])
    args = (i32(_tables_of(rest[0], 160, 16)), i32(rest[1]), i32(rest[2]), i32(rest[3]), lens_dev, SCALE)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.sdpa_decode_paged_shared(q, keys, values, *args)
    for i in range(4):
        lens_dev.copy_(i32([max(0, n - 37 * i) for n in lens]))
        graph.replay()
        torch.cuda.synchronize()
        assert out.equal(paged.sdpa_decode_paged_shared(q, keys, values, *args))


def test_operands_outside_the_plain_case_give_the_same_results():
    q, keys, values, *rest = _case(13, 16, 2, 16, [70], [0, -1, 0], [40, 48, 7], F16, "rows")
    want = _call(q, keys, values, *rest)
    assert _call(q.transpose(0, 1).contiguous().transpose(0, 1), keys, values, *rest, scale=np.float64(SCALE)).equal(want)
    assert _call(torch.cat([q[:, :, :4], q], dim=2)[:, :, 4:], keys, values, *rest).equal(want)
    with pytest.raises(ValueError, match="workspace"):
        _call(q, keys, values, *rest, workspace=torch.empty(8, device="cuda"))
    p, n, g, t, l = rest
    assert _call(q[:0], keys, values, p, n, g[:0], t[:0], []).shape == (0, 16, 256)


def test_pages_beyond_4_gb():
    """Row offsets of 33 bits: the last pages of a pool of 5 GB a side."""
    rng = np.random.default_rng(13)
    n_pages, page = 20000, 256
    keys, values = (torch.empty(n_pages, 2, page, 256, dtype=BF16, device="cuda") for _ in range(2))
    tables, prefix = np.array([[n_pages - 1, 2], [n_pages - 2, n_pages - 4]] * 3), np.array([[n_pages - 3, 5, n_pages - 5]])
    for p in [*tables.reshape(-1), *prefix.reshape(-1)]:
        keys[p], values[p] = ref.rows(rng, (2, page, 256), BF16), ref.rows(rng, (2, page, 256), BF16)
    _check(ref.rows(rng, (6, 16, 256), BF16), keys, values, prefix, [700], [0] * 6, tables, [300, 512, 0, 1, 257, 256])


def test_two_streams_at_once():
    cases = [_case(s, 16, 2, 64, [3000], [0] * 8, [100 * s + i for i in range(8)], BF16, "rows") for s in (1, 2)]
    ints = [(i32(_tables_of(c[3], 64, 64)), *(i32(a) for a in c[4:])) for c in cases]
    want = [paged.sdpa_decode_paged_shared(*c[:3], *i, SCALE) for c, i in zip(cases, ints)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(6):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(paged.sdpa_decode_paged_shared(*cases[k][:3], *ints[k], SCALE))
    torch.cuda.synchronize()
    assert all(g.equal(want[k]) for k in (0, 1) for g in got[k])


@pytest.mark.parametrize("dtype,form", FEW)
def test_what_is_no_number_stays_with_its_query(dtype, form):
    """A query, a prefix's row and a request's own row that hold NaN or infinities: the results of all others keep their bits."""
    q, keys, values, prefix_tables, prefix_lens, groups, tables, lens = _case(31, 16, 2, 16, [300, 50, 40], [0] * 7 + [1] * 7 + [2, -1, 2], [40, 1, 0, 17, 70] * 3 + [9, 5], dtype, form)
    args = prefix_tables, prefix_lens, groups, tables, lens
    want = _call(q, keys, values, *args)
    odd = q.clone()
    odd[3], odd[8, ::2], odd[9, :, 5] = float("nan"), float("inf"), float("-inf")
    got = _call(odd, keys, values, *args)
    others = [r for r in range(len(lens)) if r not in (3, 8, 9)]
    assert got[others].equal(want[others]) and got[8, 1::2].equal(want[8, 1::2]) and got[3].isnan().all()
    for side in (keys, values):
        for t in (side,) if torch.is_tensor(side) else side[1:]:
            t[int(prefix_tables[2][1]), :, 3], t[int(tables[15][0]), :, 2] = float("nan"), float("inf")
    got = _call(q, keys, values, *args)
    others = [r for r in range(len(lens)) if r not in (14, 15, 16)]
    assert got[others].equal(want[others]) and not got[14].isfinite().any() and not got[16].isfinite().any()
