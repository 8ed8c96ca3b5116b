"""Bounds of pages and the selection from them (whole numbers: equal to the oracle), and attention over the selected pages."""

import numpy as np
import pytest
import torch

import paged_reference as ref
from paged_reference import BF16, F16, F32, i32
from moespresso_amd.runtime.qwen import paged
from oracle import paged as oracle

pytestmark = pytest.mark.gpu

SCALE = 256 ** -0.5


def _empty(n_pages, n_kv, fill=0):
    return (torch.full((n_pages, n_kv, 2, 256), fill, dtype=torch.int8, device="cuda"),
            torch.full((n_pages, n_kv), float(fill), dtype=F32, device="cuda"))


def _values(keys):
    """Rows [n_pages, Hkv, page, 256] in float64."""
    if torch.is_tensor(keys):
        return keys.double().cpu().numpy()
    codes, scales, biases = keys
    s, z = (t.double().repeat_interleave(64, -1) for t in (scales, biases))
    return (codes.view(torch.uint8).double() * s + z).cpu().numpy()


def _slots(table, page, first, last):
    return [int(table[i // page]) * page + i % page for i in range(first, last)]


def _check_bounds(keys, codes, scales, held):
    """``held``: rows that every page of the pool holds."""
    values, codes, scales = _values(keys), codes.cpu().numpy(), scales.cpu().numpy()
    for p, n in held.items():
        for g in range(values.shape[1]):
            low, high, e = oracle.bounds(values[p, g, :n])
            assert scales[p, g] == 2.0 ** e and (codes[p, g, 0] == low).all() and (codes[p, g, 1] == high).all(), (p, g, n)


FORMS = [(F16, "rows"), (BF16, "rows"), (F32, F32), (F16, F16), (BF16, BF16)]


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("n_kv,page,steps", [
    (2, 16, [[1, 0, 5], [1, 1, 1], [1, 16, 40], [15, 0, 1], [1, 1, 1]]),
    (1, 64, [[63, 64, 65], [1, 1, 1], [200, 0, 1]]),
    (3, 256, [[256, 1, 255], [1, 255, 1], [700, 2, 300]]),
    (2, 128, [[1500, 900, 0], [1, 1, 700]]),
])
def test_bounds_of_steps_are_those_of_all_rows(n_kv, page, steps, dtype, form):
    rng = np.random.default_rng(page + n_kv)
    width = -(-max(sum(s[b] for s in steps) for b in range(3)) // page)
    n_pages = 3 * width + 1
    keys, _ = ref.cache(rng, (n_pages, n_kv, page, 256), dtype, form)
    if form == "rows":  # pages of different sizes, and one whose rows grow
        keys.mul_(torch.tensor(2.0 ** rng.integers(-9, 9, n_pages), device="cuda", dtype=dtype)[:, None, None, None])
    table = rng.permutation(n_pages)[:3 * width].reshape(3, width)
    codes, scales = _empty(n_pages, n_kv, 77)
    lens = [0, 0, 0]
    for step in steps:
        slots = []
        for b, k in enumerate(step):
            slots += _slots(table[b], page, lens[b], lens[b] + k)
            lens[b] += k
        slots += [-1] * 5 + [n_pages * page, 2 ** 31 - 1]
        untouched = [p for p in range(n_pages) if p not in {s // page for s in slots}]
        before = codes.clone(), scales.clone()
        for _ in range(2):  # (again: nothing changes)
            paged.page_bounds(i32(slots), keys, codes, scales)
            held = {int(table[b][i]): min(page, lens[b] - i * page) for b in range(3) for i in range(-(-lens[b] // page))}
            _check_bounds(keys, codes, scales, held)
        assert codes[untouched].equal(before[0][untouched]) and scales[untouched].equal(before[1][untouched])


def test_bounds_of_rows_that_grow_and_edges_of_the_codes():
    """Every new row may need a larger step than the old codes have; 127 steps exactly, one more, zero, the ends of the range."""
    page = 16
    keys = torch.zeros(8, 1, page, 256, dtype=BF16, device="cuda")
    for i in range(page):
        keys[0, 0, i] = torch.linspace(-1, 1, 256, device="cuda").to(BF16) * 1.7 ** i
        keys[1, 0, i, 7] = 127 * 2.0 ** (i - 8)
        keys[2, 0, i, 9] = -127.5 * 2.0 ** (8 - i)
        keys[3, 0, i, 11] = (-1) ** i * 64 * 2.0 ** i
    keys[4, 0, :, 3] = 1e30
    keys[5, 0, :, 3], keys[5, 0, :, 4] = 1e-30, -1e-38
    keys[6] = 0
    codes, scales = _empty(8, 1)
    for i in range(page):
        slots = [p * page + i for p in range(7)]
        paged.page_bounds(i32(slots), keys, codes, scales)
        _check_bounds(keys, codes, scales, {p: i + 1 for p in range(7)})


def test_bounds_of_rows_that_are_not_numbers_stay_in_range():
    keys = torch.randn(3, 2, 32, 256, device="cuda").to(F16)
    keys[0, 0, 3, 5], keys[0, 0, 4, 6], keys[0, 0, :, 7], keys[0, 1, 2, 8] = float("nan"), float("inf"), float("nan"), float("-inf")
    codes, scales = _empty(3, 2)
    paged.page_bounds(i32(range(32)), keys, codes, scales)
    c, s = codes[0].long(), scales[0]
    assert (c[0, :, 7] == 0).all() and (c.abs() <= 127).all() and (s == 2.0 ** 50).all() and (c[0, 0] <= c[0, 1]).all()


def test_many_rows_a_workgroup():
    """Steps long enough that a workgroup looks after several rows, with requests of all lengths in them."""
    rng = np.random.default_rng(5)
    page, n_kv, new = 32, 2, [int(n) for n in rng.integers(1, 90, 80)] + [1] * 300
    held = [-(-n // page) for n in new]
    order = list(rng.permutation(sum(held) + 1))
    keys = ref.rows(rng, (len(order), n_kv, page, 256), BF16)
    slots, rows = [], {}
    for n, h in zip(new, held):
        pages = [int(order.pop()) for _ in range(h)]
        slots += _slots(pages, page, 0, n)
        rows.update({p: min(page, n - i * page) for i, p in enumerate(pages)})
    assert len(slots) >= 2048
    codes, scales = _empty(sum(held) + 1, n_kv)
    paged.page_bounds(i32(slots), keys, codes, scales)
    _check_bounds(keys, codes, scales, rows)


def _some_bounds(rng, n_pages, n_kv):
    lo, hi = np.sort(rng.integers(-127, 128, (2, n_pages, n_kv, 256)), axis=0)
    codes = torch.tensor(np.stack([lo, hi], axis=2), dtype=torch.int8, device="cuda")
    return codes, torch.tensor(2.0 ** rng.integers(-7, -4, (n_pages, n_kv)), dtype=F32, device="cuda")


def _check_select(q, codes, scales, tables, lens, page, selected, first, recent, requests=None):
    got = paged.select_pages(q, codes, scales, i32(tables), i32(lens), selected, page_size=page, first=first, recent=recent,
                             requests=None if requests is None else i32(requests))
    want = oracle.select_pages(q.double().cpu().numpy(), codes.cpu().numpy(), scales.cpu().numpy(), tables, lens, page, selected, first,
                               recent, requests)
    for x, y in zip(got, want):
        assert x.dtype == torch.int32 and x.is_contiguous() and (x.cpu().numpy() == y).all()
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,n_kv,page,selected,first,recent,lens", [
    (16, 2, 16, 4, 1, 2, [0, 1, 16, 17, 63, 64, 65, 80, 81, 500]),
    (1, 1, 32, 1, 0, 1, [32, 33, 64, 500]),
    (16, 1, 64, 3, 2, 1, [191, 192, 193, 2000]),
    (15, 3, 16, 40, 0, 4, [600, 640, 641, 1600]),
    (8, 8, 256, 5, 1, 4, [1300, 2000, 5000]),
    (8, 2, 16, 100, 3, 3, [30000, 1601, 9999]),
])
def test_the_selection(heads, n_kv, page, selected, first, recent, lens, dtype):
    rng = np.random.default_rng(heads + page)
    width = -(-max(lens) // page) + 1
    n_pages = min(500, sum(-(-n // page) for n in lens) + 2)
    codes, scales = _some_bounds(rng, n_pages, n_kv)
    tables = rng.integers(0, n_pages, (len(lens), width))
    q = ref.rows(rng, (len(lens), heads, 256), dtype) * torch.tensor(2.0 ** rng.integers(-3, 4, heads), device="cuda", dtype=dtype)[None, :, None]
    _check_select(q, codes, scales, tables, lens, page, selected, first, recent)


def test_ties_go_to_the_lower_page():
    """All pages alike; and two kinds of them, of which more than are wanted are the better."""
    codes, scales = _some_bounds(np.random.default_rng(0), 2, 1)
    q = ref.rows(np.random.default_rng(1), (3, 4, 256), F16)
    for tables in (np.zeros((3, 300), dtype=int), np.arange(900).reshape(3, 300) % 2, np.arange(900).reshape(3, 300) // 7 % 2):
        got, _ = _check_select(q, codes, scales, tables, [4800, 4777, 3333], 16, 37, 1, 2)
    got, lens = _check_select(q, codes, scales, np.zeros((3, 300), dtype=int), [4800, 4777, 3333], 16, 37, 1, 2)
    assert (lens.cpu().numpy()[:, 0] == [592, 585, 581]).all()


@pytest.mark.parametrize("width", [1000, 4000, 8000, 20000])
def test_worths_that_are_alike(width):
    """Most pages within a hair of each other and one far below, so that they fall into one bin; many of them the same."""
    rng = np.random.default_rng(width)
    codes, scales = _some_bounds(rng, 40, 1)
    codes[1:] = codes[0]
    codes[1:39, 0, 1, 0] = torch.arange(38, device="cuda").to(torch.int8) + 80
    scales[:] = 2.0 ** -6
    codes[39], scales[39] = torch.where(codes[0] > 0, -127, -126), 2.0 ** 20
    tables = rng.integers(0, 39, (3, width))
    tables[0, 77], tables[1, 5:50], tables[2, 100:] = 39, -1, 7
    q = ref.rows(rng, (3, 4, 256), F32).abs()
    for selected in (3, 30, 700):
        _check_select(q, codes, scales, tables, [16 * width, 16 * width - 5, 16 * width - 16], 16, selected, 1, 2)


def test_pages_that_are_not_in_the_pool_come_last():
    rng = np.random.default_rng(2)
    codes, scales = _some_bounds(rng, 30, 2)
    tables = rng.integers(0, 30, (5, 40))
    tables[0, ::2], tables[1, 1::3], tables[2, 5:], tables[3], tables[4, [0, 38, 39]] = -1, 30, 2 ** 31 - 1, -2 ** 31, -5
    _check_select(ref.rows(rng, (5, 8, 256), BF16), codes, scales, tables, [640, 633, 640, 100, 640], 16, 12, 1, 2)


def test_queries_that_share_a_request_and_lengths_beyond_the_tables():
    rng = np.random.default_rng(3)
    codes, scales = _some_bounds(rng, 60, 2)
    tables = rng.integers(0, 60, (3, 50))
    requests, lens = [2, 2, 2, 0, -1, 1, 3, 2 ** 31 - 1, 2, 0, 0], [600, 601, 602, 7, 500, 799, 500, 500, 603, 2 ** 31 - 1, -3]
    _check_select(ref.rows(rng, (11, 16, 256), F16), codes, scales, tables, lens, 16, 10, 1, 2, requests)


def test_queries_of_any_size():
    """Heads of zeros, and of sizes that reach the ends of the exponents; what is not a number selects pages all the same."""
    rng = np.random.default_rng(4)
    codes, scales = _some_bounds(rng, 64, 1)
    tables = rng.permutation(64)[None].repeat(2, 0)
    q = ref.rows(rng, (2, 8, 256), F32) * torch.tensor([1e30, 1e-30, 0, 1, 1e-10, 3e38, 1e10, 1e-44], device="cuda")[None, :, None]
    q = q.clamp(-3e38, 3e38)
    scales[3], scales[4] = 2.0 ** 50, 2.0 ** -50
    _check_select(q, codes, scales, tables, [1024, 1000], 16, 9, 1, 2)
    q[0, 0, 5], q[1, 2, 7], q[1, 3] = float("nan"), float("inf"), float("nan")
    got, lens = paged.select_pages(q, codes, scales, i32(tables), i32([1024, 1000]), 9, page_size=16)
    for r in range(2):
        at = [list(tables[r]).index(int(p)) for p in got[r, 0]]
        assert at == sorted(set(at)) and at[0] == 0 and at[-2:] == ([62, 63] if r == 0 else [61, 62])


@pytest.mark.parametrize("width", [300, 1024, 1025, 2048, 4100, 8192, 32768])
def test_long_tables(width):
    rng = np.random.default_rng(width)
    codes, scales = _some_bounds(rng, 700, 2)
    tables = rng.integers(0, 700, (2, width))
    for selected in (3, 64, 4096):
        _check_select(ref.rows(rng, (2, 4, 256), BF16), codes, scales, tables, [16 * width, 16 * width - 777], 16, selected, 1, 2)


def _sparse(q, keys, values, codes, scales, tables, lens, selected, scale=SCALE, requests=None, **kw):
    rest = (codes, scales, i32(tables), i32(lens), scale, selected)
    kw["requests"] = None if requests is None else i32(requests)
    if torch.is_tensor(keys):
        return paged.sdpa_decode_paged_sparse(q, keys, values, *rest, **kw)
    return paged.sdpa_decode_paged_sparse_q8(q, *keys, *values, *rest, **kw)


def _case(seed, heads, n_kv, page, lens, dtype, form):
    rng = np.random.default_rng(seed)
    n_pages = sum(-(-n // page) for n in lens) + 2
    keys, values = ref.cache(rng, (n_pages, n_kv, page, 256), dtype, form)
    tables = ref.tables(rng, lens, page, -(-max(lens) // page) + 1, n_pages, list(rng.permutation(n_pages)))
    codes, scales = _empty(n_pages, n_kv)
    paged.page_bounds(i32([s for b, n in enumerate(lens) for s in _slots(tables[b], page, 0, n)]), keys, codes, scales)
    return ref.rows(rng, (len(lens), heads, 256), dtype) * 2, keys, values, codes, scales, tables, lens


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("heads,n_kv,page,selected,lens", [
    (16, 2, 16, 5, [0, 1, 16, 81, 90, 700, 2000]),
    (4, 1, 64, 3, [300, 128, 900]),
    (15, 3, 32, 20, [1500, 641, 640]),
])
def test_attention_over_the_selected_pages(heads, n_kv, page, selected, lens, dtype, form):
    q, keys, values, codes, scales, tables, lens = _case(heads, heads, n_kv, page, lens, dtype, form)
    got = _sparse(q, keys, values, codes, scales, tables, lens, selected)
    chosen, rows = oracle.select_pages(q.double().cpu().numpy(), codes.cpu().numpy(), scales.cpu().numpy(), tables, lens, page, selected, 1, 2)
    n_pages = codes.shape[0]
    at = [[ref.places(np.where(chosen[r, g] < 0, -1, chosen[r, g] // n_kv), rows[r, g], page, n_pages) for g in range(n_kv)]
          for r in range(len(lens))]
    ref.check(got, q, keys, values, at, SCALE)


def test_the_separate_calls_give_the_same_bits():
    q, keys, values, codes, scales, tables, lens = _case(9, 16, 2, 16, [1000, 70, 333, 0], BF16, "rows")
    want = _sparse(q, keys, values, codes, scales, tables, lens, 11, first=2, recent=3)
    t, n = paged.select_pages(q, codes, scales, i32(tables), i32(lens), 11, page_size=16, first=2, recent=3)
    flat = [x.view(-1, 1, 16, 256) for x in (keys, values)]
    got = paged.sdpa_decode_paged(q.view(8, 8, 256), *flat, t.view(8, 11), n.view(8), SCALE)
    assert got.view(4, 16, 256).equal(want)


def test_captured_calls_follow_the_lengths():
    q, keys, values, codes, scales, tables, lens = _case(10, 16, 2, 16, [3000, 70, 333, 1], BF16, "rows")
    t, n = i32(tables), i32(lens)
    graph = torch.cuda.CUDAGraph()
    ws = torch.full((1 << 22,), float("nan"), device="cuda")
    with torch.cuda.graph(graph):
        out = paged.sdpa_decode_paged_sparse(q, keys, values, codes, scales, t, n, SCALE, 11, workspace=ws)
    for cut in (0, 1, 40, 300):
        n.copy_(i32([max(0, x - cut) for x in lens]))
        graph.replay()
        torch.cuda.synchronize()
        assert out.equal(paged.sdpa_decode_paged_sparse(q, keys, values, codes, scales, t, n, SCALE, 11))


def test_operands_outside_the_plain_case_give_the_same_results():
    q, keys, values, codes, scales, tables, lens = _case(11, 16, 2, 16, [1000, 70, 333], F16, "rows")
    want = _sparse(q, keys, values, codes, scales, tables, lens, 6)
    assert _sparse(q.transpose(0, 1).contiguous().transpose(0, 1), keys, values, codes, scales, tables, lens, 6, np.float64(SCALE)).equal(want)
    with pytest.raises(ValueError, match="workspace"):
        _sparse(q, keys, values, codes, scales, tables, lens, 6, workspace=torch.empty(8, device="cuda"))
    with pytest.raises(ValueError, match="must not be negative"):
        _sparse(q, keys, values, codes, scales, tables, lens, 6, -SCALE)
    assert _sparse(q[:0], keys, values, codes, scales, tables[:0], [], 6).shape == (0, 16, 256)
    paged.page_bounds(i32([]), keys, codes, scales)


def test_pages_beyond_2_gb_of_bounds():
    """Offsets of 32 bits and more into the bounds: the last pages of a pool of 2.2 GB of codes."""
    rng = np.random.default_rng(13)
    n_pages, n_kv, page = 550000, 8, 16
    codes = torch.zeros((n_pages, n_kv, 2, 256), dtype=torch.int8, device="cuda")
    scales = torch.ones((n_pages, n_kv), device="cuda")
    some = np.concatenate([np.arange(40), n_pages - 1 - np.arange(40)])
    b, s = _some_bounds(rng, 80, n_kv)
    codes[torch.tensor(some, device="cuda")], scales[torch.tensor(some, device="cuda")] = b, s
    q = ref.rows(rng, (1, 8, 256), BF16)
    order = rng.permutation(80)
    got, _ = paged.select_pages(q, codes, scales, i32(some[order])[None], i32([80 * 16]), 7, page_size=16)
    want, _ = oracle.select_pages(q.double().cpu().numpy(), b.cpu().numpy(), s.cpu().numpy(), order[None], [80 * 16], 16, 7, 1, 2)
    at = want // n_kv
    assert (got.cpu().numpy() == some[at].astype(np.int64) * n_kv + want % n_kv).all()


def test_a_query_that_is_not_a_number_stays_alone():
    """Its own pages are some of its request's, those of the others what they were."""
    rng = np.random.default_rng(40)
    n_pages, page = 90, 16
    keys, values = ref.cache(rng, (n_pages, 2, page, 256), BF16, "rows")
    codes, scales = _empty(n_pages, 2)
    paged.page_bounds(i32(np.arange(n_pages * page)), keys, codes, scales)
    tables = i32(rng.permutation(n_pages)[:80].reshape(4, 20))
    lens = i32([320, 300, 319, 33])
    q = ref.rows(rng, (4, 16, 256), BF16)
    args = (codes, scales, tables, lens)
    want = paged.select_pages(q, *args, 6, page_size=page)
    out = paged.sdpa_decode_paged_sparse(q, keys, values, *args, SCALE, 6)
    odd = q.clone()
    odd[1], odd[2, 3, 7], odd[2, 9, 8] = float("nan"), float("inf"), float("-inf")
    got = paged.select_pages(odd, *args, 6, page_size=page)
    assert got[1].equal(want[1]) and got[0][[0, 3]].equal(want[0][[0, 3]])
    for r in (1, 2):
        for g in range(2):
            at = [int(p) // 2 for p in got[0][r, g]]
            assert len(set(at)) == 6 and set(at) <= set(tables[r].tolist()) and all(int(p) % 2 == g for p in got[0][r, g])
    after = paged.sdpa_decode_paged_sparse(odd, keys, values, *args, SCALE, 6)
    assert after[[0, 3]].equal(out[[0, 3]]) and after[1].isnan().all()
