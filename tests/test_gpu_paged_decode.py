"""GPU parity of decode attention over pages with float64 attention over the rows as stored.

Tolerance, from the arithmetic. A score is a float32 sum of 256 exact products and a few more steps: off by at most
260 * 2^-24 * A, A = scale * sum |q| |k| at its largest over the keys (natural units; the same relative to the exponent's
argument for its rounding). An error d of every score moves the result by at most 2 d of sum p |v|. A weight is two terms
of a 16-bit type, each off by half a step of it (bfloat16 pages 2^-8 of 2^-8 of the weight, float16 operands 2^-11 of 2^-11), or
one float16 term (8-bit pages, bfloat16 result: 2^-11); float16 operands are taken 2^11 times as large and end at 2^-25, so
that n weights lose at most n * 2^-36 of the largest value together (8-bit pages: of 128 times twice the largest scale). Sums
over n keys run over n / 8 float32 additions at most where four waves share a row of keys, over n / 4 where one has it for
itself (128 rows or more: a lane adds eight weights of every 32 keys), counted for both the weights' and the values' sums; the
result is rounded once more, to eps / 2 of its type.
"""

import numpy as np
import pytest
import torch

from moespresso_amd.runtime.qwen import paged
from oracle import paged as oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SCALE = 256 ** -0.5


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _tables(rng, lens, page, width, n_pages):
    """Pages in any order; the entries behind a request's rows hold what they like."""
    order = rng.permutation(n_pages)
    junk = np.array([-1, -2 ** 31, 2 ** 31 - 1, n_pages, 0])
    tables, used = rng.choice(junk, (len(lens), width)).astype(np.int64), 0
    for b, n in enumerate(lens):
        h = -(-n // page)
        tables[b, :h] = order[used:used + h]
        used += h
    return tables


def _rows(rng, shape, dtype):
    gen = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    return torch.randn(shape, device="cuda", generator=gen).to(dtype)


def _codes(rng, shape, dtype, spread=0.03):
    gen = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    codes = torch.randint(0, 256, shape, device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8)
    scales = (spread * (0.5 + torch.rand(shape[:3] + (4,), device="cuda", generator=gen))).to(dtype)
    biases = (scales.float() * -(96 + 64 * torch.rand(scales.shape, device="cuda", generator=gen))).to(dtype)
    return codes.view(torch.int32).view(torch.uint32), scales, biases


def _stored(side):
    if torch.is_tensor(side):
        return side.double()
    codes, scale, bias = side
    return codes.view(torch.uint8).double() * scale.double().repeat_interleave(64, -1) + bias.double().repeat_interleave(64, -1)


def _reference(q, keys, values, tables, lens, scale, requests=None):
    """(float64 result, bound of the error without the last rounding) of every query."""
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    n_pages, G, page = (keys if torch.is_tensor(keys) else keys[0]).shape[:3]
    rep = q.shape[1] // G
    terms = 2.0 ** (-16 if torch.is_tensor(keys) and q.dtype == BF16 else -11 if q.dtype == BF16 else -22)
    for r in range(q.shape[0]):
        b = r if requests is None else int(requests[r])
        n = min(max(int(lens[r]), 0), tables.shape[1] * page) if 0 <= b < len(tables) else 0
        at = [(int(tables[b][i]), min(page, n - i * page)) for i in range(-(-n // page))]
        at = [(p, c) for p, c in at if 0 <= p < n_pages]
        if not at:
            continue
        p = torch.tensor([p for p, _ in at], device="cuda")
        keep = (torch.arange(page, device="cuda")[None, :] < torch.tensor([c for _, c in at], device="cuda")[:, None]).reshape(-1)
        for g in range(G):
            k, v = (_stored(s[p, g][:, None] if torch.is_tensor(s) else tuple(_pick(t, p)[:, g][:, None] for t in s)).reshape(-1, 256)[keep]
                    for s in (keys, values))
            x = q[r, g * rep:(g + 1) * rep].double()
            w = torch.softmax(x @ k.t() * scale, -1)
            most = (x.abs() @ k.abs().t()).amax(-1, keepdim=True) * abs(scale)
            size = w @ v.abs()
            out[r, g * rep:(g + 1) * rep] = w @ v
            largest = v.abs().max()
            if not torch.is_tensor(values):  # codes (from 128 on) and biases are summed apart: their magnitudes count, not the values'
                c, s, z = (_pick(t, p)[:, g] for t in values)
                s, z = (t.double().repeat_interleave(64, -1) for t in (s, z))
                c = ((c.view(torch.uint8).double() - 128) * s).abs() + (z + 128 * s).abs()
                size = w @ c.reshape(-1, 256)[keep]
                largest = 128 * 2 * s.abs().reshape(-1, 256)[keep].max()
                c, s, z = (_pick(t, p)[:, g] for t in keys)
                s, z = (t.double().repeat_interleave(64, -1) for t in (s, z))
                c = ((c.view(torch.uint8).double() - 128) * s).abs() + (z + 128 * s).abs()
                most = (x.abs() @ c.reshape(-1, 256)[keep].t()).amax(-1, keepdim=True) * abs(scale)
            adds = k.shape[0] / (8 if q.shape[0] * G < 128 else 4) + 8
            bound[r, g * rep:(g + 1) * rep] = size * (2 * 260 * 2.0 ** -24 * most + terms + 2 * adds * 2.0 ** -24)
            if q.dtype != BF16 or not torch.is_tensor(keys):
                bound[r, g * rep:(g + 1) * rep] += k.shape[0] * 2.0 ** -36 * largest
    return out, bound


def _pick(t, p):
    return t.view(torch.int32)[p].view(t.dtype) if t.dtype == torch.uint32 else t[p]


def _attend(q, keys, values, tables, lens, scale, **kw):
    if torch.is_tensor(keys):
        return paged.sdpa_decode_paged(q, keys, values, _i32(tables), _i32(lens), scale, **kw)
    return paged.sdpa_decode_paged_q8(q, *keys, *values, _i32(tables), _i32(lens), scale, **kw)


def _check(q, keys, values, tables, lens, scale=SCALE, requests=None):
    got = _attend(q, keys, values, tables, lens, scale, requests=None if requests is None else _i32(requests))
    assert got.dtype == q.dtype and got.shape == q.shape
    want, bound = _reference(q, keys, values, tables, lens, scale, requests)
    bound = bound + torch.finfo(q.dtype).eps / 2 * want.abs() + torch.finfo(q.dtype).tiny
    err = (got.double() - want).abs()
    assert (err <= bound).all(), ((err / bound).nan_to_num(9e9).max(), err.max())
    return got


FORMS = [(F16, "rows"), (BF16, "rows"), (F32, F32), (F32, BF16), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (BF16, F16), (F32, F16),
         (F16, BF16)]


def _cache(rng, shape, dtype, form):
    if form == "rows":
        return _rows(rng, shape, dtype), _rows(rng, shape, dtype)
    return _codes(rng, shape, form), _codes(rng, shape, form)


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("heads,n_kv,page,lens", [
    (16, 2, 16, [1]),
    (16, 2, 64, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65]),
    (1, 1, 32, [127, 128, 129, 0, 160]),
    (16, 1, 16, [300, 4099, 5]),
    (15, 3, 128, [777, 1024, 64]),
    (8, 8, 256, [500, 1]),
])
def test_lengths_heads_and_pages(heads, n_kv, page, lens, dtype, form):
    rng = np.random.default_rng(heads * 100 + page)
    width = -(-max(lens) // page) + 1
    n_pages = sum(-(-n // page) for n in lens) + 2
    keys, values = _cache(rng, (n_pages, n_kv, page, 256), dtype, form)
    q = _rows(rng, (len(lens), heads, 256), dtype) * 2
    got = _check(q, keys, values, _tables(rng, lens, page, width, n_pages), lens)
    for b, n in enumerate(lens):
        assert n or (got[b] == 0).all()


def test_the_oracle_of_one_case_by_hand():
    """The float64 reference above against the row-by-row oracle."""
    rng = np.random.default_rng(5)
    keys, values = _cache(rng, (7, 2, 16, 256), F16, "rows")
    q, tables = _rows(rng, (2, 4, 256), F16), np.array([[3, 1, 99], [6, -1, 0]])
    for lens, requests in (([40, 48], None), ([3, 0], None), ([20, 17], [1, 0])):
        want = oracle.paged_attention(q.double().cpu().numpy(), keys.double().cpu().numpy(), values.double().cpu().numpy(), tables, lens,
                                      SCALE, requests)
        np.testing.assert_allclose(_reference(q, keys, values, tables, lens, SCALE, requests)[0].cpu().numpy(), want, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("dtype,form", [(BF16, "rows"), (F16, "rows"), (F32, F32), (BF16, BF16)])
def test_long_and_ragged_batches(dtype, form):
    rng = np.random.default_rng(8)
    for lens, n_kv, page in (([37000, 1, 20011], 2, 64), ([int(n) for n in rng.integers(0, 900, 70)], 2, 16),
                             ([int(n) for n in rng.integers(0, 60, 300)], 1, 16), ([40000] + [3] * 20, 4, 256)):
        n_pages = sum(-(-n // page) for n in lens) + 1
        keys, values = _cache(rng, (n_pages, n_kv, page, 256), dtype, form)
        q = _rows(rng, (len(lens), 8 * n_kv, 256), dtype) * 2
        _check(q, keys, values, _tables(rng, lens, page, -(-max(lens) // page), n_pages), lens)


@pytest.mark.parametrize("dtype,form", [(BF16, "rows"), (F32, F32), (F16, BF16)])
@pytest.mark.parametrize("n_kv,page,lens", [
    (4, 64, [8000] + [1] * 31),                # rows in tens of parts among whole ones
    (2, 16, [1] * 20 + [5000, 0, 3000] + [40] * 20),
    (8, 32, [70, 3] * 64 + [3000, 65]),        # more rows than shares, one in more than sixteen parts
    (2, 16, [129, 0, 64] * 21 + [1]),          # as few rows as are dealt out to single waves
    (1, 16, [129, 0, 64] * 42 + [1]),          # one fewer
])
def test_long_rows_among_many(n_kv, page, lens, dtype, form):
    rng = np.random.default_rng(len(lens))
    n_pages = sum(-(-n // page) for n in lens) + 1
    keys, values = _cache(rng, (n_pages, n_kv, page, 256), dtype, form)
    q = _rows(rng, (len(lens), 3 * n_kv, 256), dtype) * 2
    _check(q, keys, values, _tables(rng, lens, page, -(-max(lens) // page), n_pages), lens)


@pytest.mark.parametrize("dtype,form", [(BF16, "rows"), (F16, "rows"), (F32, F32), (F16, F16)])
def test_rows_that_do_not_count_may_hold_anything(dtype, form):
    """NaN and infinities behind the last row of a page, and in pages that no table names."""
    rng = np.random.default_rng(2)
    lens, page, n_pages = [1, 16, 17, 40, 63, 64], 64, 9
    keys, values = _cache(rng, (n_pages, 2, page, 256), dtype, form)
    tables = np.arange(6)[:, None] + 1
    want = _attend(_rows(np.random.default_rng(1), (6, 16, 256), dtype), keys, values, tables, lens, SCALE)
    for side in (keys, values):
        for t in (side,) if torch.is_tensor(side) else side[1:]:
            for bad, where in ((float("nan"), 0), (float("inf"), 1), (float("-inf"), 2)):
                t[0], t[7:] = bad, bad
                for p, n in zip(tables[:, 0], lens):
                    t[p, :, n + where::3] = bad
    got = _check(_rows(np.random.default_rng(1), (6, 16, 256), dtype), keys, values, tables, lens)
    assert got.equal(want)


@pytest.mark.parametrize("dtype,form", [(BF16, "rows"), (F32, F32)])
def test_pages_that_are_not_in_the_pool_are_left_out(dtype, form):
    rng = np.random.default_rng(3)
    lens, page, n_pages = [200, 128, 90, 33], 16, 30
    keys, values = _cache(rng, (n_pages, 2, page, 256), dtype, form)
    for t in (keys, values) if form == "rows" else keys[1:] + values[1:]:
        t[0] = float("nan")  # where a page that is not there would be read instead
    tables = rng.integers(1, n_pages, (4, 13))
    tables[0, 3], tables[0, 12], tables[1, :2], tables[2, 5] = -1, n_pages, (2 ** 31 - 1, -2 ** 31), -5
    tables[3] = -1
    got = _check(_rows(rng, (4, 16, 256), dtype), keys, values, tables, lens)
    assert (got[3] == 0).all()


@pytest.mark.parametrize("batch,n_kv", [(64, 2), (65, 2), (128, 1), (129, 8), (1000, 2), (4097, 1), (5000, 2)])
def test_many_queries_of_few_tables(batch, n_kv):
    """More queries than lanes, and more chunks of them than lanes; lengths from none to some tiles, runs of zeros among them."""
    rng = np.random.default_rng(batch)
    keys, values = _cache(rng, (12, n_kv, 16, 256), BF16, "rows")
    tables = rng.integers(0, 12, (7, 9))
    lens, requests = rng.integers(0, 145, batch), rng.integers(0, 7, batch)
    lens[rng.random(batch) < 0.3] = 0
    lens[batch // 3:batch // 2] = 0
    q = _rows(rng, (batch, 2 * n_kv, 256), BF16)
    got = _attend(q, keys, values, tables, lens, SCALE, requests=_i32(requests))
    some = rng.choice(batch, 40, replace=False)
    some[:2] = 0, batch - 1
    want, bound = _reference(q[some], keys, values, tables, lens[some], SCALE, requests[some])
    bound = bound + torch.finfo(BF16).eps / 2 * want.abs() + torch.finfo(BF16).tiny
    assert ((got[some].double() - want).abs() <= bound).all()
    assert (got[torch.from_numpy(lens == 0).cuda()] == 0).all() and not got.isnan().any()


def test_lengths_beyond_the_table_and_below_zero():
    rng = np.random.default_rng(4)
    keys, values = _cache(rng, (9, 2, 16, 256), BF16, "rows")
    got = _check(_rows(rng, (4, 16, 256), BF16), keys, values, np.array([[1, 2], [3, 4], [5, 6], [7, 8]]), [32, 2 ** 31 - 1, -1, -2 ** 31])
    assert (got[2:] == 0).all()


@pytest.mark.parametrize("dtype,form", [(F16, "rows"), (BF16, BF16)])
def test_queries_that_share_a_request(dtype, form):
    """New rows of one chunk, each with what it sees; queries of requests that no table has see nothing."""
    rng = np.random.default_rng(6)
    keys, values = _cache(rng, (40, 2, 16, 256), dtype, form)
    tables = rng.permutation(36).reshape(3, 12)
    requests, lens = [2, 2, 2, 0, -1, 1, 3, 2 ** 31 - 1, 2], [100, 101, 102, 7, 50, 192, 50, 50, 103]
    got = _check(_rows(rng, (9, 16, 256), dtype), keys, values, tables, lens, requests=requests)
    assert (got[4] == 0).all() and (got[6:8] == 0).all()


def test_sharp_and_flat_weights():
    """One key far above all others, and a key above 40000 whose weights are 2^-20 of its: none may be lost."""
    rng = np.random.default_rng(7)
    n, page = 40000, 64
    for dtype in (F16, BF16):
        keys, values = (torch.zeros(n // page + 1, 1, page, 256, dtype=dtype, device="cuda") for _ in range(2))
        tables = rng.permutation(n // page + 1)[None, :n // page]
        values[:, 0, :, 0], values[:, 0, :, 1] = 1, -0.5
        hot = int(tables[0, 300])
        keys[hot, 0, 11, 0], values[hot, 0, 11] = 1, 0
        q = torch.zeros(1, 4, 256, dtype=dtype, device="cuda")
        q[0, :, 0] = torch.tensor([0.0, 13.8629, 30.0, 80.0])
        _check(q, keys, values, tables, [n], scale=1.0)


@pytest.mark.parametrize("dtype,form", [(F32, F32), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("batch", [3, 300])
def test_every_weight_keeps_its_digits(batch, dtype, form):
    """Small queries, whose scores are off by next to nothing, over few keys: a weight of which a term is off by a step of its
    type shows. 300 requests meet 150000 products of a weight and a scale."""
    rng = np.random.default_rng(batch)
    lens = [int(n) for n in rng.integers(1, 12, batch)]
    keys, values = _cache(rng, (batch + 1, 1, 16, 256), dtype, form)
    q = _rows(rng, (batch, 16, 256), dtype) * 2.0 ** -9
    _check(q, keys, values, _tables(rng, lens, 16, 1, batch + 1), lens)


def test_large_queries_of_8_bit_rows():
    """Queries beyond float16's range, and heads of very different sizes."""
    rng = np.random.default_rng(9)
    keys, values = _codes(rng, (6, 1, 32, 256), F32, spread=1e-7), _codes(rng, (6, 1, 32, 256), F32, spread=1e-6)
    q = _rows(rng, (1, 4, 256), F32) * torch.tensor([1e6, 1.0, 1e-6, 0.0], device="cuda")[None, :, None]
    _check(q, keys, values, np.arange(6)[None], [190])
    _check(q.bfloat16(), keys, values, np.arange(6)[None], [190])


def test_values_of_any_size():
    rng = np.random.default_rng(10)
    values = _rows(rng, (6, 1, 32, 256), BF16) * 1e30
    _check(_rows(rng, (1, 4, 256), BF16), _rows(rng, (6, 1, 32, 256), BF16), values, np.arange(6)[None], [190])
    values = _rows(rng, (6, 1, 32, 256), F16) * 2.0 ** -14
    _check(_rows(rng, (1, 4, 256), F16), _rows(rng, (6, 1, 32, 256), F16), values, np.arange(6)[None], [190])


def test_the_same_call_gives_the_same_bits():
    """Whatever the workspace held before."""
    rng = np.random.default_rng(11)
    lens = [int(n) for n in rng.integers(0, 3000, 20)]
    n_pages = sum(-(-n // 16) for n in lens) + 1
    keys, values = _cache(rng, (n_pages, 2, 16, 256), BF16, "rows")
    q, tables = _rows(rng, (20, 16, 256), BF16), _tables(rng, lens, 16, 190, n_pages)
    want = _attend(q, keys, values, tables, lens, SCALE)
    ws = torch.full((1 << 23,), float("nan"), device="cuda")
    assert all(_attend(q, keys, values, tables, lens, SCALE, workspace=ws).equal(want) for _ in range(5))


def test_operands_outside_the_plain_case_give_the_same_results():
    rng = np.random.default_rng(12)
    keys, values = _cache(rng, (9, 2, 16, 256), F16, "rows")
    q, tables, lens = _rows(rng, (3, 16, 256), F16), np.arange(9).reshape(3, 3), [40, 48, 7]
    want = _attend(q, keys, values, tables, lens, SCALE)
    assert _attend(q.transpose(0, 1).contiguous().transpose(0, 1), keys, values, tables, lens, np.float64(SCALE)).equal(want)
    wide = torch.cat([q[:, :, :4], q], dim=2)[:, :, 4:]
    assert _attend(wide, keys, values, tables, lens, SCALE).equal(want)
    with pytest.raises(ValueError, match="workspace"):
        _attend(q, keys, values, np.tile(tables, 40), lens, SCALE, workspace=torch.empty(8, device="cuda"))
    assert _attend(q[:0], keys, values, tables[:0], [], SCALE).shape == (0, 16, 256)


def test_pages_beyond_4_gb():
    """Row offsets of 33 bits: the last pages of a pool of 5 GB a side."""
    rng = np.random.default_rng(13)
    n_pages, page = 20000, 256
    keys, values = (torch.empty(n_pages, 2, page, 256, dtype=BF16, device="cuda") for _ in range(2))
    tables = np.array([[n_pages - 1, 2, n_pages - 3], [n_pages - 2, n_pages - 4, 5]])
    for p in tables.reshape(-1):
        keys[p], values[p] = _rows(rng, (2, page, 256), BF16), _rows(rng, (2, page, 256), BF16)
    _check(_rows(rng, (2, 16, 256), BF16), keys, values, tables, [700, 512])


def test_on_a_stream_of_its_own():
    rng = np.random.default_rng(14)
    keys, values = _cache(rng, (200, 2, 64, 256), BF16, "rows")
    tables, lens = _i32(rng.permutation(200).reshape(4, 50)), _i32([3200, 1, 3000, 2])
    q = _rows(rng, (4, 16, 256), BF16)
    want = paged.sdpa_decode_paged(q, keys, values, tables, lens, SCALE)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = [paged.sdpa_decode_paged(q, keys, values, tables, lens, SCALE) for _ in range(8)]
    stream.synchronize()
    assert all(g.equal(want) for g in got)
