"""GPU parity of page_step with the request-by-request oracle: whole numbers, equal."""

import numpy as np
import pytest
import torch

from moespresso_amd.runtime.qwen import paged
from oracle import paged as oracle

pytestmark = pytest.mark.gpu

NAMES = {"lens": "lens", "head": "head", "starts": "starts", "slots": "slots", "positions": "positions", "visible": "visible",
         "requests": "requests", "counts": "counts"}


def _dev(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _pool(rng, lens, page, width, spare):
    """Tables of the lengths' pages in any order, the stack of the others and its top."""
    held = [-(-n // page) for n in lens]
    total = sum(held) + spare
    order = rng.permutation(max(total, 1)).astype(np.int32)
    tables, used = np.full((len(lens), width), -1, dtype=np.int32), 0
    for b, h in enumerate(held):
        tables[b, :h] = order[used:used + h]
        used += h
    free = np.full(max(total, 1), -1, dtype=np.int32)
    free[used:] = order[used:]
    return tables, free, used


def _check(lens, new, tables, free, head, page, n_rows):
    want = oracle.page_step(lens, new, tables, free, head, page, n_rows)
    t, f = _dev(tables), _dev(free)
    got = paged.page_step(_dev(lens), _dev(new), t, f, _dev([head]), page_size=page, n_rows=n_rows)
    for name in NAMES:
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), np.asarray(want[name]), err_msg=name)
    np.testing.assert_array_equal(t.cpu().numpy(), want["tables"])
    np.testing.assert_array_equal(f.cpu().numpy(), want["free_pages"])
    return got, want


@pytest.mark.parametrize("batch,page,width,chunk,ended", [
    (1, 16, 1, 1, 0), (1, 64, 40, 200, 0), (2, 16, 9, 40, 50), (64, 32, 20, 33, 10), (65, 16, 30, 5, 30), (256, 16, 8, 20, 5),
    (257, 128, 4, 90, 20), (1000, 16, 64, 60, 10), (1025, 16, 5, 3, 40), (2048, 32, 6, 7, 25),
])
@pytest.mark.parametrize("spare", ["many", "few", "none"])
def test_steps_of_all_sizes(batch, page, width, chunk, ended, spare):
    rng = np.random.default_rng(batch + page)
    cap = page * width
    new = np.where(rng.random(batch) * 100 < ended, -1, rng.integers(0, chunk + 1, batch))
    lens = rng.integers(0, cap + 1, batch)
    lens[rng.random(batch) < 0.2] = 0
    wanted = int(np.maximum(new, 0).sum() // page + batch)
    tables, free, head = _pool(rng, lens, page, width, {"many": wanted, "few": wanted // 3, "none": 0}[spare])
    n_rows = int(np.maximum(new, 0).sum())
    for rows in sorted({n_rows, n_rows + 37, n_rows * 2 // 3}):  # the batch, padded, and too short for what is asked
        _check(lens, new, tables, free, head, page, rows)


def test_all_requests_end_and_none_ask():
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 500, 30)
    tables, free, head = _pool(rng, lens, 16, 32, 5)
    got, _ = _check(lens, np.full(30, -1), tables, free, head, 16, 0)
    assert int(got.head) == 0 and got.slots.numel() == 0
    _check(lens, np.zeros(30, dtype=int), tables, free, head, 16, 9)


def test_pages_given_back_are_taken_in_the_same_step():
    tables = np.array([[3, 1, -1], [2, -1, -1], [-1, -1, -1]], dtype=np.int32)
    got, want = _check([20, 16, 0], [-1, 1, 17], tables, np.array([-1, -1, -1, 0], dtype=np.int32), 3, 16, 18)
    # request 0 gives back 3 and 1, which lie below the free page 0: request 1 takes 3, request 2 takes 1 and 0
    assert want["tables"][1, 1] == 3 and list(want["tables"][2, :2]) == [1, 0] and int(got.counts[1]) == 0


def test_lengths_and_stack_that_are_out_of_range_stay_in_the_buffers():
    """Lengths beyond the table or below zero, a top outside the stack, more pages given back than were lent, page numbers that
    no pool has: nothing outside the buffers is touched and no row gets a slot outside the pool."""
    B, width, page, n = 8, 4, 16, 10
    guard = torch.full((3 * 64 + B * width + n,), 12345, dtype=torch.int32, device="cuda")
    tables, free = guard[64:64 + B * width].view(B, width), guard[128 + B * width:128 + B * width + n]
    rng = np.random.default_rng(0)
    for head in (-5, 0, 4, 10, 99):
        for new in ([1] * B, [-1] * B, [40, -1] * 4, [2 ** 31 - 1] * B):
            tables.copy_(_dev(rng.integers(-3, 14, (B, width))))
            free.copy_(_dev(rng.integers(-3, 14, n)))
            step = paged.page_step(_dev([-7, 0, 3, 64, 65, 2 ** 31 - 1, 17, 16]), _dev(new), tables.contiguous(), free, _dev([head]),
                                   page_size=page, n_rows=50)
            slots = step.slots.cpu().numpy()
            assert ((slots >= -1) & (slots < n * page)).all()
            assert ((step.lens >= 0) & (step.lens <= width * page)).all() and 0 <= int(step.head) <= n
    edge = torch.cat([guard[:64], guard[64 + B * width:128 + B * width], guard[128 + B * width + n:]])
    assert (edge == 12345).all()


@pytest.mark.parametrize("batch", [40, 1025, 2048])
def test_asked_for_rows_that_add_up_beyond_all_integers(batch):
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 64, batch)
    tables, free, head = _pool(rng, lens, 16, 8, 30)
    new = np.full(batch, 2 ** 31 - 1)
    new[0], new[3], new[9:17] = 5, 0, -1
    got, want = None, oracle.page_step(lens, new, tables, free, head, 16, 300)
    t, f = _dev(tables), _dev(free)
    got = paged.page_step(_dev(lens), _dev(new), t, f, _dev([head]), page_size=16, n_rows=300)
    for name in NAMES:
        if name != "counts":
            np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), np.asarray(want[name]), err_msg=name)
    assert got.counts.tolist()[0] == 2 ** 31 - 1 and got.counts.tolist()[2:] == want["counts"][2:]
    np.testing.assert_array_equal(t.cpu().numpy(), want["tables"])


def test_a_server_of_many_steps_keeps_every_page_in_one_place():
    rng = np.random.default_rng(11)
    B, page, n_pages = 37, 16, 150
    t = paged.PageTables(B, n_pages, page_size=page, max_tokens=400)
    lens, tables, free, head = np.zeros(B, dtype=int), t.tables.cpu().numpy(), t.free_pages.cpu().numpy(), 0
    for _ in range(40):
        new = np.where(rng.random(B) < 0.1, -1, np.where(rng.random(B) < 0.2, rng.integers(0, 60, B), 1))
        n_rows = int(np.maximum(new, 0).sum()) + 3
        want = oracle.page_step(lens, new, tables, free, head, page, n_rows)
        got = t.step(_dev(new), n_rows)
        for name in NAMES:
            np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), np.asarray(want[name]), err_msg=name)
        lens, tables, free, head = np.array(want["lens"]), want["tables"], want["free_pages"], want["head"][0]
        held = np.concatenate([tables[b, :-(-lens[b] // page)] for b in range(B)])
        np.testing.assert_array_equal(np.sort(np.concatenate([held, free[head:]])), np.arange(n_pages))
        np.testing.assert_array_equal(t.lens.cpu().numpy(), lens)
