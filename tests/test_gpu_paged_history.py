"""A server's steps through a layer against float64 attention over each request's own history, which is kept on the host from the
layer's projections: neither tables nor slots nor pages nor what a step says of its rows goes into it.

The projection of the output is left out (an identity), so that every channel of every row has a bound of its own. A result of the
attention is off by what its scores are off by (260 * 2^-24 of the sum of a score's products' magnitudes, twice, of the sum of the
weighted values' magnitudes; codes from 128 on and biases count apart), by its weights' two terms (2^-16 of bfloat16 rows,
2^-22 else) and by its sums (n / 4 + 8 additions, twice), and is rounded to its type (eps / 2). The gate is a sigmoid of the type
(eps: half for its rounding, half for the function), their product is rounded once more (eps / 2).
"""

import pytest
import torch

from moespresso_amd.runtime.qwen import kquant, paged
from test_gpu_paged_attention import BF16, F16, F32, HEADS, HIDDEN, KV_HEADS, STEPS, _Block, _ints

pytestmark = pytest.mark.gpu

REP = HEADS // KV_HEADS


class _History:
    """What one request has seen: rows as the pages should hold them, a part per tensor of a side."""

    def __init__(self, quantized, dtype):
        self.quantized, self.dtype, self.sides = quantized, dtype, ([], [])

    def add(self, k, v):
        for side, row in zip(self.sides, (k, v)):
            side.append(kquant.quantize(row[None].contiguous()) if self.quantized else (row[None].to(self.dtype),))

    def parts(self, side):
        return [torch.cat([p.view(torch.int32) if p.dtype == torch.uint32 else p for p in part]) for part in zip(*self.sides[side])]

    def rows(self, side):
        """(float64 rows [n, KV heads, 256], the magnitudes that are summed for them)"""
        parts = self.parts(side)
        if not self.quantized:
            return parts[0].double(), parts[0].double().abs()
        scale, bias = (t.double().repeat_interleave(64, -1) for t in parts[1:])
        codes = parts[0].view(torch.uint8).double() - 128
        bias = bias + 128 * scale
        return codes * scale + bias, (codes * scale).abs() + bias.abs()


def _attend(q, history, n, scale, out_eps):
    """One query over the first n rows: float64 result [HEADS, 256], and what a kernel's may be off by."""
    (k, k_size), (v, v_size) = (tuple(t[:n] for t in history.rows(side)) for side in (0, 1))
    want, bound = torch.empty(HEADS, 256, dtype=torch.float64, device="cuda"), torch.empty(HEADS, 256, dtype=torch.float64, device="cuda")
    terms = 2.0 ** (-16 if history.dtype == BF16 and not history.quantized else -22)
    for h in range(HEADS):
        g = h // REP
        w = torch.softmax(k[:, g] @ q[h].double() * scale, 0)
        most = (k_size[:, g] @ q[h].double().abs()).max() * scale
        want[h] = w @ v[:, g]
        bound[h] = (w @ v_size[:, g]) * (2 * 260 * 2.0 ** -24 * most + terms + 2 * (n / 4 + 8) * 2.0 ** -24)
        bound[h] += n * 2.0 ** -36 * 256 * v_size.max() + out_eps / 2 * want[h].abs()
    return want, bound


@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("dtype,quantized", [(F32, True), (BF16, False), (F16, False), (BF16, True), (F16, True), (F32, False)])
def test_a_server_against_its_requests_histories(dtype, quantized, axes):
    gen = torch.Generator(device="cuda").manual_seed(15 + axes)
    pages = BF16 if dtype == F32 and not quantized else dtype
    block = _Block(11, dtype)
    block.o_proj = torch.nn.Identity()
    layer = paged.PagedAttention(block, paged.PagedKVCache(14, KV_HEADS, page_size=16, quantized=quantized, dtype=pages))
    tables = paged.PageTables(4, 14, page_size=16, max_tokens=128)
    histories = [_History(quantized, pages) for _ in range(4)]
    eps = torch.finfo(dtype).eps
    missed = 0
    for new in STEPS:
        owner = [b for b, n in enumerate(new) for _ in range(max(n, 0))]
        for b, n in enumerate(new):
            if n < 0:
                histories[b] = _History(quantized, pages)
        seen, before = [], [len(h.sides[0]) for h in histories]
        for b in owner:
            before[b] += 1
            seen.append(before[b])
        rows = len(owner)
        x = torch.randn(rows + 3, HIDDEN, device="cuda", generator=gen).to(dtype)
        step = tables.step(_ints(new), rows + 3)
        # three axes as a prompt with pictures has them; behind the rows any position
        at = torch.tensor([n - 1 for n in seen] + [5, 0, 9], dtype=torch.int32, device="cuda")
        if axes == 3:
            at = torch.stack([at, at // 3, at % 3])
        got = layer(x, step, tables, at if axes == 3 else None)
        assert got.shape == (rows + 3, HEADS * 256) and (got[rows:] == 0).all()
        q, gate = block.q_proj(x).reshape(rows + 3, HEADS, 512).chunk(2, dim=-1)
        k, v = block.k_proj(x).reshape(rows + 3, KV_HEADS, 256), block.v_proj(x).reshape(rows + 3, KV_HEADS, 256)
        q, k = paged.qk_norm_rope(q, k, block.q_norm.weight, block.k_norm.weight, at, block.rope.inv_freq,
                                  sections=block.rope.sections if axes == 3 else None)
        for r, b in enumerate(owner):
            histories[b].add(k[r], v[r])
        asked = q if quantized else q.to(pages)
        gate = torch.sigmoid(gate.double())
        got = got.double().reshape(rows + 3, HEADS, 256)
        for r, (b, n) in enumerate(zip(owner, seen)):
            want, bound = _attend(asked[r], histories[b], n, block.scale, eps if quantized else torch.finfo(pages).eps)
            bound = gate[r] * (bound + 1.5 * eps * (want.abs() + bound)) + torch.finfo(dtype).tiny
            off = (got[r] - gate[r] * want).abs()
            assert (off <= bound).all(), (r, b, n, float((off / bound).max()))
            if n > 1 and r % 5 == 0:  # (a query that misses its newest key is not let through)
                less = _attend(asked[r], histories[b], n - 1, block.scale, eps)[0]
                assert ((got[r] - gate[r] * less).abs() > bound).any()
                missed += 1
        # the pages hold every history, whole and as it is
        for b, history in enumerate(histories):
            n = len(history.sides[0])
            assert int(tables.lens[b]) == n
            if n == 0:
                continue
            held = tables.tables[b, :-(-n // 16)].long()
            for side, stored in enumerate((layer.cache.keys, layer.cache.values)):
                for part, t in zip(history.parts(side), stored if quantized else (stored,)):
                    t = t.view(torch.int32) if t.dtype == torch.uint32 else t
                    assert t[held].transpose(1, 2).flatten(0, 1)[:n].equal(part)
    assert missed > 10
