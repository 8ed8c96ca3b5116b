"""Float64 attention over rows of pages as stored, with a bound of what the kernels' arithmetic may lose (test infrastructure).

The bound is that of ``test_gpu_paged_decode.py`` (its docstring derives it): an error d of every score moves a result by at most 2 d of
sum p |v|, a score being a float32 sum of 256 exact products and a few steps more; a weight is two terms of a 16-bit type; float16
operands lose 2^-36 of the largest value a key; sums over n keys take n / 8 float32 additions where the four waves of a workgroup share
them, and one for every sixteenth piece that is joined (64 pieces: 4, with the waves' 8 and the joins' tree 24 more at most).
"""

import numpy as np
import torch

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def rows(rng, shape, dtype):
    gen = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    return torch.randn(shape, device="cuda", generator=gen).to(dtype)


def codes(rng, shape, dtype, spread=0.03):
    gen = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    c = torch.randint(0, 256, shape, device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8)
    scales = (spread * (0.5 + torch.rand(shape[:3] + (4,), device="cuda", generator=gen))).to(dtype)
    biases = (scales.float() * -(96 + 64 * torch.rand(scales.shape, device="cuda", generator=gen))).to(dtype)
    return c.view(torch.int32).view(torch.uint32), scales, biases


def cache(rng, shape, dtype, form):
    """Keys and values: 16-bit rows of ``dtype``, or 8-bit ones with scales of ``form``."""
    if form == "rows":
        return rows(rng, shape, dtype), rows(rng, shape, dtype)
    return codes(rng, shape, form), codes(rng, shape, form)


def tables(rng, lens, page, width, n_pages, order):
    """Pages of ``order`` (used up from its end); the entries behind a request's rows hold what they like."""
    junk = np.array([-1, -2 ** 31, 2 ** 31 - 1, n_pages, 0])
    out = rng.choice(junk, (len(lens), width)).astype(np.int64)
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            out[b, i] = order.pop()
    return out


def _pick(t, p):
    return t.view(torch.int32)[p].view(t.dtype) if t.dtype == torch.uint32 else t[p]


def stored(side, places, g):
    """Rows at ``places`` ([page], [row]) of KV head ``g`` in 64 bits; of 8-bit rows also what is summed apart, and the largest scales."""
    p, o = places
    if torch.is_tensor(side):
        x = side[p, g, o].double()
        return x, x.abs(), x.abs().max()
    c, s, z = (_pick(t, p)[:, g] for t in side)
    at = torch.arange(len(p), device="cuda")
    s, z = (t[at, o].double().repeat_interleave(64, -1) for t in (s, z))
    c = c.contiguous().view(torch.uint8)[at, o].double()
    return c * s + z, ((c - 128) * s).abs() + (z + 128 * s).abs(), 128 * 2 * s.abs().max()


def places(table, n, page, n_pages):
    """Pages and rows of the first ``n`` rows of a table, less those of pages that are not in the pool."""
    at = [(int(table[i // page]), i % page) for i in range(min(max(int(n), 0), len(table) * page))]
    return [(p, o) for p, o in at if 0 <= p < n_pages]


def attention(q, keys, values, at, scale, half_parts=False):
    """(float64 results, bound without the last rounding) of queries ``[R, Hq, 256]``; ``at[r][g]``: the places that r attends.
    ``half_parts``: partial sums may be stored as float16 numbers of a column's largest, each off by half a step (2^-11 of it, or, below
    2^-14 of the largest, 2^-25 of a power of two that is at most twice that); joined, they are off by the same of the attention over |V|."""
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    G = (keys if torch.is_tensor(keys) else keys[0]).shape[1]
    rep = q.shape[1] // G
    terms = 2.0 ** (-16 if torch.is_tensor(keys) and q.dtype == BF16 else -22)
    for r in range(q.shape[0]):
        for g in range(G):
            if not at[r][g]:
                continue
            where = torch.tensor(at[r][g], device="cuda").t()
            k, k_size, _ = stored(keys, where, g)
            v, v_size, v_most = stored(values, where, g)
            x = q[r, g * rep:(g + 1) * rep].double()
            w = torch.softmax(x @ k.t() * scale, -1)
            most = (x.abs() @ k_size.t()).amax(-1, keepdim=True) * abs(scale)
            h = slice(g * rep, (g + 1) * rep)
            out[r, h] = w @ v
            size = w @ v_size
            if half_parts:
                bound[r, h] = size * 2.0 ** -11 + size.amax(-1, keepdim=True) * 2.0 ** -24
            bound[r, h] += size * (2 * 260 * 2.0 ** -24 * most + terms + 2 * (len(at[r][g]) / 8 + 36) * 2.0 ** -24)
            if q.dtype != BF16 or not torch.is_tensor(keys):
                bound[r, h] += len(at[r][g]) * 2.0 ** -36 * v_most
    return out, bound


def check(got, q, keys, values, at, scale, half_parts=False):
    assert got.dtype == q.dtype and got.shape == q.shape
    want, bound = attention(q, keys, values, at, scale, half_parts)
    bound = bound + torch.finfo(q.dtype).eps / 2 * want.abs() + torch.finfo(q.dtype).tiny
    err = (got.double() - want).abs()
    assert (err <= bound).all(), ((err / bound).nan_to_num(9e9).max(), err.max())
