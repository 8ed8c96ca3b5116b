"""What the speed of the attention forms over a paged Qwen cache is measured on in which a query does not simply read every row of
its own request: a prefix that many requests share, and long contexts of which a query reads the pages that matter.

Four kinds of calls:

* ``shared``  new queries of every request over a prefix that its group shares and over the request's own pages
* ``bounds``  lower and upper bounds of the keys of every page that a step wrote to, in 8 bits
* ``select``  the pages that a query may weigh most, per KV head, from the bounds of all of its request's pages
* ``sparse``  the same selection and the attention over its pages

A pass leaves its state as it found it, or finds again what it left (bounds of the same rows are the same).
"""

import random

import torch

own = False

DIM = 256                                            # width of a head
GROUP = 64                                           # elements per scale and bias of an 8-bit row
LIMIT = 50                                           # exponents of bounds and of query codes lie within +-LIMIT
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # two requests behind a short system prompt: latency counts
        dict(name="shared_2x137", kind="shared", batch=2, rows=1, groups=1, low=137, prefix=137, own=40, heads=16, kv_heads=2,
             page=64, dtype="bfloat16", cache="rows"),
        # the served batch behind one long document
        dict(name="shared_16x32768", kind="shared", batch=16, rows=1, groups=1, low=32768, prefix=32768, own=512, heads=16,
             kv_heads=2, page=64, dtype="bfloat16", cache="rows"),
        # several system prompts of different lengths, small pages, some requests behind none, a few slots idle
        dict(name="shared_61_ragged", kind="shared", batch=61, rows=1, groups=5, low=300, prefix=9001, own=2000, heads=16,
             kv_heads=2, page=16, dtype="float16", cache="rows"),
        # a busy server behind one prompt
        dict(name="shared_256x8192", kind="shared", batch=256, rows=1, groups=1, low=8192, prefix=8192, own=700, heads=16,
             kv_heads=2, page=256, dtype="bfloat16", cache="rows"),
        # three drafted tokens a request, 8-bit rows, float32 activations
        dict(name="shared_11x3x20001_q8", kind="shared", batch=11, rows=3, groups=1, low=20001, prefix=20001, own=300, heads=16,
             kv_heads=2, page=64, dtype="float32", cache="q8"),
        # a token of every request of the served batch
        dict(name="bounds_16", kind="bounds", batch=16, chunk=1, spare=0, kv_heads=2, page=64, dtype="bfloat16", cache="rows"),
        # prompt chunks of several requests in 8-bit pages, rows padded to the batch
        dict(name="bounds_8x2011_q8", kind="bounds", batch=8, chunk=2011, spare=77, kv_heads=2, page=64, dtype="bfloat16",
             cache="q8"),
        # a single user at 8K tokens
        dict(name="select_1x8191", kind="select", batch=1, low=8191, cap=8191, heads=16, kv_heads=2, page=32, dtype="bfloat16",
             cache="rows", selected=64, first=1, recent=2),
        # the served batch at up to 128K tokens each
        dict(name="select_16_ragged", kind="select", batch=16, low=1, cap=131072, heads=16, kv_heads=2, page=64, dtype="bfloat16",
             cache="rows", selected=64, first=1, recent=2),
        # a single user at 128K tokens
        dict(name="sparse_1x131071", kind="sparse", batch=1, low=131071, cap=131071, heads=16, kv_heads=2, page=64,
             dtype="bfloat16", cache="rows", selected=64, first=1, recent=2),
        # many requests of all lengths, some shorter than what is selected, small pages, idle slots
        dict(name="sparse_48_ragged", kind="sparse", batch=48, low=0, cap=30011, heads=16, kv_heads=2, page=16, dtype="float16",
             cache="rows", selected=200, first=2, recent=4),
        # a batch of eight at 37000 tokens with 8-bit rows and float32 activations
        dict(name="sparse_8x37000_q8", kind="sparse", batch=8, low=37000, cap=37000, heads=16, kv_heads=2, page=64,
             dtype="float32", cache="q8", selected=64, first=1, recent=2),
    ]


def draw(rng):
    def spread(low, high):
        high = max(low, high)
        return min(high, max(low, int(round(low * (high / low) ** rng.random()))))

    kind = rng.choice(["shared", "shared", "shared", "bounds", "select", "sparse", "sparse"])
    page = rng.choice([16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 8, 16] if kv_heads <= 2 else [1, 2, 4, 8])
    cache = rng.choice(["rows", "rows", "q8"])
    dtype = rng.choice(["float16", "bfloat16"] if cache == "rows" else ["float32", "float16", "bfloat16"])
    case = dict(kind=kind, kv_heads=kv_heads, page=page, dtype=dtype, cache=cache)
    if kind == "bounds":
        chunk = spread(1, 2048)
        case.update(batch=spread(1, min(256, 16384 // (chunk * kv_heads) + 1)), chunk=chunk, spare=rng.randrange(100))
        return case
    case["heads"] = heads
    if kind == "shared":
        rows = rng.choice([1, 1, 1, 2, 5])
        batch = spread(1, 256 // rows)
        room = (1 << 21) // (batch * rows * kv_heads)
        prefix = spread(1, min(32768, room))
        case.update(batch=batch, rows=rows, groups=rng.randint(1, min(batch, 6)), low=prefix if rng.random() < 0.3 else 1,
                    prefix=prefix, own=spread(1, min(4096, room // 4 + 1)))
        return case
    batch = spread(1, 64)
    cap = min(spread(1, 131072), (1 << 22) // (batch * kv_heads))
    first, recent = rng.randint(0, 3), rng.randint(1, 4)
    case.update(batch=batch, low=cap if rng.random() < 0.3 else rng.choice([0, 1]), cap=cap,
                selected=max(first + recent, spread(4, 8192 // page)), first=first, recent=recent)
    return case


# ---------------------------------------------------------------------------------------------- inputs

def _pages(n, page):
    return -(-n // page)


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lens(case):
    """Lengths of the case, the same for every seed."""
    r = _rng(case)
    if case["kind"] == "shared":
        prefix = [r.randint(case["low"], case["prefix"]) for _ in range(case["groups"])]
        prefix[r.randrange(len(prefix))] = case["prefix"]
        # (of several groups, a request in ten belongs to none; an idle slot has no rows of its own)
        group = [-1 if case["groups"] > 1 and r.random() < 0.1 else r.randrange(case["groups"]) for _ in range(case["batch"])]
        own_rows = [r.randint(1, case["own"]) for _ in range(case["batch"])]
        if case["groups"] > 1:
            own_rows = [0 if g < 0 and r.random() < 0.3 else n for g, n in zip(group, own_rows)]
        return prefix, group, own_rows
    if case["kind"] == "bounds":
        new = [r.randint(1, case["chunk"]) for _ in range(case["batch"])]
        return [r.randint(0, 2 * case["page"]) for _ in new], new
    lens = [r.randint(case["low"], case["cap"]) for _ in range(case["batch"])]
    lens[r.randrange(len(lens))] = case["cap"]
    return lens


def _fill(shape, dtype, dev, gen):
    """Rows of pages ``[n, Hkv, page, 256]``: neighbouring tokens are alike, so that a page has a centre of its own."""
    rows = torch.empty(shape, dtype=dtype, device=dev).normal_(0, 0.7, generator=gen)
    return rows.add_(torch.empty((*shape[:2], 1, shape[3]), dtype=dtype, device=dev).normal_(0, 0.7, generator=gen))


def _side(case, total, dev, gen):
    shape = (total, case["kv_heads"], case["page"], DIM)
    dtype = DTYPES[case["dtype"]]
    if case["cache"] == "rows":
        return _fill(shape, dtype, dev, gen)
    codes = _fill(shape, torch.float16, dev, gen).mul_(40).add_(128).clamp_(0, 255).to(torch.uint8)
    scales = torch.rand((*shape[:3], DIM // GROUP), device=dev, generator=gen) * 0.01 + 0.02
    return codes.view(torch.int32).view(torch.uint32), scales.to(dtype), (scales * -128).to(dtype)


def _tables(held, width, order, dev):
    tables = torch.full((len(held), width), -1, dtype=torch.int32, device=dev)
    used = torch.arange(width, device=dev)[None, :] < torch.tensor(held, dtype=torch.int32, device=dev)[:, None]
    tables[used] = order
    return tables


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    page, G = case["page"], case["kv_heads"]
    state = {"case": case}

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    def queries(n):
        return (2 * torch.randn((n, case["heads"], DIM), device=dev, generator=gen)).to(DTYPES[case["dtype"]])

    if case["kind"] == "shared":
        prefix, group, own_rows = _lens(case)
        held = [_pages(n, page) for n in prefix + own_rows]
        total = sum(held) + 1
        order = torch.randperm(total, device=dev, generator=gen).to(torch.int32)
        n = sum(held[:len(prefix)])
        rows = case["rows"]
        state.update(
            q=queries(case["batch"] * rows), scale=DIM ** -0.5,
            prefix_tables=_tables(held[:len(prefix)], max(held[:len(prefix)]), order[:n], dev), prefix_lens=ints(prefix),
            groups=ints(group), tables=_tables(held[len(prefix):], max(1, *held[len(prefix):]), order[n:total - 1], dev),
            # (row i of a request's new ones sees those before it; with one row a request there is no need to name it)
            lens=ints([max(0, m - rows + 1 + i) for m in own_rows for i in range(rows)]),
            requests=None if rows == 1 else ints([b for b in range(case["batch"]) for _ in range(rows)]))
        state["keys"], state["values"] = _side(case, total, dev, gen), _side(case, total, dev, gen)
        return state

    if case["kind"] == "bounds":
        lens, new = _lens(case)
        held = [_pages(n + k, page) for n, k in zip(lens, new)]
        total = sum(held) + 1
        order = torch.randperm(total, device=dev, generator=gen).tolist()
        state["keys"] = _side(case, total, dev, gen)
        before, after, at = [], [], 0
        for n, k, h in zip(lens, new, held):
            slots = [order[at + i // page] * page + i % page for i in range(n + k)]
            before += slots[:n]
            after += slots[n:]
            at += h
        state["codes"] = torch.zeros((total, G, 2, DIM), dtype=torch.int8, device=dev)
        state["scales"] = torch.zeros((total, G), dtype=torch.float32, device=dev)
        if before:
            _update(state["keys"], ints(before), state["codes"], state["scales"], page)
        # (the state of a page that holds rows is that of its rows before the step; rows behind the batch have no slot)
        state["slots"] = ints(after + [-1] * case["spare"])
        return state

    lens = _lens(case)
    held = [_pages(n, page) for n in lens]
    total = sum(held) + 1
    order = torch.randperm(total, device=dev, generator=gen).to(torch.int32)
    state.update(q=queries(len(lens)), tables=_tables(held, max(1, _pages(case["cap"], page)), order[:sum(held)], dev),
                 lens=ints(lens), scale=DIM ** -0.5)
    state["keys"] = _side(case, total, dev, gen)
    state["codes"] = torch.zeros((total, G, 2, DIM), dtype=torch.int8, device=dev)
    state["scales"] = torch.zeros((total, G), dtype=torch.float32, device=dev)
    _whole_pages(state, page)
    if case["kind"] == "sparse":
        state["values"] = _side(case, total, dev, gen)
    else:
        del state["keys"]
    return state


def _whole_pages(s, page):
    """Bounds of all rows that the requests hold, a few pages at a time."""
    keys = s["keys"]
    held = (s["lens"] + page - 1) // page
    for b, n in enumerate(held.tolist()):
        for i in range(0, n, 256):
            at = s["tables"][b, i:min(n, i + 256)].long()
            rows = _values(_at(keys, at))
            count = (int(s["lens"][b]) - torch.arange(i, i + len(at), device=rows.device) * page).clamp(max=page)
            dead = (torch.arange(page, device=rows.device)[None, :] >= count[:, None])[:, None, :, None]
            low = rows.masked_fill(dead, torch.inf).amin(2)
            high = rows.masked_fill(dead, -torch.inf).amax(2)
            s["codes"][at], s["scales"][at] = _bound_codes(low, high)


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from moespresso_amd.runtime.qwen import paged

    case = s["case"]
    if case["kind"] == "shared":
        rest = (s["prefix_tables"], s["prefix_lens"], s["groups"], s["tables"], s["lens"], s["scale"])
        if case["cache"] == "rows":
            return paged.sdpa_decode_paged_shared(s["q"], s["keys"], s["values"], *rest, requests=s["requests"])
        return paged.sdpa_decode_paged_shared_q8(s["q"], *s["keys"], *s["values"], *rest, requests=s["requests"])
    if case["kind"] == "bounds":
        paged.page_bounds(s["slots"], s["keys"], s["codes"], s["scales"])
        return s["codes"].float() * s["scales"][:, :, None, None]
    some = dict(first=case["first"], recent=case["recent"])
    if case["kind"] == "select":
        return paged.select_pages(s["q"], s["codes"], s["scales"], s["tables"], s["lens"], case["selected"],
                                  page_size=case["page"], **some)
    rest = (s["codes"], s["scales"], s["tables"], s["lens"], s["scale"], case["selected"])
    if case["cache"] == "rows":
        return paged.sdpa_decode_paged_sparse(s["q"], s["keys"], s["values"], *rest, **some)
    return paged.sdpa_decode_paged_sparse_q8(s["q"], *s["keys"], *s["values"], *rest, **some)


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "shared":
        return _shared(s)
    if kind == "bounds":
        _update(s["keys"], s["slots"], s["codes"], s["scales"], s["case"]["page"])
        return s["codes"].float() * s["scales"][:, :, None, None]
    tables, lens = _select(s)
    return (tables, lens) if kind == "select" else _sparse(s, tables, lens)


def _at(side, pages):
    if torch.is_tensor(side):
        return side[pages]
    return tuple(t.view(torch.int32)[pages].view(t.dtype) if t.dtype == torch.uint32 else t[pages] for t in side)


def _values(side, kind=torch.float32):
    """The rows of pages in 32 bits (or more): 16-bit rows, or code * scale + bias."""
    if torch.is_tensor(side):
        return side.to(kind)
    codes, scales, biases = side
    codes = codes.view(torch.uint8).reshape(*scales.shape, GROUP).to(kind)
    return (codes * scales.to(kind)[..., None] + biases.to(kind)[..., None]).flatten(-2)


def _attend(q, keys, values, seen, scale):
    """``q [R, Hkv, rep, 256]`` over ``keys, values [R, Hkv, N, 256]`` where ``seen``; 0 where a row sees nothing."""
    scores = torch.matmul(q, keys.transpose(-1, -2)) * scale
    scores = scores.masked_fill(~seen, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    return torch.matmul(weights, values) / torch.where(total == 0, 1.0, total)


def _shared(s):
    case, q = s["case"], s["q"]
    R, H, _ = q.shape
    G, page = case["kv_heads"], case["page"]
    request = torch.arange(R, device=q.device) if s["requests"] is None else s["requests"].long()
    group = s["groups"].long()[request]
    prefix = torch.where(group < 0, 0, s["prefix_lens"].long()[group.clamp(min=0)])
    wide = s["prefix_tables"].shape[1] * page
    out = torch.empty_like(q)
    # (the rows of every query one behind the other, for as many queries at a time as a few gigabytes hold)
    some = max(1, (1 << 21) // (G * (wide + s["tables"].shape[1] * page)))
    for i in range(0, R, some):
        r = slice(i, min(R, i + some))
        pages = torch.cat([s["prefix_tables"].long()[group[r].clamp(min=0)], s["tables"].long()[request[r]]], dim=1).clamp(min=0)

        def dense(side):
            return _values(_at(side, pages)).transpose(1, 2).flatten(2, 3)

        k = torch.arange(pages.shape[1] * page, device=q.device)[None, :]
        seen = torch.where(k < wide, k < prefix[r, None], k - wide < s["lens"][r, None])
        x = _attend(q[r].float().view(-1, G, H // G, DIM), dense(s["keys"]), dense(s["values"]), seen[:, None, None, :], s["scale"])
        out[r] = x.view(-1, H, DIM).to(q.dtype)
    return out


def _exponent(top):
    """The smallest ``e`` with ``top <= 127 * 2^e``, within the limit."""
    m, e = torch.frexp(top)
    e = e - 7 + (m > 127 / 128)
    return torch.where(top > 0, e, -LIMIT).clamp(-LIMIT, LIMIT)


def _bound_codes(low, high):
    """8-bit codes below ``low`` and above ``high`` (``[n, Hkv, 256]``), and their power of two."""
    e = _exponent(torch.maximum(low.abs(), high.abs()).amax(-1))
    one = torch.ones_like(e, dtype=torch.float32)
    by = torch.ldexp(one, -e)[..., None]
    codes = torch.stack([torch.floor(low * by), torch.ceil(high * by)], dim=2)
    return codes.clamp(-127, 127).to(torch.int8), torch.ldexp(one, e)


def _update(keys, slots, codes, scales, page):
    """Bounds of the pages of ``slots``: of the new rows alone where the page's first is among them, else with the old ones."""
    here = slots >= 0
    slot = slots.long()[here]
    at, row = slot // page, slot % page
    if torch.is_tensor(keys):
        rows = keys[at, :, row].float()
    else:  # in 64 bits: a value next to a whole number of steps must not be rounded to it
        rows = _values(tuple((t.view(torch.int32) if t.dtype == torch.uint32 else t)[at, :, row] for t in keys), torch.float64)
    n, G = scales.shape
    index = at[:, None, None].expand(-1, G, DIM)
    empty = rows.new_full((n, G, DIM), torch.inf)
    low, high = empty.scatter_reduce(0, index, rows, "amin"), empty.neg().scatter_reduce(0, index, rows, "amax")
    touched = torch.zeros(n, dtype=torch.bool, device=rows.device).index_fill_(0, at, True)
    fresh = torch.zeros(n, dtype=torch.bool, device=rows.device).index_fill_(0, at[row == 0], True)
    old = codes.float() * scales[:, :, None, None]
    keep = (touched & ~fresh)[:, None, None]
    low = torch.where(keep, torch.minimum(low, old[:, :, 0]), low)
    high = torch.where(keep, torch.maximum(high, old[:, :, 1]), high)
    low, high = (torch.where(touched[:, None, None], x, 0.0) for x in (low, high))
    new_codes, new_scales = _bound_codes(low, high)
    codes.copy_(torch.where(touched[:, None, None, None], new_codes, codes))
    scales.copy_(torch.where(touched[:, None], new_scales, scales))


def _select(s):
    case, q = s["case"], s["q"]
    R, H, _ = q.shape
    G, page, K = case["kv_heads"], case["page"], case["selected"]
    P = s["tables"].shape[1]
    pages = s["tables"].clamp(min=0).long()
    n = (s["lens"].long() + page - 1) // page
    q = q.float().view(R, G, H // G, DIM)
    e = _exponent(q.abs().amax(-1))
    one = torch.ones_like(e, dtype=torch.float32)
    c = torch.round(q * torch.ldexp(one, -e)[..., None])
    both = torch.cat([c.clamp(max=0), c.clamp(min=0)], dim=-1)  # with the lower bounds, with the upper ones
    codes = s["codes"][pages].transpose(1, 2).flatten(3).float()  # [R, G, P, 512]
    score = torch.matmul(both, codes.transpose(-1, -2)) * torch.ldexp(one, e)[..., None]
    score = score * s["scales"][pages].transpose(1, 2)[:, :, None, :]
    p = torch.arange(P, device=q.device)
    score = score.masked_fill((p[None, :] >= n[:, None])[:, None, None, :], -torch.inf)
    top = score.amax(-1, keepdim=True)
    rank = (score - torch.where(top == -torch.inf, 0.0, top)).amax(2)  # [R, G, P]
    always = (p[None, :] < case["first"]) | ((p[None, :] >= n[:, None] - case["recent"]) & (p[None, :] < n[:, None]))
    rank = torch.where(always[:, None, :], torch.inf, rank)
    some = min(K, P)
    chosen = rank.sort(dim=-1, descending=True, stable=True).indices[..., :some].sort(-1).values
    k = torch.arange(some, device=q.device)[None, None, :]
    chosen = torch.where((n <= K)[:, None, None], k, chosen)
    heads = torch.arange(G, device=q.device)[None, :, None]
    ids = torch.gather(pages, 1, chosen.flatten(1)).view(R, G, some) * G + heads
    ids = torch.where(k < n.clamp(max=K)[:, None, None], ids, -1)
    tables = torch.full((R, G, K), -1, dtype=torch.int32, device=q.device)
    tables[..., :some] = ids.int()
    lens = torch.where(n > K, s["lens"] - (n - K) * page, s["lens"])
    return tables, lens.int()[:, None].expand(R, G).contiguous()


def _sparse(s, tables, lens):
    case, q = s["case"], s["q"]
    R, H, _ = q.shape
    G, page = case["kv_heads"], case["page"]

    def dense(side):
        if torch.is_tensor(side):
            return side.flatten(0, 1)[ids].float().flatten(2, 3)
        flat = tuple((t.view(torch.int32) if t.dtype == torch.uint32 else t).flatten(0, 1) for t in side)
        return _values(tuple(t[ids] for t in flat)).flatten(2, 3)

    ids = tables.clamp(min=0).long()
    k = torch.arange(ids.shape[2] * page, device=q.device)
    seen = k[None, None, :] < lens[:, :, None]
    x = _attend(q.float().view(R, G, H // G, DIM), dense(s["keys"]), dense(s["values"]), seen[:, :, None, :], s["scale"])
    return x.view(R, H, DIM).to(q.dtype)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    size, G, page = SIZE[case["dtype"]], case["kv_heads"], case["page"]
    row = DIM + DIM // GROUP * 2 * size if case["cache"] == "q8" else DIM * 2
    bound = 2 * DIM + 4
    if case["kind"] == "bounds":
        lens, new = _lens(case)
        touched = sum(_pages(n + k, page) - n // page for n, k in zip(lens, new))
        old = sum(n % page > 0 for n in lens)
        return {"bytes": sum(new) * (4 + G * row) + (touched + old) * G * bound, "flops": 0}
    H = case["heads"]
    if case["kind"] == "shared":
        prefix, group, own_rows = _lens(case)
        R = case["batch"] * case["rows"]
        keys = sum(n for g, n in enumerate(prefix) if g in group) + sum(own_rows)
        seen = sum((prefix[g] if g >= 0 else 0) * case["rows"] + sum(max(0, n - i) for i in range(case["rows"]))
                   for g, n in zip(group, own_rows))
        return {"bytes": keys * G * 2 * row + 2 * R * H * DIM * size + 4 * _pages(keys, page), "flops": 4 * seen * H * DIM}
    lens, K = _lens(case), case["selected"]
    scored = sum(n for n in (_pages(m, page) for m in lens) if n > K)
    bytes_ = scored * G * bound + 4 * sum(_pages(m, page) for m in lens) + len(lens) * H * DIM * size
    flops = 2 * scored * H * 2 * DIM
    if case["kind"] == "select":
        return {"bytes": bytes_ + 4 * len(lens) * G * (K + 1), "flops": flops}
    keys = sum(m if _pages(m, page) <= K else m - (_pages(m, page) - K) * page for m in lens)
    return {"bytes": bytes_ + len(lens) * H * DIM * size + keys * G * 2 * row, "flops": flops + 4 * keys * H * DIM}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    if case["kind"] == "select":
        return None  # whole numbers
    s = prepare(case, seed)
    page, G = case["page"], case["kv_heads"]

    def rows(side, at, g):
        """Rows of KV head ``g`` in pages ``at``, one behind the other."""
        if torch.is_tensor(side):
            return side[at, g].double().reshape(-1, DIM)
        codes, scales, biases = side
        scale, bias = (torch.repeat_interleave(t[at, g].double(), GROUP, dim=-1) for t in (scales, biases))
        return (codes.view(torch.uint8)[at, g].double() * scale + bias).reshape(-1, DIM)

    if case["kind"] == "bounds":
        # all rows that a page holds behind the step
        lens, new = _lens(case)
        slots, at = s["slots"].tolist(), 0
        out = s["codes"].double() * s["scales"].double()[:, :, None, None]
        for n, k in zip(lens, new):
            i = 0
            while i < k:
                p, first = divmod(slots[at + i], page)
                count = min(page - first, k - i)
                for g in range(G):
                    x = rows(s["keys"], torch.tensor([p], device="cuda"), g)[:first + count]
                    low, high = x.min(0).values, x.max(0).values
                    top = float(torch.maximum(-low.min(), high.max()))
                    e = -LIMIT
                    while top > 127 * 2.0 ** e and e < LIMIT:
                        e += 1
                    out[p, g, 0] = torch.floor(low / 2.0 ** e).clamp(-127, 127) * 2.0 ** e
                    out[p, g, 1] = torch.ceil(high / 2.0 ** e).clamp(-127, 127) * 2.0 ** e
                i += count
            at += k
        return out

    rep = case["heads"] // G
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")

    def attend(r, g, keys, values):
        if len(keys):
            h = slice(g * rep, (g + 1) * rep)
            out[r, h] = torch.softmax(s["q"][r, h].double() @ keys.t() * s["scale"], dim=-1) @ values

    if case["kind"] == "shared":
        prefix, group, own_rows = _lens(case)
        for g in range(G):
            shared = [tuple(rows(s[x], s["prefix_tables"][i, :_pages(n, page)].long(), g)[:n] for x in ("keys", "values"))
                      for i, n in enumerate(prefix)]
            for b, (i, n) in enumerate(zip(group, own_rows)):
                at = s["tables"][b, :_pages(n, page)].long()
                k, v = (rows(s[x], at, g) for x in ("keys", "values"))
                for j in range(case["rows"]):
                    m = max(0, n - case["rows"] + 1 + j)
                    ks, vs = ([shared[i][x]] if i >= 0 else [] for x in (0, 1))
                    attend(b * case["rows"] + j, g, torch.cat(ks + [k[:m]]), torch.cat(vs + [v[:m]]))
        return out

    for r, m in enumerate(_lens(case)):
        n = _pages(m, page)
        at = s["tables"][r, :n].long()
        for g in range(G):
            keep = torch.arange(n, device="cuda")
            if n > case["selected"]:
                x = s["q"][r, g * rep:(g + 1) * rep].double()
                worth = torch.full((n,), -torch.inf, dtype=torch.float64, device="cuda")
                low, high = (s["codes"][at, g, i].double() * s["scales"][at, g].double()[:, None] for i in (0, 1))
                for h in range(rep):
                    top = float(x[h].abs().max())
                    e = -LIMIT
                    while top > 127 * 2.0 ** e and e < LIMIT:
                        e += 1
                    y = torch.round(x[h] / 2.0 ** e) * 2.0 ** e
                    most = torch.maximum(y * low, y * high).sum(-1)
                    worth = torch.maximum(worth, (most - most.max()).float().double())
                worth[:case["first"]] = torch.inf
                worth[n - case["recent"]:] = torch.inf
                order = sorted(range(n), key=worth.neg().tolist().__getitem__)  # (a stable sort: ties to the lower page)
                keep = torch.tensor(sorted(order[:case["selected"]]), device="cuda")
            last = m - (n - 1) * page if n else 0
            count = (len(keep) - 1) * page + last if n else 0
            attend(r, g, *(rows(s[x], at[keep], g)[:count] for x in ("keys", "values")))
    return out
