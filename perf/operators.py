"""What the speed of the operators of a paged Qwen cache is measured on: the calls that a server of many requests makes
around one full-attention layer, whose keys and values lie in pages that a table per request names.

Four kinds of calls, in the order of a step:

* ``step``    the tables of a step from the requests' lengths: pages taken and given back, a slot for every new row
* ``rotate``  norm of every query and key head with the rotary position in the same pass, one position axis or three
* ``append``  the same for a step's rows, whose keys and values go to their slots in the pages in that pass
* ``attend``  one new query of every request over the request's pages, of 16-bit or of affine 8-bit rows
"""

import random

import torch

own = False

HEADS, KV_HEADS, DIM = 16, 2, 256                    # Qwen full attention, as served
GROUP = 64                                           # elements per scale and bias of an 8-bit row
ROTARY, THETA, EPS = 64, 1e7, 1e-6                   # rotary width of a head, its base, the norm's epsilon
SECTIONS = (11, 11, 10)                              # frequencies of the time, height and width axes, dealt in turn
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # every request of the served batch decodes a token, in a pool for 128K tokens each: latency counts
        dict(name="step_16", kind="step", batch=16, page=64, cap=131072, chunk=1, ended=0, spare=0,
             short=0),
        # a busy server: one request in twenty ends, one in ten brings a chunk of its prompt, rows padded to the batch
        dict(name="step_1000_turnover", kind="step", batch=1000, page=16, cap=8192, chunk=300, ended=5, spare=77,
             short=0),
        # a single user's next token
        dict(name="rotate_1", kind="rotate", rows=1, heads=16, kv_heads=2, rotary=64, axes=1, gated=True, dtype="bfloat16"),
        # a prompt of text, images and video (three axes) with float32 activations
        dict(name="rotate_3844_axes", kind="rotate", rows=3844, heads=16, kv_heads=2, rotary=64, axes=3, gated=True,
             dtype="float32"),
        # the served batch's next tokens into bfloat16 pages
        dict(name="append_16", kind="append", rows=16, heads=16, kv_heads=2, rotary=64, axes=1, gated=True, page=64,
             dtype="bfloat16", cache="rows"),
        # prompt chunks of several requests, 16384 rows together
        dict(name="append_16384", kind="append", rows=16384, heads=16, kv_heads=2, rotary=64, axes=1, gated=True, page=256,
             dtype="bfloat16", cache="rows"),
        # an odd chunk of a follow-up turn into 8-bit pages
        dict(name="append_517_q8", kind="append", rows=517, heads=16, kv_heads=2, rotary=64, axes=1, gated=True, page=64,
             dtype="bfloat16", cache="q8"),
        # a single user's next token at 8K tokens
        dict(name="attend_1x8191", kind="attend", batch=1, low=8191, cap=8191, heads=16, kv_heads=2, page=64,
             dtype="bfloat16", cache="rows"),
        # a batch of eight at 37000 tokens
        dict(name="attend_8x37000", kind="attend", batch=8, low=37000, cap=37000, heads=16, kv_heads=2, page=256,
             dtype="bfloat16", cache="rows"),
        # many requests of all lengths, a few slots of the batch idle, small pages
        dict(name="attend_64_ragged", kind="attend", batch=64, low=0, cap=16384, heads=16, kv_heads=2, page=16,
             dtype="float16", cache="rows"),
        # a single user at 37000 tokens with 8-bit rows and float32 activations
        dict(name="attend_1x37000_q8", kind="attend", batch=1, low=37000, cap=37000, heads=16, kv_heads=2, page=64,
             dtype="float32", cache="q8"),
        # the served batch with 8-bit rows, up to 128K tokens each
        dict(name="attend_16_ragged_q8", kind="attend", batch=16, low=1, cap=131072, heads=16, kv_heads=2, page=64,
             dtype="bfloat16", cache="q8"),
    ]


def draw(rng):
    def spread(low, high):
        return min(high, max(low, int(round(low * (high / low) ** rng.random()))))

    kind = rng.choice(["step", "rotate", "append", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "step":
        batch = spread(1, 1000)
        return dict(kind=kind, batch=batch, page=page, cap=spread(page, 131072 if batch <= 32 else 8192),
                    chunk=spread(1, 300), ended=rng.choice([0, 5, 30]), spare=rng.randrange(100),
                    short=rng.choice([0, 0, 50]))  # (per cent of the pages wanted that the pool lacks)
    kv_heads = rng.choice([1, 2, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 8, 16] if kv_heads <= 2 else [1, 2, 4, 8])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    if kind == "attend":
        batch = spread(1, 256)
        cap = min(spread(1, 131072), (1 << 20) // (batch * kv_heads))
        cache = rng.choice(["rows", "q8"])
        dtype = rng.choice(["float16", "bfloat16"]) if cache == "rows" else dtype
        low = cap if rng.random() < 0.3 else rng.choice([0, 1])
        return dict(kind=kind, batch=batch, low=low, cap=cap, heads=heads, kv_heads=kv_heads, page=page, dtype=dtype,
                    cache=cache)
    rows = spread(1, min(16384, 16384 * 20 // (heads + 2 * kv_heads)) // (2 if dtype == "float32" else 1))
    case = dict(kind=kind, rows=rows, heads=heads, kv_heads=kv_heads, rotary=rng.choice([64, 64, 128, 256]),
                axes=rng.choice([1, 3]), gated=rng.random() < 0.5, dtype=dtype)
    if kind == "append":
        # (float32 rows in 8-bit pages: a key on the border between two codes may go to either; the codes are compared with
        # the separate calls by the tests)
        cache = rng.choice(["rows", "q8"]) if dtype != "float32" else "rows"
        case.update(page=page, cache=cache)
    return case


# ---------------------------------------------------------------------------------------------- inputs

def _lens(case):
    """Tokens in the cache per request and new ones, the same for every seed."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, cap = case["batch"], case["cap"]
    if case["kind"] == "attend":
        lens = [r.randint(case["low"], cap) for _ in range(n)]
        lens[r.randrange(n)] = cap
        return lens, None
    new = [-1 if r.random() * 100 < case["ended"] else r.randint(1, case["chunk"]) if r.random() < 0.1 else 1 for _ in range(n)]
    return [r.randint(0, max(0, cap - max(k, 0))) for k in new], new


def _pages(n, page):
    return -(-n // page)


def _sections(rotary):
    """Frequencies of the three axes: as served for the served width, in the same proportion for another."""
    half = rotary // 2
    return SECTIONS if half == sum(SECTIONS) else (half - 2 * (half // 3), half // 3, half // 3)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    state = {"case": case}

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, device=dev, generator=gen, dtype=torch.float32).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    if case["kind"] == "step":
        # tables of the requests' pages, which lie in the pool in any order; the other pages are free
        lens, new = _lens(case)
        page, width = case["page"], _pages(case["cap"], case["page"])
        held = [_pages(n, page) for n in lens]
        more = sum(_pages(n + k, page) - _pages(n, page) for n, k in zip(lens, new) if k > 0)
        total = sum(held) + (more + width // 4 + 1 if not case["short"] else more - more * case["short"] // 100)
        order = torch.randperm(total, device=dev, generator=gen).to(torch.int32)
        tables = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
        used = torch.arange(width, device=dev)[None, :] < ints(held)[:, None]
        tables[used] = order[:sum(held)]
        free = torch.full((total,), -1, dtype=torch.int32, device=dev)
        free[sum(held):] = order[sum(held):]
        rows = sum(max(k, 0) for k in new) + case["spare"]
        state.update(lens=ints(lens), new=ints(new), tables=tables, free=free, head=ints([sum(held)]), page=page, rows=rows)
        return state

    dtype, H, G = DTYPES[case["dtype"]], case["heads"], case["kv_heads"]
    if case["kind"] == "attend":
        lens, _ = _lens(case)
        page, width = case["page"], _pages(case["cap"], case["page"])
        held = [_pages(n, page) for n in lens]
        total = sum(held) + 1
        order = torch.randperm(total, device=dev, generator=gen).to(torch.int32)
        tables = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
        tables[torch.arange(width, device=dev)[None, :] < ints(held)[:, None]] = order[:sum(held)]
        state.update(q=(2 * randn(len(lens), H, DIM)).to(dtype), tables=tables, lens=ints(lens), scale=DIM ** -0.5)
        for side in ("keys", "values"):
            if case["cache"] == "rows":
                rows = torch.empty((total, G, page, DIM), dtype=dtype, device=dev)
                state[side] = rows.normal_(generator=gen)
            else:
                codes = torch.empty((total, G, page, DIM), dtype=torch.float16, device=dev).normal_(128, 40, generator=gen)
                codes = codes.clamp_(0, 255).to(torch.uint8)
                scales = torch.rand((total, G, page, DIM // GROUP), device=dev, generator=gen) * 0.01 + 0.02
                state[side] = (codes.view(torch.int32).view(torch.uint32), scales.to(dtype), (scales * -128).to(dtype))
        return state

    # rows of a step as the projections leave them: a query beside its output gate, or heads in one dense row
    T = case["rows"]
    if case["gated"]:
        q = randn(T, H, 2 * DIM, dtype=dtype)[:, :, :DIM]
        k, v = randn(T, G, DIM, dtype=dtype), randn(T, G, DIM, dtype=dtype)
    else:
        row = randn(T, H + 2 * G, DIM, dtype=dtype)
        q, k, v = row[:, :H], row[:, H:H + G], row[:, H + G:]
    inv = (1.0 / THETA ** (torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])).float().to(dev)
    first = int(torch.randint(0, 120000, (1,), device=dev, generator=gen))
    if case["axes"] == 1:
        positions = (first + torch.arange(T, device=dev)).to(torch.int32)
    else:
        t = torch.arange(T, device=dev)
        positions = (first + torch.stack([t // 64, t // 8 % 8, t % 8])).to(torch.int32)
    state.update(q=q, k=k, v=v, inv=inv, positions=positions, q_weight=(1 + 0.1 * randn(DIM)).to(dtype),
                 k_weight=(1 + 0.1 * randn(DIM)).to(dtype), sections=None if case["axes"] == 1 else _sections(case["rotary"]))
    if case["kind"] == "append":
        # slots in pages that lie anywhere in a pool just larger than the rows; some rows of the padded batch have none
        page = case["page"]
        total = _pages(T, page) + 1
        slots = torch.randperm(total - 1, device=dev, generator=gen)[:, None] * page + torch.arange(page, device=dev)
        slots = slots.reshape(-1)[:T].to(torch.int32)
        slots[T - T // 50:] = -1
        state["slots"] = slots
        for side in ("keys", "values"):
            if case["cache"] == "rows":
                kind = torch.bfloat16 if dtype == torch.float32 else dtype
                state[side] = torch.zeros((total, G, page, DIM), dtype=kind, device=dev)
            else:
                state[side] = (torch.zeros((total, G, page, DIM // 4), dtype=torch.int32, device=dev).view(torch.uint32),
                               torch.zeros((total, G, page, DIM // GROUP), dtype=dtype, device=dev),
                               torch.zeros((total, G, page, DIM // GROUP), dtype=dtype, device=dev))
    return state


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from moespresso_amd.runtime.qwen import kquant, paged

    kind = s["case"]["kind"]
    if kind == "step":
        step = paged.page_step(s["lens"], s["new"], s["tables"], s["free"], s["head"], page_size=s["page"], n_rows=s["rows"])
        return {"lens": step.lens, "head": step.head, "starts": step.starts, "slots": step.slots, "positions": step.positions,
                "visible": step.visible, "requests": step.requests, "counts": step.counts, "tables": s["tables"], "free": s["free"]}
    if kind == "attend":
        if s["case"]["cache"] == "rows":
            return paged.sdpa_decode_paged(s["q"], s["keys"], s["values"], s["tables"], s["lens"], s["scale"])
        return paged.sdpa_decode_paged_q8(s["q"], *s["keys"], *s["values"], s["tables"], s["lens"], s["scale"])
    if kind == "rotate":
        return paged.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv"], eps=EPS,
                                  sections=s["sections"])
    q = paged.qk_norm_rope_append(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["positions"], s["inv"], s["slots"],
                                  s["keys"], s["values"], eps=EPS, sections=s["sections"])
    if s["case"]["cache"] == "rows":
        return q, s["keys"], s["values"]
    return q, kquant.dequantize(*s["keys"]), kquant.dequantize(*s["values"])


def _run_plain(s):
    return {"step": _step, "attend": _attend, "rotate": _rotate, "append": _append}[s["case"]["kind"]](s)


def _step(s):
    lens, new, tables, page, n_rows = s["lens"].long(), s["new"].long(), s["tables"], s["page"], s["rows"]
    B, P = tables.shape
    total = s["free"].numel()
    col = torch.arange(P, device=tables.device)
    ended, add = new < 0, new.clamp(min=0)
    held = (lens + page - 1) // page
    goal = (lens + add).clamp(max=P * page)
    need = torch.where(ended, 0, (goal + page - 1) // page - held)
    back = torch.where(ended, held, 0)
    base = s["head"].long() - back.sum()
    # pages of ended requests go on the stack, in the order of the requests (the entry behind the end takes the others)
    at = torch.where(col[None, :] < back[:, None], base + (back.cumsum(0) - back)[:, None] + col[None, :], total)
    free = torch.cat([s["free"], s["free"][:1]]).scatter_(0, at.reshape(-1), tables.reshape(-1))[:total]
    # and the others take theirs from it, as far as there are any
    first = need.cumsum(0) - need
    got = torch.minimum((total - base - first).clamp(min=0), need)
    length = torch.where(ended, 0, torch.minimum(goal, (held + got) * page))
    take = (col[None, :] >= held[:, None]) & (col[None, :] < (held + got)[:, None])
    taken = free[(base + (first - held)[:, None] + col[None, :]).clamp(0, total - 1)]
    table = torch.where(take, taken, tables)
    starts = torch.cat([add.new_zeros(1), add.cumsum(0)])
    # a slot for every new row
    row = torch.arange(n_rows, device=tables.device)
    request = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    live = request < B
    r = request.clamp(max=B - 1)
    position = lens[r] + row - starts[r]
    fits = live & (position < length[r])
    place = table[r, (position // page).clamp(0, P - 1)].long() * page + position % page
    s["tables"].copy_(table)
    s["free"].copy_(free)
    counts = torch.stack([starts[-1], (add - (length - lens) * ~ended).sum(), got.sum(), back.sum()])
    head = base + got.sum()
    return {"lens": length.int(), "head": head.int(), "starts": starts.int(), "slots": torch.where(fits, place, -1).int(),
            "positions": torch.where(live, position, 0).int(),
            "visible": torch.where(fits, position + 1, 0).int(), "requests": torch.where(live, request, -1).int(),
            "counts": counts.int(), "tables": s["tables"], "free": s["free"]}


def _values(side):
    """The rows of pages in 32 bits: 16-bit rows, or code * scale + bias."""
    if torch.is_tensor(side):
        return side.float()
    codes, scales, biases = side
    codes = codes.view(torch.uint8).reshape(*scales.shape, GROUP).float()
    return (codes * scales.float()[..., None] + biases.float()[..., None]).flatten(-2)


def _dense(side, pages):
    """The pages of every request one behind the other: ``[B, Hkv, P * page, 256]``."""
    rows = _values(side[pages] if torch.is_tensor(side) else tuple(_take(t, pages) for t in side))
    return rows.transpose(1, 2).flatten(2, 3)


def _take(t, pages):
    return t.view(torch.int32)[pages].view(t.dtype) if t.dtype == torch.uint32 else t[pages]


def _attend(s):
    q, lens = s["q"], s["lens"]
    pages = s["tables"].clamp(min=0).long()
    B, H, _ = q.shape
    G = s["case"]["kv_heads"]
    keys = _dense(s["keys"], pages)
    scores = torch.matmul(q.float().view(B, G, H // G, DIM), keys.transpose(-1, -2)) * s["scale"]
    seen = torch.arange(keys.shape[2], device=q.device)[None, :] < lens[:, None]
    scores = scores.masked_fill(~seen[:, None, None, :], -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, _dense(s["values"], pages)) / torch.where(total == 0, 1.0, total)
    return out.view(B, H, DIM).to(q.dtype)


def _axis(sections, half, device):
    """The position axis of every frequency: the axes take turns until the shorter ones are used up."""
    i = torch.arange(half, device=device)
    axis = torch.where((i % 3 == 1) & (i < 3 * sections[1]), 1, 0)
    return torch.where((i % 3 == 2) & (i < 3 * sections[2]), 2, axis)


def _norm_rope(x, weight, positions, inv, sections):
    """In 32 bits, the angles in 64; not rounded."""
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.float()
    half = inv.numel()
    if sections is None:
        angle = positions.double()[:, None] * inv.double()
    else:
        angle = positions.double().transpose(0, 1)[:, _axis(sections, half, x.device)] * inv.double()
    angle = torch.remainder(angle, 2 * torch.pi)
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    a, b = y[..., :half], y[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], dim=-1)


def _rotate(s):
    return tuple(_norm_rope(s[x], s[x + "_weight"], s["positions"], s["inv"], s["sections"]).to(s[x].dtype) for x in "qk")


def _quantize(x):
    """Affine codes of groups of 64: the edge of larger magnitude is met exactly."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((high - low) / 255.0).clamp(min=1e-7)
    side = low.abs() > high.abs()
    scale = torch.where(side, scale, -scale)
    edge = torch.where(side, low, high)
    steps = torch.round(edge / scale)
    zero = steps == 0
    scale = torch.where(zero, scale, edge / torch.where(zero, 1.0, steps))
    bias = torch.where(zero, 0.0, edge)
    codes = torch.round((g - bias) / scale).clamp(0, 255).to(torch.uint8).flatten(-2)
    return codes.view(torch.int32), scale.squeeze(-1).to(x.dtype), bias.squeeze(-1).to(x.dtype)


def _put(pages, rows, slots):
    """Rows ``[T, Hkv, W]`` to their slots; those without one write again what the unused last page begins with."""
    page = pages.shape[2]
    here = slots >= 0
    at = torch.where(here, slots.long(), pages.shape[0] * page - page)
    rows = torch.where(here[:, None, None], rows.to(pages.dtype), pages[-1, :, 0])
    pages[at // page, :, at % page] = rows


def _append(s):
    q = _norm_rope(s["q"], s["q_weight"], s["positions"], s["inv"], s["sections"]).to(s["q"].dtype)
    k = _norm_rope(s["k"], s["k_weight"], s["positions"], s["inv"], s["sections"])
    for side, x in (("keys", k), ("values", s["v"])):
        if s["case"]["cache"] == "rows":
            _put(s[side], x, s["slots"])
        else:
            for pages, rows in zip(s[side], _quantize(x.to(s["v"].dtype))):
                _put(pages.view(torch.int32) if pages.dtype == torch.uint32 else pages, rows, s["slots"])
    if s["case"]["cache"] == "rows":
        return q, s["keys"], s["values"]
    return q, _values(s["keys"]).to(q.dtype), _values(s["values"]).to(q.dtype)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "step":
        lens, new = _lens(case)
        rows = sum(max(k, 0) for k in new) + case["spare"]
        taken = sum(_pages(n + k, case["page"]) - _pages(n, case["page"]) for n, k in zip(lens, new) if k > 0)
        back = sum(_pages(n, case["page"]) for n, k in zip(lens, new) if k < 0)
        return {"bytes": 16 * len(lens) + 16 * rows + 8 * (taken + back), "flops": 0}
    size, H, G = SIZE[case["dtype"]], case["heads"], case["kv_heads"]
    row = DIM + DIM // GROUP * 2 * size if case.get("cache") == "q8" else DIM * 2
    if case["kind"] == "attend":
        lens, _ = _lens(case)
        keys = sum(lens)
        return {"bytes": keys * G * 2 * row + 2 * len(lens) * H * DIM * size + 4 * sum(_pages(n, case["page"]) for n in lens),
                "flops": 4 * keys * H * DIM}
    T = case["rows"]
    if case["kind"] == "rotate":
        return {"bytes": T * (2 * (H + G) * DIM * size + 4 * case["axes"]), "flops": 0}
    kept = T - T // 50
    return {"bytes": T * (2 * H * DIM * size + 4 * case["axes"] + 4) + kept * 2 * G * (DIM * size + row), "flops": 0}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    if case["kind"] == "step":
        return None  # whole numbers
    s = prepare(case, seed)

    def wide(side):
        if torch.is_tensor(side):
            return side.double()
        codes = side[0].view(torch.uint8).double()
        scale, bias = (torch.repeat_interleave(t.double(), GROUP, dim=-1) for t in side[1:])
        return codes * scale + bias

    if case["kind"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        G, rep = case["kv_heads"], case["heads"] // case["kv_heads"]
        for b, n in enumerate(_lens(case)[0]):
            if n == 0:
                continue
            at = s["tables"][b, :_pages(n, case["page"])].long()
            for g in range(G):
                def rows(side):
                    part = side[at, g] if torch.is_tensor(side) else tuple(_take(t, at)[:, g] for t in side)
                    return wide(part).reshape(-1, DIM)[:n]

                p = torch.softmax(s["q"][b, g * rep:(g + 1) * rep].double() @ rows(s["keys"]).t() * s["scale"], dim=-1)
                out[b, g * rep:(g + 1) * rep] = p @ rows(s["values"])
        return out

    def coded(x, dtype):
        x = x.view(*x.shape[:-1], DIM // GROUP, GROUP)
        low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        edge = torch.where(-low > high, low, high)  # the one of larger magnitude is a whole number of steps from zero
        step = torch.maximum((high - low) / 255, torch.full_like(low, 1e-7)) * torch.where(-low > high, 1, -1)
        n = torch.round(edge / step)
        step, bias = torch.where(n == 0, step, edge / n), torch.where(n == 0, 0, edge)
        codes = ((x - bias) / step).round().clamp(0, 255)
        return (codes * step.to(dtype).double() + bias.to(dtype).double()).reshape(*x.shape[:-2], DIM)

    def turned(x, weight):
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.double()
        half = case["rotary"] // 2
        for i in range(half):
            if s["sections"] is None:
                where = s["positions"]
            else:
                axis = i % 3 if i % 3 and i < 3 * s["sections"][i % 3] else 0
                where = s["positions"][axis]
            angle = where.double() * s["inv"][i].double()
            c, d = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            a, b = x[:, :, i].clone(), x[:, :, i + half].clone()
            x[:, :, i], x[:, :, i + half] = a * c - b * d, a * d + b * c
        return x

    q, k = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"])
    if case["kind"] == "rotate":
        return q, k
    if case["cache"] == "q8":  # a key is rounded to its type, then to a code; scales and biases have its type too
        k = coded(k.to(s["k"].dtype).double(), s["k"].dtype)
        s["v"] = coded(s["v"].double(), s["v"].dtype)
    pages = []
    for x in (k, s["v"].double()):
        total = _pages(case["rows"], case["page"]) + 1
        pool = x.new_zeros((total * case["page"], case["kv_heads"], DIM))
        here = s["slots"] >= 0
        pool[s["slots"][here].long()] = x[here]
        pages.append(pool.view(total, case["page"], case["kv_heads"], DIM).transpose(1, 2))
    return q, pages[0], pages[1]
