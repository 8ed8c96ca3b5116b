"""What the operators over shared prefixes and selected pages refuse, before anything is launched (CPU)."""

import contextlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from moespresso_amd import _lib
from moespresso_amd.runtime.qwen import paged

I32 = torch.int32
LONG = torch.zeros(3, dtype=torch.int64)


def _ints(*shape):
    return torch.zeros(shape, dtype=I32)


def _rows(n=5, heads=2, page=16, dtype=torch.float16):
    return torch.zeros(n, heads, page, 256, dtype=dtype)


def _triplet(n=5, heads=2, page=16, dtype=torch.float32):
    return (torch.zeros(n, heads, page, 64, dtype=I32), torch.zeros(n, heads, page, 4, dtype=dtype),
            torch.zeros(n, heads, page, 4, dtype=dtype))


def _bounds(n=5, heads=2):
    return dict(codes=torch.zeros(n, heads, 2, 256, dtype=torch.int8), scales=torch.ones(n, heads))


OPERANDS = [
    (dict(queries=torch.zeros(3, 4, 128).half()), "queries must be"),
    (dict(queries=torch.zeros(3, 3, 256).half()), "multiple"),
    (dict(queries=torch.zeros(3, 34, 256).half()), "multiple"),
    (dict(queries=torch.zeros(3, 4, 256)), "dtype of queries"),
    (dict(tables=_ints(2, 4), groups=_ints(2)), "table of its own"),
    (dict(tables=_ints(3, 0)), "tables must be"),
    (dict(lens=_ints(2)), "lens must be"),
    (dict(lens=LONG), "lens must be"),
    (dict(requests=_ints(2)), "requests must be"),
    (dict(requests=LONG), "requests must be"),
    (dict(keys=_triplet(), values=_triplet()), "8-bit ones"),
    (dict(keys=_rows(page=24), values=_rows(page=24)), "power of two"),
    (dict(keys=_rows(), values=_rows(n=4)), "share a shape"),
]


@pytest.mark.parametrize("change,message", OPERANDS + [
    (dict(prefix_tables=_ints(2)), "prefix_tables must be"),
    (dict(prefix_tables=_ints(0, 3), prefix_lens=_ints(0)), "prefix_tables must be"),
    (dict(prefix_tables=_ints(2, 0)), "prefix_tables must be"),
    (dict(prefix_tables=_ints(3, 2).t()), "prefix_tables must be a contiguous"),
    (dict(prefix_tables=torch.zeros(2, 3, dtype=torch.int64)), "prefix_tables must be a contiguous int32"),
    (dict(prefix_lens=_ints(3)), "prefix_lens must be"),
    (dict(prefix_lens=LONG[:2]), "prefix_lens must be"),
    (dict(groups=_ints(2)), "groups must be"),
    (dict(groups=LONG), "groups must be"),
    (dict(prefix_tables=_ints(2049, 3), prefix_lens=_ints(2049)), "at most 2048 prefixes"),
    (dict(queries=torch.zeros(2049, 4, 256).half(), lens=_ints(2049), requests=_ints(2049)), "at most 2048 queries"),
])
def test_shared_prefixes_refuse(change, message):
    a = dict(queries=torch.zeros(3, 4, 256).half(), keys=_rows(), values=_rows(), prefix_tables=_ints(2, 3), prefix_lens=_ints(2),
             groups=_ints(3), tables=_ints(3, 4), lens=_ints(3), requests=None)
    a.update(change)
    requests = a.pop("requests")
    with pytest.raises(ValueError, match=message):
        paged.sdpa_decode_paged_shared(*a.values(), 0.1, requests=requests)


@pytest.mark.parametrize("change,message", [
    (dict(slots=LONG), "slots must be"),
    (dict(slots=_ints(3, 1)), "slots must be"),
    (dict(codes=torch.zeros(5, 2, 2, 256, dtype=torch.uint8)), "codes must be int8"),
    (dict(codes=torch.zeros(5, 2, 256, dtype=torch.int8)), "codes must be int8"),
    (dict(codes=torch.zeros(4, 2, 2, 256, dtype=torch.int8)), "codes must be int8"),
    (dict(codes=torch.zeros(5, 1, 2, 256, dtype=torch.int8)), "codes must be int8"),
    (dict(codes=torch.zeros(5, 2, 256, 2, dtype=torch.int8).transpose(2, 3)), "contiguous"),
    (dict(codes=torch.zeros(5 * 1024 + 1, dtype=torch.int8)[1:].reshape(5, 2, 2, 256)), "16-byte aligned"),
    (dict(scales=torch.ones(5, 2).half()), "scales must be float32"),
    (dict(scales=torch.ones(5)), "scales must be float32"),
    (dict(scales=torch.ones(2, 5).t()), "contiguous"),
    (dict(keys=_rows(dtype=torch.float32)), "float16 or bfloat16 pages"),
    (dict(keys=_rows(page=8)), "power of two"),
    (dict(keys=_triplet()[:2]), "must be .codes, scales, biases"),
])
def test_bounds_refuse(change, message):
    a = dict(slots=_ints(3), keys=_rows(), **_bounds())
    a.update(change)
    with pytest.raises(ValueError, match=message):
        paged.page_bounds(*a.values())


SELECTION = [
    (dict(n_selected=0), "n_selected must be"),
    (dict(n_selected=4097), "n_selected must be"),
    (dict(n_selected=-1), "n_selected must be"),
    (dict(first=-1), "n_selected must be"),
    (dict(recent=0), "n_selected must be"),
    (dict(first=2, recent=2), "n_selected must be"),
    (dict(tables=_ints(3, 32769)), "at most 32768 pages"),
    (dict(queries=torch.zeros(32768, 4, 256).half(), lens=_ints(32768), requests=_ints(32768)), "at most 65535"),
    (dict(codes=torch.zeros(5, 2, 2, 128, dtype=torch.int8)), "codes must be int8"),
    (dict(scales=torch.ones(4, 2)), "scales must be float32"),
]


@pytest.mark.parametrize("change,message", [c for c in OPERANDS if not {"keys", "values"} & set(c[0]) and "dtype of" not in c[1]] + SELECTION + [
    (dict(queries=torch.zeros(3, 4, 256).double()), "float32, float16 or bfloat16"),
    (dict(page_size=24), "power of two"),
    (dict(codes=torch.zeros(5, 2, 256, dtype=torch.int8)), "codes must be int8"),
    (dict(codes=torch.zeros(5, 0, 2, 256, dtype=torch.int8)), "codes must be int8"),
])
def test_the_selection_refuses(change, message):
    a = dict(queries=torch.zeros(3, 4, 256).half(), **_bounds(), tables=_ints(3, 4), lens=_ints(3), n_selected=3, page_size=16, first=1,
             recent=2, requests=None)
    a.update({k: v for k, v in change.items() if k != "groups"})
    kwargs = {k: a.pop(k) for k in ("page_size", "first", "recent", "requests")}
    with pytest.raises(ValueError, match=message):
        paged.select_pages(*a.values(), **kwargs)


@pytest.mark.parametrize("change,message", OPERANDS + SELECTION + [
    (dict(codes=torch.zeros(4, 2, 2, 256, dtype=torch.int8), scales=torch.ones(4, 2)), "codes must be int8"),
])
def test_selected_pages_refuse(change, message):
    a = dict(queries=torch.zeros(3, 4, 256).half(), keys=_rows(), values=_rows(), **_bounds(), tables=_ints(3, 4), lens=_ints(3), scale=0.1,
             n_selected=3, first=1, recent=2, requests=None)
    a.update({k: v for k, v in change.items() if k != "groups"})
    kwargs = {k: a.pop(k) for k in ("first", "recent", "requests")}
    with pytest.raises(ValueError, match=message):
        paged.sdpa_decode_paged_sparse(*a.values(), **kwargs)


def test_8_bit_forms_refuse():
    q, t, n = torch.zeros(3, 4, 256), _ints(3, 4), _ints(3)
    k, b = _triplet(), _bounds().values()
    wide = torch.zeros(5, 2, 16, 256, dtype=torch.uint8)

    def shared(q=q, k=k, **kwargs):
        return paged.sdpa_decode_paged_shared_q8(q, *k, *k, _ints(2, 3), _ints(2), _ints(3), t, n, 0.1, **kwargs)

    def sparse(q=q, k=k, **kwargs):
        return paged.sdpa_decode_paged_sparse_q8(q, *k, *k, *b, t, n, 0.1, 3, **kwargs)

    for call in (shared, sparse):
        with pytest.raises(ValueError, match="group_size=64, bits=8"):
            call(bits=4)
        with pytest.raises(ValueError, match="group_size=64, bits=8"):
            call(group_size=32)
        with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
            call(q.double())
        with pytest.raises(ValueError, match="uint32 pages"):
            call(k=(wide,) + _triplet()[1:])


def test_host_tensors_are_refused():
    q, b = torch.zeros(3, 4, 256).half(), _bounds()
    for call in (lambda: paged.sdpa_decode_paged_shared(q, _rows(), _rows(), _ints(2, 3), _ints(2), _ints(3), _ints(3, 4), _ints(3), 0.1),
                 lambda: paged.page_bounds(_ints(3), _rows(), **b),
                 lambda: paged.select_pages(q, *b.values(), _ints(3, 4), _ints(3), 3, page_size=16),
                 lambda: paged.sdpa_decode_paged_sparse(q, _rows(), _rows(), *b.values(), _ints(3, 4), _ints(3), 0.1, 3)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


@pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")
def test_the_library_refuses_what_its_kernels_do_not_take():
    """The same through the C-ABI, with pointers that are never followed."""
    lib, p = _lib.lib(), _lib.c_void_p(4096)

    def shared(dtype=1, q=4096, batch=3, hq=4, hkv=2, dim=256, pages=5, page=16, prefixes=2, pwidth=3, tables=3, width=4, ws=1 << 40,
               requests=None, groups=4096, at=4096):
        return lib.mspr_sdpa_decode_paged_shared(q, p, p, dtype, p, p, groups, p, p, requests, batch, hq, hkv, dim, pages, page, prefixes,
                                                 pwidth, tables, width, 0.1, p, at, ws, None)

    def shared_q8(dtype=0, sb=0, size=64, bits=8, k=4096, ws=1 << 40, prefixes=2):
        return lib.mspr_sdpa_decode_paged_shared_q8(p, dtype, k, p, p, p, p, p, sb, p, p, p, p, p, None, 3, 4, 2, 256, 5, 16, prefixes, 3, 3, 4,
                                                    0.1, size, bits, p, p, ws, None)

    def bounds(dtype=1, slots=4096, tokens=3, hkv=2, dim=256, pages=5, page=16, codes=4096):
        return lib.mspr_page_bounds(slots, p, dtype, tokens, hkv, dim, pages, page, codes, p, None)

    def bounds_q8(sb=0, k=4096, tokens=3):
        return lib.mspr_page_bounds_q8(p, k, p, p, sb, tokens, 2, 256, 5, 16, p, p, None)

    def select(dtype=1, q=4096, codes=4096, batch=3, hq=4, hkv=2, dim=256, pages=5, page=16, tables=3, width=4, selected=3, first=1, recent=2,
               ws=1 << 40, requests=None, out=4096):
        return lib.mspr_select_pages(q, dtype, codes, p, p, p, requests, batch, hq, hkv, dim, pages, page, tables, width, selected, first,
                                     recent, out, p, p, ws, None)

    def sparse(dtype=1, q=4096, k=4096, batch=3, pages=5, page=16, width=4, selected=3, recent=2, scale=0.1, ws=1 << 40):
        return lib.mspr_sdpa_decode_paged_sparse(q, k, p, dtype, p, p, p, p, None, batch, 4, 2, 256, pages, page, batch, width, selected, 1,
                                                 recent, scale, p, p, ws, None)

    def sparse_q8(dtype=0, sb=0, k=4096, size=64, bits=8, scale=0.1, ws=1 << 40):
        return lib.mspr_sdpa_decode_paged_sparse_q8(p, dtype, k, p, p, p, p, p, sb, p, p, p, p, None, 3, 4, 2, 256, 5, 16, 3, 4, 3, 1, 2, scale,
                                                    size, bits, p, p, ws, None)

    nan = float("nan")
    refused = [shared(dtype=0), shared(dtype=3), shared(q=None), shared(q=4104), shared(batch=0), shared(batch=2049, tables=2049), shared(hq=3),
               shared(hq=34), shared(hkv=0), shared(dim=128), shared(pages=0), shared(pages=1 << 28), shared(page=24), shared(page=8),
               shared(prefixes=0), shared(prefixes=2049), shared(pwidth=0), shared(pwidth=1 << 27), shared(tables=2), shared(tables=0, requests=4096),
               shared(width=0), shared(width=1 << 27), shared(ws=64), shared(groups=None), shared(at=None), shared(at=4100),
               shared(batch=2048, tables=2048, hkv=1024, hq=1024, width=1 << 20),
               shared_q8(dtype=3), shared_q8(sb=3), shared_q8(size=32), shared_q8(bits=4), shared_q8(k=4104), shared_q8(ws=64), shared_q8(prefixes=0),
               bounds(dtype=0), bounds(slots=None), bounds(tokens=0), bounds(tokens=-1), bounds(hkv=0), bounds(dim=128), bounds(pages=0),
               bounds(pages=1 << 28), bounds(page=24), bounds(codes=4104), bounds_q8(sb=3), bounds_q8(k=None), bounds_q8(tokens=0),
               select(dtype=3), select(q=None), select(q=4104), select(codes=4104), select(batch=0), select(batch=32768, tables=32768), select(hq=3),
               select(hq=34), select(hkv=0), select(dim=128), select(pages=0), select(pages=1 << 27), select(page=24), select(tables=2),
               select(tables=0, requests=4096), select(width=0), select(width=32769), select(selected=0), select(selected=4097), select(first=-1),
               select(recent=0), select(first=2), select(ws=0), select(out=None),
               sparse(dtype=0), sparse(q=None), sparse(k=None), sparse(k=4104), sparse(batch=0), sparse(pages=1 << 27), sparse(page=8), sparse(width=0),
               sparse(selected=0), sparse(selected=2), sparse(recent=0), sparse(scale=-0.1), sparse(scale=nan), sparse(ws=64),
               sparse(page=1 << 20, selected=4096, pages=1, width=1024),
               sparse_q8(dtype=3), sparse_q8(sb=3), sparse_q8(k=None), sparse_q8(k=4104), sparse_q8(size=32), sparse_q8(bits=4), sparse_q8(scale=-1.0),
               sparse_q8(ws=64)]
    assert refused == [_lib.MSPR_ERR_ARG] * len(refused)


def _on(dev, *shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device=dev)


def _calls(dev):
    def ints(*shape):
        return _on(dev, *shape, dtype=I32)

    def triplet():
        return ints(5, 2, 16, 64), _on(dev, 5, 2, 16, 4), _on(dev, 5, 2, 16, 4)

    q, pages = _on(dev, 3, 4, 256), _on(dev, 5, 2, 16, 256)
    bounds = _on(dev, 5, 2, 2, 256, dtype=torch.int8), _on(dev, 5, 2, dtype=torch.float32)
    prefixes, own = (ints(2, 3), ints(2), ints(3)), (ints(3, 4), ints(3))
    return {
        "mspr_sdpa_decode_paged_shared": lambda: paged.sdpa_decode_paged_shared(q, pages, pages, *prefixes, *own, 0.1),
        "mspr_sdpa_decode_paged_shared_q8": lambda: paged.sdpa_decode_paged_shared_q8(q, *triplet(), *triplet(), *prefixes, *own, 0.1),
        "mspr_page_bounds": lambda: paged.page_bounds(ints(3), pages, *bounds),
        "mspr_page_bounds_q8": lambda: paged.page_bounds(ints(3), triplet(), *bounds),
        "mspr_select_pages": lambda: paged.select_pages(q, *bounds, *own, 3, page_size=16),
        "mspr_sdpa_decode_paged_sparse": lambda: paged.sdpa_decode_paged_sparse(q, pages, pages, *bounds, *own, 0.1, 3),
        "mspr_sdpa_decode_paged_sparse_q8": lambda: paged.sdpa_decode_paged_sparse_q8(q, *triplet(), *triplet(), *bounds, *own, 0.1, 3),
    }


ENTRIES = ["mspr_sdpa_decode_paged_shared", "mspr_sdpa_decode_paged_shared_q8", "mspr_page_bounds", "mspr_page_bounds_q8", "mspr_select_pages",
           "mspr_sdpa_decode_paged_sparse", "mspr_sdpa_decode_paged_sparse_q8"]


@pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")
@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("current", [0, 1])
def test_a_call_is_launched_on_the_stream_of_its_operands_device(monkeypatch, entry, current):
    on, launched, real = [current], [], _lib.lib()

    @contextlib.contextmanager
    def device(d):
        on.append(d.index)
        yield
        on.pop()

    class Library:
        def __getattr__(self, name):
            if name.endswith("_bytes"):
                return getattr(real, name)
            return lambda *args: launched.append((name, on[-1], args[-1])) or 0

    monkeypatch.setattr(_lib, "lib", Library)
    monkeypatch.setattr(_lib, "ptr", lambda t: None)
    monkeypatch.setattr(_lib, "stream_ptr", lambda: f"stream of {on[-1]}")
    monkeypatch.setattr(torch.cuda, "current_device", lambda: on[-1])
    monkeypatch.setattr(torch.cuda, "device", device)
    with FakeTensorMode():
        _calls("cuda:1")[entry]()
    assert launched == [(entry, 1, "stream of 1")] and on == [current]


def test_operands_on_different_devices_are_refused():
    with FakeTensorMode():
        pages, q = _on("cuda:0", 5, 2, 16, 256), _on("cuda:0", 3, 4, 256)
        ints = lambda dev, *shape: _on(dev, *shape, dtype=I32)
        with pytest.raises(RuntimeError, match="same HIP device"):
            paged.sdpa_decode_paged_shared(q, pages, pages, ints("cuda:0", 2, 3), ints("cuda:0", 2), ints("cuda:1", 3), ints("cuda:0", 3, 4),
                                           ints("cuda:0", 3), 0.1)
        with pytest.raises(RuntimeError, match="same HIP device"):
            paged.select_pages(q, _on("cuda:0", 5, 2, 2, 256, dtype=torch.int8), _on("cuda:1", 5, 2, dtype=torch.float32), ints("cuda:0", 3, 4),
                               ints("cuda:0", 3), 3, page_size=16)


# ---------------------------------------------------------------------------------------------- tables, pages and a layer


class _Norm(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.weight, self.eps = torch.nn.Parameter(1 + 0.1 * torch.randn(256), requires_grad=False), 1e-6


class _Rope(torch.nn.Module):
    inv_freq, sections = torch.ones(32), (11, 11, 10)


class _Block(torch.nn.Module):
    def __init__(self, scale=0.0625):
        super().__init__()
        self.q_proj, self.k_proj = torch.nn.Linear(32, 4 * 512), torch.nn.Linear(32, 512)
        self.v_proj, self.o_proj = torch.nn.Linear(32, 512), torch.nn.Linear(4 * 256, 32)
        self.q_norm, self.k_norm, self.rope = _Norm(), _Norm(), _Rope()
        self.scale, self.num_attention_heads, self.num_key_value_heads = scale, 4, 2


def _cache(**kwargs):
    return paged.PagedKVCache(4, 2, page_size=16, device="cpu", dtype=torch.float16, **kwargs)


def _tables(**kwargs):
    return paged.PageTables(2, 4, page_size=16, max_tokens=64, device="cpu", **kwargs)


def test_tables_refuse_prefixes_they_have_no_place_for():
    assert _tables().prefixes is None and _tables().groups is None
    with pytest.raises(ValueError, match="no prefix"):
        _tables().continue_prefix(0, 0)
    tables = _tables(n_prefixes=2)
    assert [tuple(t.shape) for t in tables.prefixes] == [(2, 4), (2,), (4,)]
    for request, prefix in ((-1, 0), (2, 0), (0, 2), (0, -1)):
        with pytest.raises(ValueError, match="of these tables"):
            tables.continue_prefix(request, prefix)
    tables.continue_prefix(1, 1)
    assert tables.groups.tolist() == [-1, 1, -1, -1]
    tables.continue_prefix(1, None)
    assert tables.groups.tolist() == [-1] * 4
    for batch, n in ((2047, 2), (0, 1), (1, -1), (1, 2048)):
        with pytest.raises(ValueError, match="1 to 2048 together"):
            paged.PageTables(batch, 4, page_size=16, max_tokens=64, device="cpu", n_prefixes=n)


def test_tables_refuse_lengths_of_prefixes():
    for kwargs in (dict(max_prefix_tokens=16), dict(n_prefixes=1, max_prefix_tokens=0), dict(n_prefixes=1, max_prefix_tokens=65)):
        with pytest.raises(ValueError, match="max_prefix_tokens"):
            _tables(**kwargs)
    assert [tuple(t.shape) for t in _tables(n_prefixes=2, max_prefix_tokens=17).prefixes] == [(2, 2), (2,), (4,)]


def test_a_prefix_ends_with_its_pages(monkeypatch):
    """Rows behind ``max_prefix_tokens`` are seen by nobody, and positions count on from there."""
    tables = _tables(n_prefixes=2, max_prefix_tokens=20)
    ints = lambda *a: torch.tensor(a, dtype=I32)
    step = paged.PageStep(ints(5, 2, 40, 7), ints(3), ints(0, 2, 3, 3, 3), ints(3, 4, 5), ints(3, 4, 1), ints(4, 5, 2), ints(0, 0, 1), ints(0, 0, 0, 0))
    monkeypatch.setattr(paged, "page_step", lambda *a, **k: step)
    tables.tables.copy_(torch.arange(16, dtype=I32).reshape(4, 4))
    tables.continue_prefix(0, 0)
    tables.continue_prefix(1, 1)
    held = tables.prefix_tables
    got = tables.step(ints(2, 1, 0, 0), 3)
    assert got.positions.tolist() == [35, 36, 8] and tables.prefixes[0] is held and held.tolist() == [[8, 9], [12, 13]]


def test_positions_are_counted_from_the_prefix(monkeypatch):
    """(The step itself is stood in for.) Places that name no prefix, and rows of no request, are left as they are."""
    tables = _tables(n_prefixes=2)
    ints = lambda *a: torch.tensor(a, dtype=I32)
    lens = ints(5, 2, 40, 7)
    step = paged.PageStep(lens, ints(3), ints(0, 2, 3, 3, 3), ints(3, 4, -1, -1), ints(3, 4, 1, 0), ints(4, 5, 0, 0), ints(0, 0, 1, -1), ints(0, 0, 0, 0))
    monkeypatch.setattr(paged, "page_step", lambda *a, **k: step)
    for groups, want in (((0, 1, -1, -1), (43, 44, 8, 0)), ((-1, 2, 0, 0), (3, 4, 1, 0)), ((1, -(1 << 31), -1, -1), (10, 11, 1, 0)),
                         (((1 << 31) - 1, 0, 0, 0), (3, 4, 41, 0))):
        tables.groups.copy_(ints(*groups))
        got = tables.step(ints(2, 1, 0, 0), 4)
        assert got.positions.tolist() == list(want) and got.positions.dtype == I32
        assert got.requests.tolist() == [0, 0, -1, -1] and got.requests.dtype == I32
        assert got.visible is step.visible and tables.lens.tolist() == lens.tolist()
    plain = _tables()
    plain.lens = torch.zeros(4, dtype=I32)
    assert plain.step(ints(2, 1, 0, 0), 4) is step


@pytest.mark.parametrize("kwargs,message", [
    (dict(n_selected=0), "n_selected must be"),
    (dict(n_selected=4097), "n_selected must be"),
    (dict(n_selected=2), "n_selected must be"),
    (dict(n_selected=4, recent=0), "n_selected must be"),
    (dict(n_selected=4, bounds=False), "must have them"),
    (dict(n_selected=4, scale=-0.1), "not negative"),
])
def test_a_layer_refuses_a_selection(kwargs, message):
    cache, block = _cache(bounds=kwargs.pop("bounds", True)), _Block(kwargs.pop("scale", 0.0625))
    with pytest.raises(ValueError, match=message):
        paged.PagedAttention(block, cache, **kwargs)


def test_a_step_that_cannot_be_attended_writes_nothing(monkeypatch):
    """What does not fit is refused in front of the append."""
    layer = paged.PagedAttention(_Block(), _cache(bounds=True), n_selected=3)
    monkeypatch.setattr(layer.cache, "append", lambda *a, **k: pytest.fail("appended"))
    n = torch.zeros(5, dtype=I32)
    step, x = paged.PageStep(n, n, n, n, n, n, n, n), torch.randn(5, 32)
    with pytest.raises(ValueError, match="continue no prefix"):
        layer(x, step, _tables(n_prefixes=1))
    wide = _tables()
    wide.tables = torch.zeros(2, 32769, dtype=I32)
    with pytest.raises(ValueError, match="at most 32768 pages"):
        layer(x, step, wide)
    with pytest.raises(ValueError, match="continue no prefix"):
        layer.cache.attend(x, None, None, 0.1, prefixes=(n, n, n), selected=(3, 1, 2))
    with pytest.raises(ValueError, match="without bounds"):
        _cache().attend(x, None, None, 0.1, selected=(3, 1, 2))


def test_what_a_layer_asks_of_its_cache(monkeypatch):
    layer, asked = paged.PagedAttention(_Block(), _cache(bounds=True), n_selected=4, first=0, recent=3), []
    monkeypatch.setattr(layer.cache, "append", lambda q, *a, **k: q.detach().contiguous())
    monkeypatch.setattr(layer.cache, "attend", lambda q, *a, **k: asked.append((len(q), k)) or torch.tanh(q.detach()))
    n = torch.zeros(4100, dtype=I32)
    step, x = paged.PageStep(n, n, n, n, n, n, n, n), torch.randn(4100, 32)
    with torch.no_grad():
        layer(x, step, _tables())
        assert [a[0] for a in asked] == [2048, 2048, 4] and all(a[1]["selected"] == (4, 0, 3) and "prefixes" not in a[1] for a in asked)
        del asked[:]
        layer(x, step, _tables(), dense=True)
        assert [a[0] for a in asked] == [4100] and set(asked[0][1]) == {"requests"}
        del asked[:]
        tables = _tables(n_prefixes=1)
        layer(x, step, tables, dense=True)
        assert [a[0] for a in asked] == [2048, 2048, 4] and all(a[1]["prefixes"][2] is tables.groups and "selected" not in a[1] for a in asked)
    # a backward pass is refused as without prefixes
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        layer(x, step, tables, dense=True).sum().backward()
