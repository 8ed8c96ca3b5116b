"""What the operators of a paged cache refuse, before anything is launched (CPU)."""

import contextlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from moespresso_amd import _lib
from moespresso_amd.runtime.qwen import paged

I32 = torch.int32


def _ints(*shape):
    return torch.zeros(shape, dtype=I32)


def _step(lens=_ints(3), new=_ints(3), tables=_ints(3, 5), free=_ints(20), head=_ints(1), page_size=16, n_rows=3):
    return paged.page_step(lens, new, tables, free, head, page_size=page_size, n_rows=n_rows)


@pytest.mark.parametrize("change,message", [
    (dict(page_size=24), "power of two"),
    (dict(page_size=8), "power of two"),
    (dict(page_size=-16), "power of two"),
    (dict(lens=_ints(0), new=_ints(0), tables=_ints(0, 5)), "1 to 2048 requests"),
    (dict(lens=_ints(2049), new=_ints(2049), tables=_ints(2049, 5)), "1 to 2048 requests"),
    (dict(lens=torch.zeros(3, dtype=torch.int64)), "lens must be a contiguous int32"),
    (dict(new=_ints(4)), "new_lens must be"),
    (dict(tables=_ints(4, 5)), "tables must be"),
    (dict(tables=_ints(5, 3).t()), "tables must be a contiguous"),
    (dict(tables=_ints(3, 0)), "at least one page"),
    (dict(free=_ints(0)), "at least one page"),
    (dict(head=_ints(2)), "head must be"),
    (dict(n_rows=-1), "must not be negative"),
    (dict(lens=_ints(3, 1)), "lens must be"),
])
def test_step_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        _step(**change)


def _rope_args(T=3, dtype=torch.float32, **change):
    a = dict(q=torch.zeros(T, 4, 256, dtype=dtype), k=torch.zeros(T, 2, 256, dtype=dtype), q_weight=torch.zeros(256, dtype=dtype),
             k_weight=torch.zeros(256, dtype=dtype), positions=_ints(T), inv_freq=torch.zeros(32))
    sections = change.pop("sections", None)
    a.update(change)
    return tuple(a.values()), sections


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(3, 4, 128)), "q must be"),
    (dict(q=torch.zeros(3, 1024)), "q must be"),
    (dict(q=torch.zeros(3, 4, 256, dtype=torch.float64)), "float32/float16/bfloat16"),
    (dict(k=torch.zeros(2, 2, 256)), "number of tokens"),
    (dict(k=torch.zeros(3, 2, 256).half()), "share a float32"),
    (dict(k=torch.zeros(3, 0, 256)), "at least one head"),
    (dict(q_weight=torch.zeros(128)), "q_weight must be"),
    (dict(k_weight=torch.zeros(256).half()), "k_weight must be"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions must be"),
    (dict(positions=_ints(3, 3)), "positions must be"),
    (dict(positions=_ints(2)), "positions must be"),
    (dict(sections=(11, 11, 10)), "positions must be"),
    (dict(positions=_ints(3, 3), sections=(11, 11, 11)), "sections must be"),
    (dict(positions=_ints(3, 3), sections=(12, 20)), "sections must be"),
    (dict(positions=_ints(3, 3), sections=(34, -1, -1)), "sections must be"),
    (dict(positions=_ints(3, 3), sections=(10, 12, 10)), "more frequencies than their turns"),
    (dict(positions=_ints(3, 3), sections=(10, 11, 11)), "more frequencies than their turns"),
    (dict(inv_freq=torch.zeros(20)), "multiple of 16"),
    (dict(inv_freq=torch.zeros(136)), "multiple of 16"),
    (dict(inv_freq=torch.zeros(0)), "multiple of 16"),
    (dict(inv_freq=torch.zeros(32).half()), "inv_freq must be"),
])
def test_norm_and_rope_refuse(change, message):
    args, sections = _rope_args(**change)
    with pytest.raises(ValueError, match=message):
        paged.qk_norm_rope(*args, sections=sections)


def _rows(n=5, heads=2, page=16, dtype=torch.float16):
    return torch.zeros(n, heads, page, 256, dtype=dtype)


def _codes(n=5, heads=2, page=16, dtype=torch.float32):
    return (torch.zeros(n, heads, page, 64, dtype=I32), torch.zeros(n, heads, page, 4, dtype=dtype),
            torch.zeros(n, heads, page, 4, dtype=dtype))


@pytest.mark.parametrize("change,message", [
    (dict(v=torch.zeros(3, 2, 256).half()), "share a float32"),
    (dict(v=torch.zeros(2, 2, 256)), "number of tokens"),
    (dict(v=torch.zeros(3, 1, 256)), "number of KV heads"),
    (dict(slots=_ints(2)), "slots must be"),
    (dict(slots=torch.zeros(3, dtype=torch.int64)), "slots must be"),
    (dict(keys=_rows(heads=1), values=_rows(heads=1)), "number of KV heads"),
    (dict(keys=_rows(dtype=torch.float32), values=_rows(dtype=torch.float32)), "float16 or bfloat16 pages"),
    (dict(keys=_rows(), values=_rows(dtype=torch.bfloat16)), "share a shape and a dtype"),
    (dict(keys=_rows(), values=_rows(n=4)), "share a shape and a dtype"),
    (dict(keys=_rows(page=24), values=_rows(page=24)), "power of two"),
    (dict(keys=_rows(n=0), values=_rows(n=0)), "at least one page"),
    (dict(keys=_rows(), values=_codes()), "must both be"),
    (dict(keys=_codes()[:2], values=_codes()), "must be .codes, scales, biases"),
    (dict(keys=_codes(dtype=torch.float16), values=_codes(dtype=torch.float16)), "dtype of q"),
    (dict(keys=_codes(), values=_codes(page=32)), "share a shape"),
    (dict(keys=_rows().transpose(1, 2), values=_rows().transpose(1, 2)), "power of two|contiguous"),
])
def test_append_refuses(change, message):
    args = dict(v=torch.zeros(3, 2, 256), slots=_ints(3), keys=_rows(), values=_rows())
    args.update(change)
    (q, k, *rest), _ = _rope_args()
    with pytest.raises(ValueError, match=message):
        paged.qk_norm_rope_append(q, k, args["v"], *rest, args["slots"], args["keys"], args["values"])


def test_append_refuses_pages_of_another_16_bit_type():
    (q, k, *rest), _ = _rope_args(dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="dtype of 16-bit rows"):
        paged.qk_norm_rope_append(q, k, torch.zeros(3, 2, 256).bfloat16(), *rest, _ints(3), _rows(), _rows())


@pytest.mark.parametrize("change,message", [
    (dict(queries=torch.zeros(3, 4, 128).half()), "queries must be"),
    (dict(queries=torch.zeros(3, 4, 1, 256).half()), "queries must be"),
    (dict(queries=torch.zeros(3, 3, 256).half()), "multiple"),
    (dict(queries=torch.zeros(3, 34, 256).half()), "multiple"),
    (dict(queries=torch.zeros(3, 4, 256)), "dtype of queries"),
    (dict(tables=_ints(2, 4)), "table of its own"),
    (dict(tables=_ints(12)), "tables must be"),
    (dict(tables=_ints(3, 0)), "tables must be"),
    (dict(lens=_ints(2)), "lens must be"),
    (dict(lens=torch.zeros(3, dtype=torch.int64)), "lens must be"),
    (dict(requests=_ints(2)), "requests must be"),
    (dict(requests=_ints(3), tables=_ints(0, 4)), "tables must be"),
    (dict(keys=_codes(), values=_codes()), "8-bit ones"),
])
def test_decode_refuses(change, message):
    a = dict(queries=torch.zeros(3, 4, 256).half(), keys=_rows(), values=_rows(), tables=_ints(3, 4), lens=_ints(3), requests=None)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        paged.sdpa_decode_paged(a["queries"], a["keys"], a["values"], a["tables"], a["lens"], 0.1, requests=a["requests"])


def test_8_bit_decode_refuses():
    q, t, n = torch.zeros(3, 4, 256), _ints(3, 4), _ints(3)
    with pytest.raises(ValueError, match="group_size=64, bits=8"):
        paged.sdpa_decode_paged_q8(q, *_codes(), *_codes(), t, n, 0.1, bits=4)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        paged.sdpa_decode_paged_q8(q.double(), *_codes(), *_codes(), t, n, 0.1)
    wide = torch.zeros(5, 2, 16, 256, dtype=torch.uint8)
    with pytest.raises(ValueError, match="uint32 pages"):
        paged.sdpa_decode_paged_q8(q, wide, *_codes()[1:], wide, *_codes()[1:], t, n, 0.1)


def test_host_tensors_are_refused():
    args, _ = _rope_args()
    for call in (_step, lambda: paged.qk_norm_rope(*args),
                 lambda: paged.sdpa_decode_paged(torch.zeros(3, 4, 256).half(), _rows(), _rows(), _ints(3, 4), _ints(3), 0.1)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


@pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")
def test_the_library_refuses_what_its_kernels_do_not_take():
    """The same through the C-ABI, with pointers that are never followed."""
    lib, p = _lib.lib(), _lib.c_void_p(4096)

    def step(batch=3, width=5, pages=20, page=16, rows=3, lens_out=8192):
        return lib.mspr_page_step(p, p, p, p, p, batch, width, pages, page, rows, lens_out, 8192, p, p, p, p, p, p, None)

    def decode(hq=4, hkv=2, dim=256, pages=5, page=16, tables=3, width=4, q=4096, ws=1 << 40, requests=None, batch=3):
        return lib.mspr_sdpa_decode_paged(q, p, p, 1, p, p, requests, batch, hq, hkv, dim, pages, page, tables, width, 0.1, p, p,
                                          ws, None)

    def rope(tokens=3, hq=4, hkv=2, dim=256, stride=1024, axes=1, height=0, width=0, rotary=64, dtype=0):
        return lib.mspr_qk_norm_rope(p, p, p, p, dtype, tokens, hq, hkv, dim, stride, 256, 512, 256, p, axes, height, width, p,
                                     rotary, 1e-6, p, p, None)

    refused = [step(batch=0), step(batch=2049), step(page=24), step(page=0), step(width=0), step(pages=0), step(rows=-1),
               step(pages=1 << 28), step(width=1 << 27), step(lens_out=4096),
               decode(hq=3), decode(hq=34), decode(hkv=0), decode(dim=128), decode(pages=0), decode(page=8), decode(tables=2),
               decode(width=0), decode(q=4104), decode(ws=64), decode(pages=1 << 28), decode(batch=0), decode(batch=65536, tables=65536),
               decode(requests=4096, tables=0),
               rope(tokens=0), rope(dim=128), rope(stride=1026), rope(axes=2), rope(rotary=24), rope(rotary=272), rope(rotary=63),
               rope(axes=3, height=12), rope(axes=3, width=11), rope(dtype=3), rope(hq=0)]
    assert refused == [_lib.MSPR_ERR_ARG] * len(refused)


def _on(dev, *shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device=dev)


def _calls(dev):
    def ints(*shape):
        return _on(dev, *shape, dtype=I32)

    def triplet():
        return ints(5, 2, 16, 64), _on(dev, 5, 2, 16, 4), _on(dev, 5, 2, 16, 4)

    q, k, w, inv = _on(dev, 3, 4, 256), _on(dev, 3, 2, 256), _on(dev, 256), _on(dev, 32, dtype=torch.float32)
    pages = _on(dev, 5, 2, 16, 256)
    return {
        "mspr_page_step": lambda: paged.page_step(ints(3), ints(3), ints(3, 5), ints(20), ints(1), page_size=16, n_rows=3),
        "mspr_qk_norm_rope": lambda: paged.qk_norm_rope(q, k, w, w, ints(3), inv),
        "mspr_qk_norm_rope_append": lambda: paged.qk_norm_rope_append(q, k, k, w, w, ints(3), inv, ints(3), pages, pages),
        "mspr_qk_norm_rope_append_q8": lambda: paged.qk_norm_rope_append(q, k, k, w, w, ints(3), inv, ints(3), triplet(), triplet()),
        "mspr_sdpa_decode_paged": lambda: paged.sdpa_decode_paged(q, pages, pages, ints(3, 4), ints(3), 0.1),
        "mspr_sdpa_decode_paged_q8": lambda: paged.sdpa_decode_paged_q8(q, *triplet(), *triplet(), ints(3, 4), ints(3), 0.1),
    }


@pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")
@pytest.mark.parametrize("entry", ["mspr_page_step", "mspr_qk_norm_rope", "mspr_qk_norm_rope_append", "mspr_qk_norm_rope_append_q8",
                                   "mspr_sdpa_decode_paged", "mspr_sdpa_decode_paged_q8"])
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
    with FakeTensorMode(), pytest.raises(RuntimeError, match="same HIP device"):
        paged.page_step(_on("cuda:0", 3, dtype=I32), _on("cuda:1", 3, dtype=I32), _on("cuda:0", 3, 5, dtype=I32),
                        _on("cuda:0", 20, dtype=I32), _on("cuda:0", 1, dtype=I32), page_size=16, n_rows=3)


def test_norms_of_two_eps_are_refused():
    class Norm:
        def __init__(self, eps):
            self.eps = eps

    class Block:
        q_norm, k_norm = Norm(1e-6), Norm(1e-5)

    with pytest.raises(ValueError, match="share an eps"):
        paged.PagedAttention(Block(), None)
