"""Scratch that a caller hands over: memory of the host or of another device, and tensors that are not as many bytes one behind the other
as they have elements, are refused before anything is launched (CPU: fake tensors, a recorded library)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from moespresso_amd import _lib
from moespresso_amd.runtime.deepseek_v4 import decode_attention_kernel as dak
from moespresso_amd.runtime.deepseek_v4 import indexed_attention_kernel as iak
from moespresso_amd.runtime.qwen import kquant, paged

pytestmark = pytest.mark.skipif(not _lib.library_available(), reason="the library is not built")


def _on(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda:0")


def _f16(*shape):
    return _on(*shape, dtype=torch.float16)


def _f32(*shape):
    return _on(*shape, dtype=torch.float32)


def _i32(*shape):
    return _on(*shape, dtype=torch.int32)


def _triplet(*shape):
    return _i32(*shape, 64), _f32(*shape, 4), _f32(*shape, 4)


def _calls():
    q, pages, side = _on(3, 4, 256), _on(5, 2, 16, 256), _triplet(5, 2, 16)
    bounds = _on(5, 2, 2, 256, dtype=torch.int8), _f32(5, 2)
    prefixes, own = (_i32(2, 3), _i32(2), _i32(3)), (_i32(3, 4), _i32(3))
    cache = _triplet(1, 2, 40)
    q8_0 = _on(1, 2, 40, 256, dtype=torch.int8), _f16(1, 2, 40, 8)
    return {
        "sparse_mla_decode": lambda ws: iak.sparse_mla_decode(_on(1, 64, 576), _on(1, 900, 576), _i32(1, 40), scale=0.1, workspace=ws),
        "fused_decode_sdpa": lambda ws: dak.fused_decode_sdpa(_f16(64, 512), _f16(128, 512), _f16(512), _f16(300, 512), _i32(64), _f16(64),
                                                             _f32(32), _i32(2), scale=0.1, workspace=ws),
        "sdpa_decode_q8": lambda ws: kquant.sdpa_decode_q8(_f32(1, 4, 1, 256), *cache, *cache, 0.1, workspace=ws),
        "sdpa_decode_q8_0": lambda ws: kquant.sdpa_decode_q8_0(_f32(1, 4, 256), *q8_0, *q8_0, 0.1, workspace=ws),
        "sdpa_fa_prefill_q8": lambda ws: kquant.sdpa_fa_prefill_q8(_f32(1, 4, 8, 256), *cache, *cache, _f32(1, 2, 8, 256), _f32(1, 2, 8, 256),
                                                                   0.1, workspace=ws),
        "flash_prefill": lambda ws: kquant.flash_prefill(_on(1, 4, 8, 256), _on(1, 2, 40, 256), _on(1, 2, 40, 256), 0.1, past_len=32,
                                                         workspace=ws),
        "sdpa_decode_paged": lambda ws: paged.sdpa_decode_paged(q, pages, pages, *own, 0.1, workspace=ws),
        "sdpa_decode_paged_q8": lambda ws: paged.sdpa_decode_paged_q8(q, *side, *side, *own, 0.1, workspace=ws),
        "sdpa_decode_paged_shared": lambda ws: paged.sdpa_decode_paged_shared(q, pages, pages, *prefixes, *own, 0.1, workspace=ws),
        "sdpa_decode_paged_shared_q8": lambda ws: paged.sdpa_decode_paged_shared_q8(q, *side, *side, *prefixes, *own, 0.1, workspace=ws),
        "select_pages": lambda ws: paged.select_pages(q, *bounds, *own, 3, page_size=16, workspace=ws),
        "sdpa_decode_paged_sparse": lambda ws: paged.sdpa_decode_paged_sparse(q, pages, pages, *bounds, *own, 0.1, 3, workspace=ws),
        "sdpa_decode_paged_sparse_q8": lambda ws: paged.sdpa_decode_paged_sparse_q8(q, *side, *side, *bounds, *own, 0.1, 3, workspace=ws),
    }


OPERATORS = ["sparse_mla_decode", "fused_decode_sdpa", "sdpa_decode_q8", "sdpa_decode_q8_0", "sdpa_fa_prefill_q8", "flash_prefill",
             "sdpa_decode_paged", "sdpa_decode_paged_q8", "sdpa_decode_paged_shared", "sdpa_decode_paged_shared_q8", "select_pages",
             "sdpa_decode_paged_sparse", "sdpa_decode_paged_sparse_q8"]


@pytest.fixture
def launched(monkeypatch):
    """Sizes of the scratch of what was launched, the last argument but the stream."""
    real, sizes = _lib.lib(), []

    class Library:
        def __getattr__(self, name):
            if name.endswith("_bytes"):
                return getattr(real, name)
            return lambda *args: sizes.append(args[-2]) or 0

    monkeypatch.setattr(_lib, "lib", Library)
    monkeypatch.setattr(_lib, "ptr", lambda t: None)
    monkeypatch.setattr(_lib, "stream_ptr", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    return sizes


@pytest.mark.parametrize("operator", OPERATORS)
def test_scratch_that_is_not_the_devices_own_is_refused(launched, operator):
    with FakeTensorMode():
        call = _calls()[operator]
        for ws in (torch.empty(1 << 20), torch.empty(1 << 20, device="cuda:1"), _f32(1).expand(1 << 20), _f32(1 << 10, 1 << 10).t(), 1 << 20):
            with pytest.raises(ValueError, match="workspace must be a contiguous tensor on the device"):
                call(ws)
    assert launched == []


@pytest.mark.parametrize("operator", OPERATORS)
def test_scratch_counts_as_the_bytes_that_it_has(launched, operator):
    with FakeTensorMode():
        for ws in (_f32(1 << 20), _f16(1 << 20), _on(1 << 20, dtype=torch.uint8)):
            _calls()[operator](ws)
    assert launched == [4 << 20, 2 << 20, 1 << 20]
