"""Serving many requests from a paged KV cache of the Qwen/Ornith full-attention layers on MI355X.

The reference serves one sequence a cache (mlx_lm's caches, ``runtime/qwen/full_attention.py:315,352-356``); this module
is an extension for a server of many. The rows of all requests lie in pages of one pool per layer, ``[n_pages, Hkv,
page_size, 256]`` for keys and for values (16-bit rows, or affine 8-bit triplets as in ``kquant``), and a table per request,
shared by the layers, names its pages. ``slot = page * page_size + row in the page``; page sizes are powers of two from 16 on.

A step of a server, every part of it enqueued without waiting for the device:

* ``page_step`` takes and gives back pages and names a slot for every new row,
* ``qk_norm_rope_append`` (each layer) normalises and rotates queries and keys and writes keys and values to their slots,
* ``sdpa_decode_paged`` / ``sdpa_decode_paged_q8`` (each layer) attends every new query over its request's pages,
* in its place, for requests that continue a prefix they share (a system prompt, a document): ``sdpa_decode_paged_shared`` and
  ``_q8``, which read the rows of a prefix once for all of them,
* or, for long requests, ``page_bounds`` (each layer, behind the append) and ``sdpa_decode_paged_sparse`` and ``_q8``, which attend
  the pages alone that ``select_pages`` finds to matter most.

``PageTables``, ``PagedKVCache`` and ``PagedAttention`` hold what such a server keeps: the tables (and the prefixes), a layer's
pages (and their bounds), a layer.
"""

from __future__ import annotations

import inspect
from ctypes import c_int64
from typing import NamedTuple

import torch

from moespresso_amd import _lib

_HEAD_DIM = 256
_GROUP = 64
MAX_REQUESTS = 2048  # requests of one page_step
MAX_SHARED = 2048    # queries, and prefixes, of one call over shared prefixes
MAX_SELECTED = 4096      # pages that a query may select
MAX_TABLE_PAGES = 32768  # pages of a request of which some are selected
_SELECTION_BYTES = 256 << 20  # scratch of one selection of a layer, about (more than a query's own: a query a call)


def _check_page_size(page_size: int):
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two from 16 on")


def _check_ints(name, t, shape):
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)}")


class PageStep(NamedTuple):
    """What a step needs: lengths and stack top behind it, and per row of its ragged batch where the row goes."""

    lens: torch.Tensor       # int32 [B], tokens of every request with this step's (0: ended)
    head: torch.Tensor       # int32 [1], the first free page on the stack
    starts: torch.Tensor     # int32 [B + 1], first row of every request, and the end
    slots: torch.Tensor      # int32 [n_rows], -1: none
    positions: torch.Tensor  # int32 [n_rows]
    visible: torch.Tensor    # int32 [n_rows], rows of the request up to this one (0 without a slot)
    requests: torch.Tensor   # int32 [n_rows], -1 behind the last
    counts: torch.Tensor     # int32 [4]: rows asked for, of them without a slot, pages taken, pages given back


def page_step(lens, new_lens, tables, free_pages, head, *, page_size: int, n_rows: int) -> PageStep:
    """Tables and slots of a step in which request ``b`` of ``lens[b]`` tokens gets ``new_lens[b]`` rows.

    A negative ``new_lens[b]`` ends the request: its pages go back to the stack, before any are taken. Rows for which no page
    is left (or no room in the table) get slot -1 and are not counted in the lengths; ``counts[1]`` says how many they are.

    Args:
        lens, new_lens: int32 ``[B]``, at most 2048 requests. Lengths as the last step left them.
        tables: int32 ``[B, P]``, the pages of every request in order, updated in place.
        free_pages: int32 ``[n_pages]``, a stack of the pool's pages, free from entry ``head`` on, updated in place.
        head: int32 ``[1]``.
        n_rows: rows of the step's ragged batch, the sum of the positive ``new_lens`` or more; the rows behind the last
            request belong to none. Rows asked for behind ``n_rows`` are not part of the step.
    """
    done = _lib.dispatch.page_step(lens, new_lens, tables, free_pages, head, page_size, n_rows)
    if done is not None:
        return tuple.__new__(PageStep, done)
    page_size, n_rows = int(page_size), int(n_rows)
    _check_page_size(page_size)
    if lens.ndim != 1 or tables.ndim != 2 or free_pages.ndim != 1:
        raise ValueError("lens must be [B], tables [B, P] and free_pages [n_pages]")
    B, width, n_pages = int(lens.shape[0]), int(tables.shape[1]), int(free_pages.shape[0])
    if not 1 <= B <= MAX_REQUESTS:
        raise ValueError(f"page_step takes 1 to {MAX_REQUESTS} requests")
    if width < 1 or n_pages < 1 or n_rows < 0:
        raise ValueError("the tables and the pool must hold at least one page, n_rows must not be negative")
    _check_ints("lens", lens, (B,))
    _check_ints("new_lens", new_lens, (B,))
    _check_ints("tables", tables, (B, width))
    _check_ints("free_pages", free_pages, (n_pages,))
    _check_ints("head", head, (1,))
    dev = _lib.require_device(lens, new_lens, tables, free_pages, head)
    out = PageStep(*(torch.empty((n,), dtype=torch.int32, device=dev) for n in (B, 1, B + 1, n_rows, n_rows, n_rows, n_rows, 4)))
    _lib.check(_lib.launch(
        dev, "mspr_page_step", _lib.ptr(lens), _lib.ptr(new_lens), _lib.ptr(tables), _lib.ptr(free_pages), _lib.ptr(head),
        B, width, n_pages, page_size, n_rows, *(_lib.ptr(t) for t in out)), "page_step")
    return out


# ---------------------------------------------------------------------------------------------- norm, rope, append


def _check_rows(name, t, tokens=None, dtype=None):
    if t.ndim != 3 or int(t.shape[2]) != _HEAD_DIM:
        raise ValueError(f"{name} must be [T, heads, 256]")
    if t.dtype not in _lib.DTYPE_CODE or (dtype is not None and t.dtype != dtype):
        raise ValueError("q, k and v must share a float32/float16/bfloat16 dtype")
    if tokens is not None and int(t.shape[0]) != tokens:
        raise ValueError("q, k and v disagree on the number of tokens")
    if int(t.shape[1]) < 1:
        raise ValueError(f"{name} must have at least one head")


def _rows(t):
    """``t`` itself where its rows are dense and 16-byte aligned (a view of a projection's output is), else a copy."""
    unit = 16 // t.element_size()
    if t.stride(2) == 1 and all(n % unit == 0 for n in (t.stride(0), t.stride(1), t.storage_offset())):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _aligned(t):
    return t if t.storage_offset() * t.element_size() % 16 == 0 else t.clone()


def _check_rope(q, q_weight, k_weight, positions, inv_freq, sections):
    """Number of position axes, and the frequencies of the height and width axes."""
    T = int(q.shape[0])
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.dtype != q.dtype or tuple(w.shape) != (_HEAD_DIM,) or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [256] tensor of the dtype of q")
    if inv_freq.dtype != torch.float32 or inv_freq.ndim != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float32 [rotary_dim / 2] tensor")
    half = int(inv_freq.shape[0])
    if half < 8 or half > _HEAD_DIM // 2 or half % 8:
        raise ValueError("the rotary width must be a multiple of 16 up to 256")
    if sections is None:
        _check_ints("positions", positions, (T,))
        return 1, 0, 0
    if len(sections) != 3 or any(int(s) < 0 for s in sections) or sum(int(s) for s in sections) != half:
        raise ValueError("sections must be three counts of frequencies that sum to those of inv_freq")
    _check_ints("positions", positions, (3, T))
    height, width = int(sections[1]), int(sections[2])
    if 3 * height > half + 1 or 3 * width > half:
        raise ValueError("the height and width axes have more frequencies than their turns")
    return 3, height, width


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, *, eps: float = 1e-6, sections=None):
    """RMS norm of every query and key head and the rotary position of its first channels, in one pass.

    The sequence ``q_norm``, ``k_norm``, ``rope`` of the reference's attention block (full_attention.py:278-315), in float32
    throughout (angles in 64 bits) and rounded once. Channels ``i`` and ``i + rotary_dim / 2`` rotate together by
    ``position * inv_freq[i]``.

    Args:
        q: ``[T, Hq, 256]``, k: ``[T, Hkv, 256]``, float32, float16 or bfloat16. Views with any token and head stride are
            read in place (queries beside their output gate, heads of one fused projection).
        q_weight, k_weight: ``[256]`` of the same dtype, multiplied as they are.
        positions: int32 ``[T]``, or ``[3, T]`` (time, height, width) with ``sections``.
        inv_freq: float32 ``[rotary_dim / 2]``, rotary_dim a multiple of 16 up to 256.
        sections: frequencies of the three axes; they are dealt in turn (frequency ``i`` to axis ``i % 3`` while that has
            any left, else to time).

    Returns:
        ``(q, k)`` dense, of the same shapes and dtype.
    """
    done = _lib.dispatch.qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps, sections)
    if done is not None:
        return done
    _check_rows("q", q)
    T = int(q.shape[0])
    _check_rows("k", k, T, q.dtype)
    axes, height, width = _check_rope(q, q_weight, k_weight, positions, inv_freq, sections)
    dev = _lib.require_device(q, k, q_weight, k_weight, positions, inv_freq)
    q_out = torch.empty(tuple(q.shape), dtype=q.dtype, device=dev)
    k_out = torch.empty(tuple(k.shape), dtype=k.dtype, device=dev)
    if T == 0:
        return q_out, k_out
    qr, kr, qw, kw = _rows(q), _rows(k), _aligned(q_weight), _aligned(k_weight)
    _lib.check(_lib.launch(
        dev, "mspr_qk_norm_rope", _lib.ptr(qr), _lib.ptr(kr), _lib.ptr(qw), _lib.ptr(kw), _lib.DTYPE_CODE[q.dtype], T,
        int(q.shape[1]), int(k.shape[1]), _HEAD_DIM, qr.stride(0), qr.stride(1), kr.stride(0), kr.stride(1),
        _lib.ptr(positions), axes, height, width, _lib.ptr(inv_freq), 2 * int(inv_freq.shape[0]), float(eps),
        _lib.ptr(q_out), _lib.ptr(k_out)), "qk_norm_rope")
    return q_out, k_out


def _check_pages(keys, values):
    """(pages, KV heads, page size) of the pages of one layer: two 16-bit tensors, or two affine 8-bit triplets."""
    sides = (("keys", keys), ("values", values))
    if torch.is_tensor(keys) != torch.is_tensor(values):
        raise ValueError("keys and values must both be 16-bit pages or both be (codes, scales, biases)")
    if torch.is_tensor(keys):
        for name, t in sides:
            if t.ndim != 4 or int(t.shape[3]) != _HEAD_DIM or t.dtype not in (torch.float16, torch.bfloat16):
                raise ValueError(f"{name} must be float16 or bfloat16 pages [n_pages, Hkv, page_size, 256]")
        if keys.shape != values.shape or keys.dtype != values.dtype:
            raise ValueError("keys and values must share a shape and a dtype")
        parts, shape = (keys, values), keys.shape
    else:
        for name, side in sides:
            if len(side) != 3:
                raise ValueError(f"{name} must be (codes, scales, biases)")
            wq, scales, biases = side
            if wq.ndim != 4 or wq.dtype not in (torch.uint32, torch.int32) or int(wq.shape[3]) != _HEAD_DIM // 4:
                raise ValueError(f"{name} codes must be uint32 pages [n_pages, Hkv, page_size, 64]")
            if scales.ndim != 4 or tuple(scales.shape) != tuple(wq.shape[:3]) + (_HEAD_DIM // _GROUP,) or \
                    biases.shape != scales.shape:
                raise ValueError(f"{name} scales and biases must be [n_pages, Hkv, page_size, 4] (group_size=64)")
            if scales.dtype not in _lib.DTYPE_CODE or biases.dtype != scales.dtype:
                raise ValueError(f"{name} scales and biases must share a float32/float16/bfloat16 dtype")
        if keys[0].shape != values[0].shape or keys[1].dtype != values[1].dtype:
            raise ValueError("keys and values must share a shape and a dtype")
        parts, shape = (*keys, *values), keys[0].shape
    if not all(t.is_contiguous() and t.storage_offset() * t.element_size() % 16 == 0 for t in parts):
        raise ValueError("pages must be contiguous and 16-byte aligned")
    n_pages, heads, page_size = (int(n) for n in shape[:3])
    _check_page_size(page_size)
    if n_pages < 1 or heads < 1:
        raise ValueError("the pool must hold at least one page of one head")
    return n_pages, heads, page_size


def qk_norm_rope_append(q, k, v, q_weight, k_weight, positions, inv_freq, slots, keys, values, *, eps: float = 1e-6,
                        sections=None):
    """``qk_norm_rope`` whose keys go, with the values, straight into their slots of a layer's pages.

    Args:
        q, k, q_weight, k_weight, positions, inv_freq, eps, sections: as for ``qk_norm_rope``; v: ``[T, Hkv, 256]``, strided
            like them.
        slots: int32 ``[T]``, distinct; rows with a negative slot (or one that is not in the pool) are not written.
        keys, values: pages ``[n_pages, Hkv, page_size, 256]`` of the dtype of ``q`` (float16 or bfloat16 for float32 rows),
            or ``(codes, scales, biases)`` triplets with scales of the dtype of ``q``; written in place. The 8-bit rows are
            byte for byte what ``kquant.quantize`` makes of the keys of ``qk_norm_rope``.

    Returns:
        the queries, dense ``[T, Hq, 256]``.
    """
    out = _lib.dispatch.qk_norm_rope_append(q, k, v, q_weight, k_weight, positions, inv_freq, slots, keys, values, eps, sections)
    if out is not None:
        return out
    _check_rows("q", q)
    T = int(q.shape[0])
    _check_rows("k", k, T, q.dtype)
    _check_rows("v", v, T, q.dtype)
    axes, height, width = _check_rope(q, q_weight, k_weight, positions, inv_freq, sections)
    n_pages, heads, page_size = _check_pages(keys, values)
    if int(k.shape[1]) != heads or int(v.shape[1]) != heads:
        raise ValueError("k, v and the pages disagree on the number of KV heads")
    _check_ints("slots", slots, (T,))
    coded = not torch.is_tensor(keys)
    kind = keys[1].dtype if coded else keys.dtype
    if kind != q.dtype and (coded or q.dtype != torch.float32):
        raise ValueError("scales must have the dtype of q" if coded else "pages must have the dtype of 16-bit rows")
    parts = (*keys, *values) if coded else (keys, values)
    dev = _lib.require_device(q, k, v, q_weight, k_weight, positions, inv_freq, slots, *parts)
    out = torch.empty(tuple(q.shape), dtype=q.dtype, device=dev)
    if T == 0:
        return out
    qr, kr, vr, qw, kw = _rows(q), _rows(k), _rows(v), _aligned(q_weight), _aligned(k_weight)
    strides = (c_int64 * 6)(*(s for t in (qr, kr, vr) for s in t.stride()[:2]))
    front = (_lib.ptr(qr), _lib.ptr(kr), _lib.ptr(vr), _lib.ptr(qw), _lib.ptr(kw), _lib.DTYPE_CODE[q.dtype], T, int(q.shape[1]),
             heads, _HEAD_DIM, strides, _lib.ptr(positions), axes, height, width, _lib.ptr(inv_freq),
             2 * int(inv_freq.shape[0]), float(eps), _lib.ptr(slots), n_pages, page_size)
    if coded:
        rc = _lib.launch(dev, "mspr_qk_norm_rope_append_q8", *front, *(_lib.ptr(t) for t in parts), _lib.ptr(out))
    else:
        rc = _lib.launch(dev, "mspr_qk_norm_rope_append", *front, _lib.DTYPE_CODE[kind], *(_lib.ptr(t) for t in parts), _lib.ptr(out))
    _lib.check(rc, "qk_norm_rope_append")
    return out


# ---------------------------------------------------------------------------------------------- attention


def _check_decode(queries, heads, tables, lens, requests):
    if queries.ndim != 3 or int(queries.shape[2]) != _HEAD_DIM:
        raise ValueError("queries must be [R, Hq, 256]")
    R, Hq = int(queries.shape[0]), int(queries.shape[1])
    if Hq < 1 or Hq % heads != 0 or Hq // heads > 16:
        raise ValueError("query heads must be a multiple (at most 16x) of the KV heads")
    if tables.ndim != 2 or int(tables.shape[1]) < 1:
        raise ValueError("tables must be [B, P]")
    _check_ints("tables", tables, tables.shape)
    _check_ints("lens", lens, (R,))
    if requests is not None:
        _check_ints("requests", requests, (R,))
        if int(tables.shape[0]) < 1:
            raise ValueError("tables must be [B, P]")
    elif int(tables.shape[0]) != R:
        raise ValueError("without requests every query needs a table of its own")
    return R, Hq


def _queries_a_call(heads: int, page_size: int, width: int) -> int:
    """How many queries one decode call takes over tables of ``width`` pages: 65535, and 2^30 tiles of 32 keys if full together."""
    return min(65535, 0x3FFFFFFF // (heads * max(2, -(-width * page_size // 32))))


def sdpa_decode_paged(queries, keys, values, tables, lens, scale, *, requests=None, workspace=None):
    """One new query of every request over the request's pages of 16-bit rows.

    Args:
        queries: ``[R, Hq, 256]`` float16 or bfloat16, already rotated.
        keys, values: pages ``[n_pages, Hkv, page_size, 256]`` of the same dtype, at most 16 query heads per KV head.
        tables: int32 ``[B, P]``.
        lens: int32 ``[R]``, the rows that a query sees: the first so many of its request (0: the output is 0).
        requests: int32 ``[R]``, the request of a query (none of the tables': it sees nothing); by default its own place.
            Rows of a chunk name the same request, each with what it sees (``PageStep.visible`` and ``.requests``).
        scale: softmax scale.

    Entries of a table behind a request's rows, and rows behind them in a page, may hold anything; rows of a page that is not
    in the pool are left out.

    Returns:
        ``[R, Hq, 256]`` in the dtype of ``queries``.
    """
    out = _lib.dispatch.sdpa_decode_paged(queries, keys, values, tables, lens, requests, scale, workspace)
    if out is not None:
        return out
    if not torch.is_tensor(keys) or not torch.is_tensor(values):
        raise ValueError("keys and values must be 16-bit pages (8-bit ones: sdpa_decode_paged_q8)")
    n_pages, heads, page_size = _check_pages(keys, values)
    if queries.dtype != keys.dtype:
        raise ValueError("pages must have the dtype of queries")
    R, Hq = _check_decode(queries, heads, tables, lens, requests)
    dev = _lib.require_device(queries, keys, values, tables, lens, requests)
    out = torch.empty(tuple(queries.shape), dtype=queries.dtype, device=dev)
    if R == 0:
        return out
    q = _aligned(queries.contiguous())
    if workspace is None:
        workspace = _lib.paged_decode_workspace(R, Hq, heads, page_size, int(tables.shape[1]), dev)
    _lib.check(_lib.launch(
        dev, "mspr_sdpa_decode_paged", _lib.ptr(q), _lib.ptr(keys), _lib.ptr(values), _lib.DTYPE_CODE[q.dtype],
        _lib.ptr(tables), _lib.ptr(lens), _lib.ptr(requests), R, Hq, heads, _HEAD_DIM, n_pages, page_size,
        int(tables.shape[0]), int(tables.shape[1]), float(scale), _lib.ptr(out), *_lib.workspace_args(workspace, dev)), "sdpa_decode_paged")
    return out


def sdpa_decode_paged_q8(queries, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, tables, lens, scale, *,
                         group_size: int = 64, bits: int = 8, requests=None, workspace=None):
    """``sdpa_decode_paged`` over pages of affine 8-bit rows (``kquant``'s layout within a page).

    Args:
        queries: ``[R, Hq, 256]`` float32, float16 or bfloat16. The codes are multiplied as whole numbers, and weights
            and float32 queries in two terms each, so that float32 queries keep float32 results.
        k_wq, v_wq: uint32 codes ``[n_pages, Hkv, page_size, 64]``; scales and biases ``[n_pages, Hkv, page_size, 4]``.
        tables, lens, requests, scale: as for ``sdpa_decode_paged``.
    """
    if group_size != 64 or bits != 8:
        raise ValueError("sdpa_decode_paged_q8 supports group_size=64, bits=8 only")
    out = _lib.dispatch.sdpa_decode_paged_q8(queries, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, tables, lens,
                                             requests, scale, workspace)
    if out is not None:
        return out
    n_pages, heads, page_size = _check_pages((k_wq, k_scales, k_biases), (v_wq, v_scales, v_biases))
    if queries.dtype not in _lib.DTYPE_CODE:
        raise ValueError("queries must be float32, float16 or bfloat16")
    R, Hq = _check_decode(queries, heads, tables, lens, requests)
    parts = (k_wq, k_scales, k_biases, v_wq, v_scales, v_biases)
    dev = _lib.require_device(queries, *parts, tables, lens, requests)
    out = torch.empty(tuple(queries.shape), dtype=queries.dtype, device=dev)
    if R == 0:
        return out
    q = _aligned(queries.contiguous())
    if workspace is None:
        workspace = _lib.paged_decode_workspace(R, Hq, heads, page_size, int(tables.shape[1]), dev)
    _lib.check(_lib.launch(
        dev, "mspr_sdpa_decode_paged_q8", _lib.ptr(q), _lib.DTYPE_CODE[q.dtype], *(_lib.ptr(t) for t in parts),
        _lib.DTYPE_CODE[k_scales.dtype], _lib.ptr(tables), _lib.ptr(lens), _lib.ptr(requests), R, Hq, heads, _HEAD_DIM,
        n_pages, page_size, int(tables.shape[0]), int(tables.shape[1]), float(scale), 64, 8, _lib.ptr(out),
        *_lib.workspace_args(workspace, dev)), "sdpa_decode_paged_q8")
    return out


def _check_prefixes(prefix_tables, prefix_lens, groups, tables):
    """Number of prefixes and the width of their tables."""
    if prefix_tables.ndim != 2 or int(prefix_tables.shape[0]) < 1 or int(prefix_tables.shape[1]) < 1:
        raise ValueError("prefix_tables must be [G, P]")
    n = int(prefix_tables.shape[0])
    if n > MAX_SHARED:
        raise ValueError(f"at most {MAX_SHARED} prefixes a call")
    _check_ints("prefix_tables", prefix_tables, prefix_tables.shape)
    _check_ints("prefix_lens", prefix_lens, (n,))
    _check_ints("groups", groups, (int(tables.shape[0]),))
    return n, int(prefix_tables.shape[1])


def sdpa_decode_paged_shared(queries, keys, values, prefix_tables, prefix_lens, groups, tables, lens, scale, *, requests=None,
                             workspace=None):
    """``sdpa_decode_paged`` for requests that continue a prefix which others continue too: its rows are read once for a group.

    A query attends the rows of its request's prefix and then those of the request's own table. Positions are the caller's:
    the first row behind a prefix is at the prefix's length.

    Args:
        queries: ``[R, Hq, 256]`` float16 or bfloat16, already rotated, at most 2048 of them.
        keys, values, tables, lens, scale, requests: as for ``sdpa_decode_paged``; ``tables`` and ``lens`` are those of the
            requests' own rows (a query that sees none of them still sees the prefix).
        prefix_tables: int32 ``[G, P]``, the pages of every prefix, in the same pool; at most 2048 prefixes.
        prefix_lens: int32 ``[G]``, the rows of every prefix; the last page may be part-filled.
        groups: int32 ``[B]``, the prefix that a request continues (none of ``G``: none). A query of no request sees nothing.

    Returns:
        ``[R, Hq, 256]`` in the dtype of ``queries``.
    """
    out = _lib.dispatch.sdpa_decode_paged_shared(queries, keys, values, prefix_tables, prefix_lens, groups, tables, lens, requests,
                                                 scale, workspace)
    if out is not None:
        return out
    if not torch.is_tensor(keys) or not torch.is_tensor(values):
        raise ValueError("keys and values must be 16-bit pages (8-bit ones: sdpa_decode_paged_shared_q8)")
    n_pages, heads, page_size = _check_pages(keys, values)
    if queries.dtype != keys.dtype:
        raise ValueError("pages must have the dtype of queries")
    R, Hq = _check_decode(queries, heads, tables, lens, requests)
    G, width = _check_prefixes(prefix_tables, prefix_lens, groups, tables)
    if R > MAX_SHARED:
        raise ValueError(f"at most {MAX_SHARED} queries a call")
    dev = _lib.require_device(queries, keys, values, prefix_tables, prefix_lens, groups, tables, lens, requests)
    out = torch.empty(tuple(queries.shape), dtype=queries.dtype, device=dev)
    if R == 0:
        return out
    q = _aligned(queries.contiguous())
    if workspace is None:
        workspace = _lib.paged_shared_workspace(R, Hq, heads, page_size, int(tables.shape[1]), G, dev)
    _lib.check(_lib.launch(
        dev, "mspr_sdpa_decode_paged_shared", _lib.ptr(q), _lib.ptr(keys), _lib.ptr(values), _lib.DTYPE_CODE[q.dtype],
        _lib.ptr(prefix_tables), _lib.ptr(prefix_lens), _lib.ptr(groups), _lib.ptr(tables), _lib.ptr(lens), _lib.ptr(requests), R,
        Hq, heads, _HEAD_DIM, n_pages, page_size, G, width, int(tables.shape[0]), int(tables.shape[1]), float(scale),
        _lib.ptr(out), *_lib.workspace_args(workspace, dev)), "sdpa_decode_paged_shared")
    return out


def sdpa_decode_paged_shared_q8(queries, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, prefix_tables, prefix_lens, groups,
                                tables, lens, scale, *, group_size: int = 64, bits: int = 8, requests=None, workspace=None):
    """``sdpa_decode_paged_shared`` over pages of affine 8-bit rows.

    Args:
        queries: ``[R, Hq, 256]`` float32, float16 or bfloat16.
        k_wq, k_scales, k_biases, v_wq, v_scales, v_biases: as for ``sdpa_decode_paged_q8``.
        prefix_tables, prefix_lens, groups, tables, lens, scale, requests: as for ``sdpa_decode_paged_shared``.
    """
    if group_size != 64 or bits != 8:
        raise ValueError("sdpa_decode_paged_shared_q8 supports group_size=64, bits=8 only")
    out = _lib.dispatch.sdpa_decode_paged_shared_q8(queries, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, prefix_tables,
                                                    prefix_lens, groups, tables, lens, requests, scale, workspace)
    if out is not None:
        return out
    n_pages, heads, page_size = _check_pages((k_wq, k_scales, k_biases), (v_wq, v_scales, v_biases))
    if queries.dtype not in _lib.DTYPE_CODE:
        raise ValueError("queries must be float32, float16 or bfloat16")
    R, Hq = _check_decode(queries, heads, tables, lens, requests)
    G, width = _check_prefixes(prefix_tables, prefix_lens, groups, tables)
    if R > MAX_SHARED:
        raise ValueError(f"at most {MAX_SHARED} queries a call")
    parts = (k_wq, k_scales, k_biases, v_wq, v_scales, v_biases)
    dev = _lib.require_device(queries, *parts, prefix_tables, prefix_lens, groups, tables, lens, requests)
    out = torch.empty(tuple(queries.shape), dtype=queries.dtype, device=dev)
    if R == 0:
        return out
    q = _aligned(queries.contiguous())
    if workspace is None:
        workspace = _lib.paged_shared_workspace(R, Hq, heads, page_size, int(tables.shape[1]), G, dev)
    _lib.check(_lib.launch(
        dev, "mspr_sdpa_decode_paged_shared_q8", _lib.ptr(q), _lib.DTYPE_CODE[q.dtype], *(_lib.ptr(t) for t in parts),
        _lib.DTYPE_CODE[k_scales.dtype], _lib.ptr(prefix_tables), _lib.ptr(prefix_lens), _lib.ptr(groups), _lib.ptr(tables),
        _lib.ptr(lens), _lib.ptr(requests), R, Hq, heads, _HEAD_DIM, n_pages, page_size, G, width, int(tables.shape[0]),
        int(tables.shape[1]), float(scale), 64, 8, _lib.ptr(out), *_lib.workspace_args(workspace, dev)), "sdpa_decode_paged_shared_q8")
    return out


# ---------------------------------------------------------------------------------------------- pages that matter


def _check_bounds(codes, scales, heads, n_pages=None):
    """Number of pages of the bounds of a layer's pages."""
    if codes.dtype != torch.int8 or codes.ndim != 4 or int(codes.shape[0]) < 1 or tuple(codes.shape[1:]) != (heads, 2, _HEAD_DIM) or \
            (n_pages is not None and int(codes.shape[0]) != n_pages):
        raise ValueError("codes must be int8 [n_pages, Hkv, 2, 256]")
    if scales.dtype != torch.float32 or tuple(scales.shape) != tuple(codes.shape[:2]):
        raise ValueError("scales must be float32 [n_pages, Hkv]")
    if not codes.is_contiguous() or not scales.is_contiguous() or codes.storage_offset() % 16 != 0:
        raise ValueError("codes and scales must be contiguous, codes 16-byte aligned")
    return int(codes.shape[0])


def page_bounds(slots, keys, codes, scales):
    """Bounds of the keys of every page that a step wrote to, kept up with its append: what ``select_pages`` reads.

    Per page and KV head, over the rows that the page holds so far: ``scale`` is the smallest power of two (from 2^-50 to 2^50)
    with ``max |k| <= 127 * scale``, ``lower = floor(min k / scale)``, ``upper = ceil(max k / scale)``. They are made of the new rows and
    of the old bounds where the page held rows before, and are what all of its rows give. (Rows that were taken back and written
    anew leave their mark until the page is begun again: the bounds are wider then, and bounds still.)

    Args:
        slots: int32 ``[T]``, as for ``qk_norm_rope_append``, behind which this is called; the rows of a page one behind the
            other, as ``page_step`` gives them.
        keys: pages ``[n_pages, Hkv, page_size, 256]`` of 16-bit rows, or ``(codes, scales, biases)`` of 8-bit ones.
        codes: int8 ``[n_pages, Hkv, 2, 256]``, lower and upper bounds, updated in place; scales: float32 ``[n_pages, Hkv]``. Of a page
            that was never written to they may hold anything.
    """
    if _lib.dispatch.page_bounds(slots, keys, codes, scales) is not None:
        return
    n_pages, heads, page_size = _check_pages(keys, keys)
    _check_bounds(codes, scales, heads, n_pages)
    if slots.ndim != 1:
        raise ValueError("slots must be [T]")
    _check_ints("slots", slots, slots.shape)
    parts = (keys,) if torch.is_tensor(keys) else tuple(keys)
    dev = _lib.require_device(slots, *parts, codes, scales)
    T = int(slots.shape[0])
    if T == 0:
        return
    rest = (T, heads, _HEAD_DIM, n_pages, page_size, _lib.ptr(codes), _lib.ptr(scales))
    if torch.is_tensor(keys):
        rc = _lib.launch(dev, "mspr_page_bounds", _lib.ptr(slots), _lib.ptr(keys), _lib.DTYPE_CODE[keys.dtype], *rest)
    else:
        rc = _lib.launch(dev, "mspr_page_bounds_q8", _lib.ptr(slots), *(_lib.ptr(t) for t in parts), _lib.DTYPE_CODE[keys[1].dtype], *rest)
    _lib.check(rc, "page_bounds")


def _check_selected(n_selected, first, recent):
    n_selected, first, recent = int(n_selected), int(first), int(recent)
    if not 1 <= n_selected <= MAX_SELECTED or first < 0 or recent < 1 or first + recent > n_selected:
        raise ValueError(f"n_selected must be 1 to {MAX_SELECTED}, first 0 or more, recent 1 or more, and both together no more than n_selected")
    return n_selected, first, recent


def _check_selection(R, heads, tables, n_selected, first, recent):
    n_selected, first, recent = _check_selected(n_selected, first, recent)
    if int(tables.shape[1]) > MAX_TABLE_PAGES:
        raise ValueError(f"tables must hold at most {MAX_TABLE_PAGES} pages a request")
    if R * heads > 65535:
        raise ValueError("at most 65535 queries times KV heads a call")
    return n_selected, first, recent


def select_pages(queries, codes, scales, tables, lens, n_selected, *, page_size: int, first: int = 1, recent: int = 2, requests=None,
                 workspace=None):
    """The pages that every query may weigh most, per KV head, from the bounds of its request's pages.

    The bound of a page and query head is the largest product of the head's query (in 8 bits, a power of two a head) with any
    key within the page's bounds. A page is worth, at the query head where that is most, how far its bound lies above (below) the
    best bound of that head. Of requests of more than ``n_selected`` pages the first ``first`` and the last ``recent`` pages are taken,
    and those of greatest worth among the others, ties to the lower page. Bounds are exact whole numbers times a power of two: the
    same call gives the same pages.

    Args:
        queries: ``[R, Hq, 256]`` float32, float16 or bfloat16, already rotated, at most 16 query heads per KV head.
        codes, scales: of ``page_bounds``.
        tables, lens, requests: as for ``sdpa_decode_paged``; at most 32768 pages a request.
        page_size: that of the pages.
        n_selected: pages a query and KV head, at most 4096.

    Returns:
        ``(tables, lens)``: int32 ``[R, Hkv, n_selected]``, the pages in the order of their positions as pages of a pool of one head
        a page (``page * Hkv + head``, -1 behind the last), and int32 ``[R, Hkv]``, the rows in them. With a layer's pages viewed as
        ``[n_pages * Hkv, 1, page_size, 256]`` and queries as ``[R * Hkv, Hq / Hkv, 256]``, they are the tables and lengths of
        ``sdpa_decode_paged``.
    """
    done = _lib.dispatch.select_pages(queries, codes, scales, tables, lens, requests, n_selected, first, recent, page_size, workspace)
    if done is not None:
        return done
    if queries.dtype not in _lib.DTYPE_CODE:
        raise ValueError("queries must be float32, float16 or bfloat16")
    page_size = int(page_size)
    _check_page_size(page_size)
    if codes.ndim != 4 or int(codes.shape[1]) < 1:
        raise ValueError("codes must be int8 [n_pages, Hkv, 2, 256]")
    heads = int(codes.shape[1])
    n_pages = _check_bounds(codes, scales, heads)
    R, Hq = _check_decode(queries, heads, tables, lens, requests)
    n_selected, first, recent = _check_selection(R, heads, tables, n_selected, first, recent)
    dev = _lib.require_device(queries, codes, scales, tables, lens, requests)
    out_tables = torch.empty((R, heads, n_selected), dtype=torch.int32, device=dev)
    out_lens = torch.empty((R, heads), dtype=torch.int32, device=dev)
    if R == 0:
        return out_tables, out_lens
    q = _aligned(queries.contiguous())
    if workspace is None:
        workspace = _lib.select_pages_workspace(R, Hq, heads, int(tables.shape[1]), dev)
    _lib.check(_lib.launch(
        dev, "mspr_select_pages", _lib.ptr(q), _lib.DTYPE_CODE[q.dtype], _lib.ptr(codes), _lib.ptr(scales), _lib.ptr(tables),
        _lib.ptr(lens), _lib.ptr(requests), R, Hq, heads, _HEAD_DIM, n_pages, page_size, int(tables.shape[0]), int(tables.shape[1]),
        n_selected, first, recent, _lib.ptr(out_tables), _lib.ptr(out_lens), *_lib.workspace_args(workspace, dev)), "select_pages")
    return out_tables, out_lens


def sdpa_decode_paged_sparse(queries, keys, values, codes, scales, tables, lens, scale, n_selected, *, first: int = 1, recent: int = 2,
                             requests=None, workspace=None):
    """``sdpa_decode_paged`` over the pages that ``select_pages`` selects for every query and KV head.

    Args:
        queries, keys, values, tables, lens, scale, requests: as for ``sdpa_decode_paged``; the scale must not be negative.
        codes, scales, n_selected, first, recent: as for ``select_pages``.
    """
    out = _lib.dispatch.sdpa_decode_paged_sparse(queries, keys, values, codes, scales, tables, lens, requests, scale, n_selected,
                                                 first, recent, workspace)
    if out is not None:
        return out
    if not torch.is_tensor(keys) or not torch.is_tensor(values):
        raise ValueError("keys and values must be 16-bit pages (8-bit ones: sdpa_decode_paged_sparse_q8)")
    n_pages, heads, page_size = _check_pages(keys, values)
    if queries.dtype != keys.dtype:
        raise ValueError("pages must have the dtype of queries")
    R, Hq = _check_decode(queries, heads, tables, lens, requests)
    _check_bounds(codes, scales, heads, n_pages)
    n_selected, first, recent = _check_selection(R, heads, tables, n_selected, first, recent)
    dev = _lib.require_device(queries, keys, values, codes, scales, tables, lens, requests)
    out = torch.empty(tuple(queries.shape), dtype=queries.dtype, device=dev)
    if R == 0:
        return out
    q = _aligned(queries.contiguous())
    if workspace is None:
        workspace = _lib.paged_sparse_workspace(R, Hq, heads, page_size, int(tables.shape[1]), n_selected, dev)
    _lib.check(_lib.launch(
        dev, "mspr_sdpa_decode_paged_sparse", _lib.ptr(q), _lib.ptr(keys), _lib.ptr(values), _lib.DTYPE_CODE[q.dtype],
        _lib.ptr(codes), _lib.ptr(scales), _lib.ptr(tables), _lib.ptr(lens), _lib.ptr(requests), R, Hq, heads, _HEAD_DIM, n_pages,
        page_size, int(tables.shape[0]), int(tables.shape[1]), n_selected, first, recent, float(scale), _lib.ptr(out),
        *_lib.workspace_args(workspace, dev)), "sdpa_decode_paged_sparse")
    return out


def sdpa_decode_paged_sparse_q8(queries, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, codes, scales, tables, lens, scale,
                                n_selected, *, first: int = 1, recent: int = 2, group_size: int = 64, bits: int = 8, requests=None,
                                workspace=None):
    """``sdpa_decode_paged_sparse`` over pages of affine 8-bit rows.

    Args:
        queries: ``[R, Hq, 256]`` float32, float16 or bfloat16.
        k_wq, k_scales, k_biases, v_wq, v_scales, v_biases: as for ``sdpa_decode_paged_q8``.
        codes, scales, tables, lens, scale, n_selected, first, recent, requests: as for ``sdpa_decode_paged_sparse``.
    """
    if group_size != 64 or bits != 8:
        raise ValueError("sdpa_decode_paged_sparse_q8 supports group_size=64, bits=8 only")
    out = _lib.dispatch.sdpa_decode_paged_sparse_q8(queries, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, codes, scales, tables,
                                                    lens, requests, scale, n_selected, first, recent, workspace)
    if out is not None:
        return out
    n_pages, heads, page_size = _check_pages((k_wq, k_scales, k_biases), (v_wq, v_scales, v_biases))
    if queries.dtype not in _lib.DTYPE_CODE:
        raise ValueError("queries must be float32, float16 or bfloat16")
    R, Hq = _check_decode(queries, heads, tables, lens, requests)
    _check_bounds(codes, scales, heads, n_pages)
    n_selected, first, recent = _check_selection(R, heads, tables, n_selected, first, recent)
    parts = (k_wq, k_scales, k_biases, v_wq, v_scales, v_biases)
    dev = _lib.require_device(queries, *parts, codes, scales, tables, lens, requests)
    out = torch.empty(tuple(queries.shape), dtype=queries.dtype, device=dev)
    if R == 0:
        return out
    q = _aligned(queries.contiguous())
    if workspace is None:
        workspace = _lib.paged_sparse_workspace(R, Hq, heads, page_size, int(tables.shape[1]), n_selected, dev)
    _lib.check(_lib.launch(
        dev, "mspr_sdpa_decode_paged_sparse_q8", _lib.ptr(q), _lib.DTYPE_CODE[q.dtype], *(_lib.ptr(t) for t in parts),
        _lib.DTYPE_CODE[k_scales.dtype], _lib.ptr(codes), _lib.ptr(scales), _lib.ptr(tables), _lib.ptr(lens), _lib.ptr(requests), R,
        Hq, heads, _HEAD_DIM, n_pages, page_size, int(tables.shape[0]), int(tables.shape[1]), n_selected, first, recent, float(scale),
        64, 8, _lib.ptr(out), *_lib.workspace_args(workspace, dev)), "sdpa_decode_paged_sparse_q8")
    return out


# ---------------------------------------------------------------------------------------------- what a server keeps


class PageTables:
    """Lengths, tables and the stack of free pages of up to ``batch`` requests, shared by the layers of a model.

    With ``n_prefixes`` there are as many requests more, behind the others, which hold prefixes: places ``batch`` to ``batch +
    n_prefixes - 1`` of ``new_lens``. A prefix gets its rows like any request (in one step or some) and gives its pages back
    like any; a request that ``continue_prefix`` named to continue it sees its rows in front of its own, and is counted on from
    its length. It has to stay as it is while requests continue it. (``n_prefixes=0``: none, and nothing is computed for them.)
    ``max_prefix_tokens``: what a prefix has at most, in whole pages; rows behind that are no part of it. Where it is far less than
    ``max_tokens`` the attention takes a form for short prefixes (how long they are is known on the device only).
    """

    def __init__(self, batch: int, n_pages: int, page_size: int = 64, max_tokens: int = 131072, device="cuda", *,
                 n_prefixes: int = 0, max_prefix_tokens: int | None = None):
        _check_page_size(page_size)
        if max_prefix_tokens is not None and (n_prefixes == 0 or not 1 <= max_prefix_tokens <= max_tokens):
            raise ValueError("max_prefix_tokens must be 1 to max_tokens, of tables with prefixes")
        if n_prefixes < 0 or (n_prefixes > 0 and not 1 <= batch <= MAX_REQUESTS - n_prefixes):
            raise ValueError(f"requests and prefixes must be 1 to {MAX_REQUESTS} together")
        self.page_size, self.batch, self.n_prefixes = page_size, batch, n_prefixes
        batch += n_prefixes
        self.lens = torch.zeros((batch,), dtype=torch.int32, device=device)
        self.tables = torch.full((batch, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(n_pages, dtype=torch.int32, device=device)
        self.head = torch.zeros((1,), dtype=torch.int32, device=device)
        # the prefix that a request continues, -1: none
        self.groups = torch.full((batch,), -1, dtype=torch.int32, device=device) if n_prefixes else None
        # the first pages of the prefixes' tables, where these are wider
        self.prefix_tables = None if max_prefix_tokens is None else torch.full(
            (n_prefixes, -(-max_prefix_tokens // page_size)), -1, dtype=torch.int32, device=device)

    def continue_prefix(self, request: int, prefix):
        """``request`` continues ``prefix`` (from 0 on; None: none) from now on: before its first row. It stays so until said otherwise."""
        if self.groups is None or not 0 <= request < self.batch or not (prefix is None or 0 <= prefix < self.n_prefixes):
            raise ValueError(f"{request} is no request, or {prefix} no prefix, of these tables")
        self.groups[request] = -1 if prefix is None else prefix

    @property
    def prefixes(self):
        """``(prefix_tables, prefix_lens, groups)`` of ``sdpa_decode_paged_shared``; None without prefixes."""
        if self.groups is None:
            return None
        return self.tables[self.batch:] if self.prefix_tables is None else self.prefix_tables, self.lens[self.batch:], self.groups

    def step(self, new_lens, n_rows: int) -> PageStep:
        """``page_step`` that carries the lengths and the stack on (in place, so that a captured step follows them); positions
        of requests that continue a prefix are counted from its first row. (Rows without a slot belong to no request then: they
        would see the prefix.)"""
        step = page_step(self.lens, new_lens, self.tables, self.free_pages, self.head, page_size=self.page_size, n_rows=n_rows)
        self.lens.copy_(step.lens)
        self.head.copy_(step.head)
        if self.groups is None:
            return step
        # (places that are none wrap round and are masked; a prefix outside the tables is none, as for the operators)
        known = (self.groups >= 0) & (self.groups < self.n_prefixes)
        lens = self.lens[self.batch:]
        if self.prefix_tables is not None:
            width = int(self.prefix_tables.shape[1])
            self.prefix_tables.copy_(self.tables[self.batch:, :width])
            lens = lens.clamp(max=width * self.page_size)
        before = torch.where(known, lens[torch.where(known, self.groups, 0)], 0)
        return step._replace(positions=step.positions + torch.where(step.requests >= 0, before[step.requests], 0),
                             requests=torch.where(step.slots >= 0, step.requests, -1))


class PagedKVCache:
    """The pages of one layer: 16-bit rows of ``dtype``, or affine 8-bit rows with scales of ``dtype`` (``quantized``).

    With ``bounds`` every append keeps up the bounds of the pages' keys (``codes`` and ``scales`` of ``page_bounds``: 516 bytes a page
    and KV head), from which ``attend`` can select pages.
    """

    def __init__(self, n_pages: int, n_kv_heads: int, page_size: int = 64, dtype=torch.bfloat16, quantized: bool = False,
                 device="cuda", *, bounds: bool = False):
        _check_page_size(page_size)
        self.quantized = quantized
        shape = (n_pages, n_kv_heads, page_size)

        def side():
            if not quantized:
                return torch.zeros(shape + (_HEAD_DIM,), dtype=dtype, device=device)
            return (torch.zeros(shape + (_HEAD_DIM // 4,), dtype=torch.int32, device=device).view(torch.uint32),
                    torch.zeros(shape + (_HEAD_DIM // _GROUP,), dtype=dtype, device=device),
                    torch.zeros(shape + (_HEAD_DIM // _GROUP,), dtype=dtype, device=device))

        self.keys, self.values = side(), side()
        self.codes = torch.zeros((n_pages, n_kv_heads, 2, _HEAD_DIM), dtype=torch.int8, device=device) if bounds else None
        self.scales = torch.ones((n_pages, n_kv_heads), dtype=torch.float32, device=device) if bounds else None

    def append(self, q, k, v, q_weight, k_weight, positions, inv_freq, slots, *, eps: float = 1e-6, sections=None):
        """``qk_norm_rope_append`` into these pages, and ``page_bounds`` where they have bounds (``slots`` in the order of ``page_step``
        then: the rows of a page one behind the other)."""
        q = qk_norm_rope_append(q, k, v, q_weight, k_weight, positions, inv_freq, slots, self.keys, self.values, eps=eps,
                                sections=sections)
        if self.codes is not None:
            page_bounds(slots, self.keys, self.codes, self.scales)
        return q

    def attend(self, queries, tables, lens, scale, *, requests=None, workspace=None, prefixes=None, selected=None):
        """One query a request over these pages (float32 queries over 16-bit rows are rounded to the rows' type).

        Args:
            prefixes: ``(prefix_tables, prefix_lens, groups)``, for ``sdpa_decode_paged_shared``.
            selected: ``(n_selected, first, recent)``, for ``sdpa_decode_paged_sparse`` over the pages' bounds. Not with ``prefixes``.
        """
        kind, extra, where, kwargs = "", (), (), dict(requests=requests, workspace=workspace)
        if prefixes is not None:
            kind, where = "_shared", tuple(prefixes)
        if selected is not None:
            if prefixes is not None:
                raise ValueError("pages are selected of requests that continue no prefix")
            if self.codes is None:
                raise ValueError("pages without bounds cannot be selected from")
            n_selected, kwargs["first"], kwargs["recent"] = selected
            kind, where, extra = "_sparse", (self.codes, self.scales), (n_selected,)
        if self.quantized:
            return _ATTEND[kind + "_q8"](queries, *self.keys, *self.values, *where, tables, lens, scale, *extra, **kwargs)
        asked = queries.to(self.keys.dtype) if queries.dtype == torch.float32 else queries
        out = _ATTEND[kind](asked, self.keys, self.values, *where, tables, lens, scale, *extra, **kwargs)
        return out.float() if queries.dtype == torch.float32 else out


# what a cache attends with, by what is to be left out or shared
_ATTEND = {"": sdpa_decode_paged, "_q8": sdpa_decode_paged_q8, "_shared": sdpa_decode_paged_shared,
           "_shared_q8": sdpa_decode_paged_shared_q8, "_sparse": sdpa_decode_paged_sparse, "_sparse_q8": sdpa_decode_paged_sparse_q8}


class _NoGradient(torch.autograd.Function):
    """``out`` as it is, in the graph of the tensors it was made from, through which there is no way back."""

    @staticmethod
    def forward(ctx, out, *made_from):
        return out

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("PagedAttention serves and has no backward pass: run it under torch.no_grad(), or detach what goes in")


def _called(module, x, **kwargs):
    """What the module makes of ``x``, None where it has no forward that takes it and gives its like."""
    call = module.forward if isinstance(module, torch.nn.Module) else module
    if getattr(call, "__func__", call) is torch.nn.Module.forward or not callable(call):
        return None
    try:
        inspect.signature(call).bind(x, **kwargs)
    except TypeError:
        return None
    with torch.no_grad():
        out = call(x, **kwargs)
    return out if torch.is_tensor(out) and out.shape == x.shape else None


def _check_modules(inner):
    """The operators take weights, eps and frequencies of the norms and the rope, not the modules: refuse modules that make
    something else of them (a weight counted from 1, another pairing of channels, angles that are scaled)."""
    for name in ("q_norm", "k_norm"):
        norm = getattr(inner, name)
        w = norm.weight
        if tuple(w.shape) != (_HEAD_DIM,):
            raise ValueError(f"{name} must have a weight of 256 channels")
        # (a row of ordinary size, and one whose mean square is about an eps)
        x = torch.cos(torch.arange(2 * _HEAD_DIM, device=w.device)).reshape(1, 2, 1, _HEAD_DIM).to(w.dtype)
        x[:, 1] *= 1e-3
        got = _called(norm, x)
        y = x.float()
        want = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + norm.eps) * w.detach().float()
        if got is not None and bool(((got.float() - want).abs().amax(-1) > 0.05 * want.abs().amax(-1)).any()):
            raise ValueError(f"{name} is not weight * x / sqrt(mean(x^2) + eps), which is what this layer computes")
    inv = inner.rope.inv_freq
    half = int(inv.shape[-1])
    x = torch.cos(torch.arange(3 * _HEAD_DIM, device=inv.device)).reshape(1, 1, 3, _HEAD_DIM).to(inner.q_norm.weight.dtype)
    got = _called(inner.rope, x, offset=5)
    if got is None:
        return
    angle = torch.arange(5, 8, device=inv.device)[:, None] * inv.float()
    a, b, rest = x.float().tensor_split((half, 2 * half), dim=-1)
    want = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), rest], dim=-1)
    if bool((got.float() - want).abs().max() > 0.05):
        raise ValueError("rope does not rotate channels i and i + rotary_dim / 2 by position * inv_freq[i], which is what this "
                         "layer computes")


class PagedAttention(torch.nn.Module):
    """One full-attention layer over a paged cache: a step's rows of many requests through the wrapped block's projections.

    ``inner`` is a block as ``full_attention.FlashPrefillD256Attention`` wraps it; of its modules this takes ``q_proj`` (with
    the output gate in the second half of every head), ``k_proj``, ``v_proj``, ``o_proj``, ``q_norm`` and ``k_norm``
    (``weight``, of the type of ``x`` and multiplied as it is, and one ``eps``), ``rope`` (``inv_freq`` and, for three position
    axes, ``sections``), ``scale``, ``num_attention_heads`` and ``num_key_value_heads``. Norms and rope are not called, but made
    anew from these: a norm or rope that can be called and gives something else is refused, and so are hooks on them. A block
    may come without ``eps``, ``inv_freq`` or ``sections`` where only the wrapper uses it; this layer needs them.

    Where the tables hold prefixes (``n_prefixes`` of ``PageTables``), requests attend the prefix they continue and their own rows. With
    ``n_selected`` (and a cache with ``bounds``) every row attends the pages alone that ``select_pages`` takes for it, ``first`` and
    ``recent`` ones among them: all there are while a request has no more.

    The layer serves: a backward pass that would have to go through its attention raises (the gate and the projection behind it
    alone would leave gradients that lack a part).
    """

    def __init__(self, inner, cache: PagedKVCache, *, n_selected=None, first: int = 1, recent: int = 2):
        super().__init__()
        if inner.q_norm.eps != inner.k_norm.eps:
            raise ValueError("q_norm and k_norm must share an eps")
        self.n_pages, kv_heads, self.page_size = _check_pages(cache.keys, cache.values)
        if inner.num_key_value_heads != kv_heads:
            raise ValueError("the block and the cache disagree on the number of KV heads")
        if inner.num_attention_heads % kv_heads != 0 or not 1 <= inner.num_attention_heads // kv_heads <= 16:
            raise ValueError("query heads must be a multiple (at most 16x) of the KV heads")
        _check_modules(inner)
        self.selected = None
        if n_selected is not None:
            self.selected = _check_selected(n_selected, first, recent)
            if cache.codes is None:
                raise ValueError("pages are selected by their bounds: the cache must have them")
            if inner.scale < 0:
                raise ValueError("pages are selected where the softmax scale is not negative")
            if self.n_pages * kv_heads * self.page_size > 0x7FFFFFFF:
                raise ValueError("pages are selected of pools of fewer than 2^31 tokens times KV heads")
        self.inner = inner
        self.cache = cache

    def _most(self, tables, selected):
        """Queries of one call; none of them without a reason that is raised, before anything is written."""
        kv_heads, width = self.inner.num_key_value_heads, int(tables.tables.shape[1])
        most = _queries_a_call(kv_heads, tables.page_size, width)
        if tables.groups is not None:
            if selected is not None:
                raise ValueError("pages are selected of requests that continue no prefix: ask for dense=True, or for tables without")
            # (at most a block of columns a query and KV head, and its own rows)
            most = min(MAX_SHARED, 0x3FFFFFFF // (2 * kv_heads * (-(-width * tables.page_size // 32) + 1)))
        if selected is not None:
            if width > MAX_TABLE_PAGES:
                raise ValueError(f"pages are selected from tables of at most {MAX_TABLE_PAGES} pages")
            # (a query and KV head is a request to the attention over its pages)
            tiles = -(-selected[0] * tables.page_size // 32) + 1
            most = min(2048, 65535 // kv_heads, 0x3FFFFFFF // (kv_heads * tiles)) if tiles <= 0x2000000 else 0
            # (of a query: a bound for every query head and page that its table could name, and the selected pages)
            scratch = 4 * (self.inner.num_attention_heads * (-(-width // 16) * 16) + kv_heads * selected[0])
            most = min(most, max(1, _SELECTION_BYTES // scratch))
        if most < 1:
            raise ValueError("the tables hold too many tokens together")
        return most

    def forward(self, x, step: PageStep, tables: PageTables, positions=None, *, dense: bool = False):
        """``x``: ``[n_rows, hidden]``, the rows of ``step``. ``positions``: int32 ``[3, n_rows]`` where the rope has sections.
        ``dense``: this step attends all pages, also where the layer selects (the steps of a prompt)."""
        inner = self.inner
        for module in (inner.q_norm, inner.k_norm, inner.rope):
            if getattr(module, "_forward_hooks", None) or getattr(module, "_forward_pre_hooks", None):
                raise RuntimeError("hooks of q_norm, k_norm and rope would not run: this layer takes their weights and frequencies")
        T = int(x.shape[0])
        heads, kv_heads = inner.num_attention_heads, inner.num_key_value_heads
        if tables.page_size != self.page_size or int(tables.free_pages.shape[0]) > self.n_pages:
            raise ValueError("the tables name pages of another size, or more of them, than the cache has")
        selected = None if dense else self.selected
        most = self._most(tables, selected)
        asked = {}
        if tables.groups is not None:
            asked["prefixes"] = tables.prefixes
        if selected is not None:
            asked["selected"] = selected
        # (widths in full: a step in which every request ends has no rows, of which a width could not be told)
        q, gate = inner.q_proj(x).reshape(T, heads, 2 * _HEAD_DIM).chunk(2, dim=-1)
        k = inner.k_proj(x).reshape(T, kv_heads, _HEAD_DIM)
        v = inner.v_proj(x).reshape(T, kv_heads, _HEAD_DIM)
        made_from = (q, k, v, inner.q_norm.weight, inner.k_norm.weight)
        q = self.cache.append(q, k, v, inner.q_norm.weight, inner.k_norm.weight,
                              step.positions if positions is None else positions, inner.rope.inv_freq, step.slots,
                              eps=inner.q_norm.eps, sections=None if positions is None else inner.rope.sections)
        if T <= most:
            out = self.cache.attend(q, tables.tables, step.visible, inner.scale, requests=step.requests, **asked)
        else:
            out = torch.cat([self.cache.attend(q[i:i + most], tables.tables, step.visible[i:i + most], inner.scale,
                                               requests=step.requests[i:i + most], **asked) for i in range(0, T, most)])
        if torch.is_grad_enabled() and any(t.requires_grad for t in made_from):
            out = _NoGradient.apply(out, *made_from)
        return inner.o_proj((out * torch.sigmoid(gate)).reshape(T, heads * _HEAD_DIM))
