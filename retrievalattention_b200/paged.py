"""Operators over one layer of a paged KV cache.

* ``rope_paged_append``  rotary positions with several axes (text, images, video) on a fused QKV projection; queries out, keys and
                         values into the cache's pages;
* ``paged_decode``       attention of one new token over the pages, optionally adding up the weight that every slot gets;
* ``paged_observe``      the weight that a prompt's last queries give to its slots;
* ``paged_evict``        the slots of least weight give way, in place.

The layer is a handful of tensors that the caller owns (``cache_hub.paged_cache`` keeps them for a whole model):

``key_pages``, ``value_pages``  bf16 or fp16 ``[pages, kv_heads, page_size, 128]``, each page dense, page_size a power of two from 8
``weight``, ``token``           fp32 and int32 ``[pages, kv_heads, page_size]``: the attention weight that a slot's key was given so
                                far, and the number of its token in its request
``page_table``, ``lengths``     int32 ``[batch, most pages of a request]`` and ``[batch]``: slot ``j`` of request ``b`` is row
                                ``j % page_size`` of page ``page_table[b, j // page_size]`` for every head, and the first
                                ``lengths[b]`` slots are in use; table entries behind them are not read.  Requests may share pages
                                that nothing is written to (no weights, rows or evictions).  Rows of the table may lie apart: workspaces
                                and the choice of kernels follow the slots that its width has room for, so hand in no more of
                                a wide one than the longest request needs (``page_table[:, :pages]``)

Every call is asynchronous on the current stream, allocates its workspace from torch's caching allocator and can be captured in a
CUDA graph.  Lengths and page tables are read on the device: an entry that names no page, or a row that its request's table has no
slot for, is reported by the next call or by ``attn_hub.check_prefill_errors``.  There are no gradients.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import os

from . import _lib, status as _status

DIM = 128
MAX_GROUP = 8                              # query heads to a KV head that paged_decode takes
_SCALE = DIM ** -0.5
_BINDING = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_paged_binding.so")


_native = None                             # the checks of the arguments and the calls (binding/paged.cpp)


def _connect():
    """Load them on first use, and hand over the library's functions."""
    global _native
    if not os.path.exists(_BINDING):
        raise ImportError(f"{_BINDING} is missing: build it with `python -m retrievalattention_b200.build`")
    spec = importlib.util.spec_from_file_location("_paged_binding", _BINDING)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    names = ("ri_last_error", "ri_rope_paged_append", "ri_paged_decode_scratch_bytes", "ri_paged_decode",
             "ri_paged_observe_scratch_bytes", "ri_paged_observe", "ri_paged_evict_scratch_bytes", "ri_paged_evict")
    addresses = {n: C.cast(getattr(_lib.lib, n), C.c_void_p).value for n in names}
    addresses["status_word"] = _status.address()
    module.connect(addresses, _status.used, _status.report_word)
    _native = module
    return module


def _sections(sections) -> list:
    if any(int(n) != n or n < 0 for n in sections):
        raise ValueError(f"sections {sections}: expected numbers of frequencies")
    return [int(n) for n in sections]


def rope_sections(*sections: int) -> tuple:
    """``axis_of`` for frequencies that follow one axis section after section: ``rope_sections(64)`` is the ordinary rotary
    embedding, ``rope_sections(16, 24, 24)`` time, height and width."""
    return tuple(a for a, n in enumerate(_sections(sections)) for _ in range(n))


def rope_interleaved(*sections: int) -> tuple:
    """``axis_of`` for frequencies that are dealt out to the axes in turn, while an axis has any left."""
    left, axes, a = _sections(sections), [], 0
    while any(left):
        if left[a]:
            left[a] -= 1
            axes.append(a)
        a = (a + 1) % len(left)
    return tuple(axes)


def _axes(axis_of) -> bytes:
    try:
        return bytes(list(axis_of))                             # a number, which bytes() takes for a length, is no list
    except (TypeError, ValueError):
        raise ValueError("rope_paged_append: axis_of names an axis for each of the 64 frequencies") from None


def rope_paged_append(qkv, cos_sin, positions, axis_of, q, key_pages, value_pages, page_table, lengths, row_start=None, *, weight=None,
                      token=None, seen=None, keys=None, values=None):
    """Rotate the query and key heads of ``qkv`` ``[rows, (q_heads + 2 kv_heads) * 128]`` (rows may lie apart), write the queries to
    ``q`` ``[rows, q_heads, 128]`` and keys and values to the cache, behind the ``lengths`` slots in use (which stay as they are: add
    the rows once the last layer has its own).

    Frequency ``i`` turns by ``positions[axis_of[i], row]`` (int64 ``[axes, rows]``), looked up in ``cos_sin``
    (``decode_layer.cos_sin_cache``; positions outside it take its ends); ``rope_sections`` and ``rope_interleaved`` make
    ``axis_of``.  Rows ``row_start[b]`` to ``row_start[b + 1] - 1`` (int32 ``[batch + 1]``) are request ``b``'s; without it row ``b``
    is.  Where ``weight`` and ``token`` are given, the new slots start with weight 0 and the token numbers ``seen[b]``,
    ``seen[b] + 1``, ...  ``keys`` and ``values`` ``[rows, kv_heads, 128]`` take the rows a second time, as
    ``retroinfer_prefill_attn`` reads them."""
    native = _native or _connect()
    native.append(qkv, cos_sin, positions, _axes(axis_of), q, key_pages, value_pages, page_table, lengths, row_start, weight, token,
                  seen, keys, values)


def paged_decode(q, key_pages, value_pages, page_table, lengths, *, out=None, lse=None, weight=None, scale=None):
    """Attention of one new token: ``q`` ``[batch, 1, q_heads, 128]`` (requests may lie apart; one to eight query heads to a KV
    head) over the slots in use, which the token's own row is one of.  Returns ``out`` like ``q``; ``lse`` fp32 ``[batch, q_heads]``
    takes the log-sum-exp of the scaled scores (``scale``: 1/sqrt(128)).  A request without slots has out 0 and lse -infinity.
    ``weight``: every slot's weight grows by the probabilities it got, summed over the query heads of its KV head."""
    native = _native or _connect()
    return native.decode(q, key_pages, value_pages, page_table, lengths, out, lse, weight, _SCALE if scale is None else scale)


def paged_observe(q, key_pages, page_table, lengths, weight, *, scale=None):
    """Add to every slot's ``weight`` the probabilities that the last queries of its request give it: ``q`` dense ``[batch, window,
    q_heads, 128]``, the rows of the last ``window`` tokens in use, each of which sees the slots up to its own; summed over queries
    and over the query heads of a KV head.  What ``paged_evict`` goes by after a prompt.  Requests shorter than the window are
    padded in front, with anything.  Slots must be in the order of their tokens (no eviction before)."""
    native = _native or _connect()
    native.observe(q, key_pages, page_table, lengths, weight, _SCALE if scale is None else scale)


def paged_evict(key_pages, value_pages, weight, token, page_table, lengths, seen, keep, n_sink=0, n_recent=0):
    """Requests of more than ``keep`` slots keep ``keep`` for every KV head: the slots of the first ``n_sink`` and the last
    ``n_recent`` of their ``seen[b]`` tokens (int32 ``[batch]``; together at most ``keep``), then those of largest weight, the lower
    slot first among equals.  In place: the i-th slot in front of ``keep`` that goes takes the key, value, weight and token number
    of the i-th one behind it that stays, so slots are no longer in the order of their tokens.  ``lengths`` and the page tables are
    left alone: clamp the lengths to ``keep`` when the last layer is done, and the pages behind are free.  Requests must not share
    pages."""
    native = _native or _connect()
    native.evict(key_pages, value_pages, weight, token, page_table, lengths, seen, keep, n_sink, n_recent)
