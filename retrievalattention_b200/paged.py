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
                                ``lengths[b]`` slots are in use; table entries behind them are not read

Every call is asynchronous on the current stream, allocates its workspace from torch's caching allocator and can be captured in a
CUDA graph.  Lengths and page tables are read on the device: an entry that names no page, or a row that its request's table has no
slot for, is reported by the next call or by ``attn_hub.check_prefill_errors``.  There are no gradients.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib, status as _status

DIM = 128
_SCALE = DIM ** -0.5


def _fail(what, message):
    raise ValueError(f"{what}: {message}")


def _layer(what, key_pages, value_pages, page_table, lengths, weight, token, group):
    """The struct that describes the layer, and the status word.  Written out: it runs once per layer and token."""
    dev = key_pages.device
    if key_pages.dim() != 4 or key_pages.shape[3] != DIM or not key_pages.is_cuda:
        _fail(what, "expected key_pages [pages, kv_heads, page_size, 128] on a GPU")
    pages, hk, page, _ = key_pages.shape
    dtype = _lib.dtype_code(key_pages.dtype)
    key_stride, value_stride, values = key_pages.stride(), None, None
    if key_stride[3] != 1 or key_stride[2] != DIM or (hk > 1 and key_stride[1] != page * DIM):
        _fail(what, "every page of key_pages must be dense")
    if value_pages is not None:
        if value_pages.shape != key_pages.shape or value_pages.dtype != key_pages.dtype or value_pages.device != dev:
            _fail(what, "value_pages must be like key_pages")
        value_stride = value_pages.stride()
        if value_stride[3] != 1 or value_stride[2] != DIM or (hk > 1 and value_stride[1] != page * DIM):
            _fail(what, "every page of value_pages must be dense")
        values = value_pages.data_ptr()
    if key_pages.requires_grad or (value_pages is not None and value_pages.requires_grad):
        _fail(what, "there are no gradients")
    if (page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != dev or not page_table.is_contiguous()):
        _fail(what, "expected a dense int32 page_table [batch, pages of a request] on the pools' GPU")
    b = page_table.shape[0]
    if lengths.shape != (b,) or lengths.dtype != torch.int32 or lengths.device != dev or not lengths.is_contiguous():
        _fail(what, "expected dense int32 lengths [batch] on the pools' GPU")
    for x, kind, name in ((weight, torch.float32, "weight"), (token, torch.int32, "token")):
        if x is not None and (x.shape != (pages, hk, page) or x.dtype != kind or x.device != dev or not x.is_contiguous()):
            _fail(what, f"expected dense {name} [pages, kv_heads, page_size] on the pools' GPU")
    status = _status.word(dev)
    dense = hk * page * DIM                                       # the stride of a dimension of one page may be anything
    return _lib.Paged(b, hk, group, page, pages, page_table.shape[1], dtype, 0, key_stride[0] if pages > 1 else dense,
                      0 if values is None else value_stride[0] if pages > 1 else dense, key_pages.data_ptr(), values,
                      None if weight is None else weight.data_ptr(), None if token is None else token.data_ptr(),
                      page_table.data_ptr(), lengths.data_ptr(), C.addressof(status)), status


def _elsewhere(tensor) -> bool:
    return tensor.is_cuda and tensor.device.index != torch.cuda.current_device()


def rope_sections(*sections: int) -> tuple:
    """``axis_of`` for frequencies that follow one axis section after section: ``rope_sections(64)`` is the ordinary rotary
    embedding, ``rope_sections(16, 24, 24)`` time, height and width."""
    return tuple(a for a, n in enumerate(sections) for _ in range(n))


def rope_interleaved(*sections: int) -> tuple:
    """``axis_of`` for frequencies that are dealt out to the axes in turn, while an axis has any left."""
    left, axes, a = list(sections), [], 0
    while any(left):
        if left[a]:
            left[a] -= 1
            axes.append(a)
        a = (a + 1) % len(left)
    return tuple(axes)


def _axes(axis_of) -> bytes:
    try:
        of = bytes(axis_of)
    except (TypeError, ValueError):
        of = b""
    if len(of) != DIM // 2:
        _fail("rope_paged_append", "axis_of names an axis for each of the 64 frequencies")
    return of


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
    what = "rope_paged_append"
    if _elsewhere(qkv):
        with torch.cuda.device(qkv.device):
            return rope_paged_append(qkv, cos_sin, positions, axis_of, q, key_pages, value_pages, page_table, lengths, row_start,
                                     weight=weight, token=token, seen=seen, keys=keys, values=values)
    hk, dev = key_pages.shape[1] if key_pages.dim() == 4 else 0, qkv.device
    if qkv.dim() != 2 or q.dim() != 3 or hk < 1 or q.shape[1] < hk or q.shape[1] % hk:
        _fail(what, "expected qkv [rows, (q_heads + 2 kv_heads) * 128] and q [rows, q_heads, 128], q_heads a multiple of kv_heads")
    rows, hq = qkv.shape[0], q.shape[1]
    if qkv.shape[1] != (hq + 2 * hk) * DIM or q.shape != (rows, hq, DIM) or (qkv.stride(1) != 1 and rows > 0):
        _fail(what, "expected qkv [rows, (q_heads + 2 kv_heads) * 128] with dense rows, and q [rows, q_heads, 128]")
    if value_pages is None:
        _fail(what, "value_pages is missing")
    for x, shape, name in ((q, (rows, hq, DIM), "q"), (keys, (rows, hk, DIM), "keys"), (values, (rows, hk, DIM), "values")):
        if x is not None and (x.shape != shape or not x.is_contiguous()):
            _fail(what, f"expected dense {name} {list(shape)}")
    for x in (qkv, q, keys, values):
        if x is not None and (x.dtype != key_pages.dtype or x.device != key_pages.device or x.requires_grad):
            _fail(what, "expected qkv, q, keys, values and the pages of one type on one GPU, without gradients")
    if cos_sin.dim() != 2 or cos_sin.shape[1] != DIM or cos_sin.dtype != torch.float32 or cos_sin.device != dev or not cos_sin.is_contiguous():
        _fail(what, "expected dense fp32 cos_sin [positions, 128]")
    axes = positions.shape[0] if positions.dim() == 2 else 1
    if (positions.dim() not in (1, 2) or positions.shape[-1] != rows or positions.dtype != torch.int64 or positions.device != dev
            or not positions.is_contiguous()):
        _fail(what, "expected dense int64 positions [axes, rows]")
    of = _axes(axis_of)
    layer, status = _layer(what, key_pages, value_pages, page_table, lengths, weight, token, hq // hk)
    for x, shape, name in ((row_start, (layer.batch + 1,), "row_start"), (seen, (layer.batch,), "seen")):
        if x is not None and (x.shape != shape or x.dtype != torch.int32 or x.device != dev or not x.is_contiguous()):
            _fail(what, f"expected dense int32 {name} {list(shape)}")
    if token is not None and seen is None:
        _fail(what, "token numbers need `seen`")
    if rows == 0:
        return
    _lib.check(_lib.lib.ri_rope_paged_append(
        C.byref(layer), qkv.data_ptr(), qkv.stride(0) if rows > 1 else qkv.shape[1], cos_sin.data_ptr(), cos_sin.shape[0],
        positions.data_ptr(), of, axes, rows, None if row_start is None else row_start.data_ptr(),
        None if seen is None else seen.data_ptr(), q.data_ptr(), None if keys is None else keys.data_ptr(),
        None if values is None else values.data_ptr(), _lib.current_stream()), what)
    torch.autograd.graph.increment_version([x for x in (q, keys, values, key_pages, value_pages, weight, token) if x is not None])
    _status.report(status)


def paged_decode(q, key_pages, value_pages, page_table, lengths, *, out=None, lse=None, weight=None, scale=None):
    """Attention of one new token: ``q`` ``[batch, 1, q_heads, 128]`` (requests may lie apart; one to eight query heads to a KV
    head) over the slots in use, which the token's own row is one of.  Returns ``out`` like ``q``; ``lse`` fp32 ``[batch, q_heads]``
    takes the log-sum-exp of the scaled scores (``scale``: 1/sqrt(128)).  A request without slots has out 0 and lse -infinity.
    ``weight``: every slot's weight grows by the probabilities it got, summed over the query heads of its KV head."""
    what = "paged_decode"
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return paged_decode(q, key_pages, value_pages, page_table, lengths, out=out, lse=lse, weight=weight, scale=scale)
    if q.dim() != 4 or key_pages.dim() != 4 or value_pages is None:
        _fail(what, "expected q [batch, 1, q_heads, 128] and pages [pages, kv_heads, page_size, 128]")
    b, one, hq, d = q.shape
    hk, strides = key_pages.shape[1], q.stride()
    if one != 1 or d != DIM or hk < 1 or hq < hk or hq % hk or page_table.shape[0] != b:
        _fail(what, "expected q [batch, 1, q_heads, 128], q_heads a multiple of kv_heads, one page table row per request")
    if strides[3] != 1 or (hq > 1 and strides[2] != DIM):
        _fail(what, "the heads of a request must lie dense in q")
    if q.dtype != key_pages.dtype or q.device != key_pages.device or q.requires_grad:
        _fail(what, "expected q and the pages of one type on one GPU, without gradients")
    layer, status = _layer(what, key_pages, value_pages, page_table, lengths, weight, None, hq // hk)
    if out is None:
        out = torch.empty((b, 1, hq, DIM), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
        _fail(what, "expected dense out like q")
    if lse is not None and (lse.shape != (b, hq) or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous()):
        _fail(what, "expected dense fp32 lse [batch, q_heads]")
    size = _lib.lib.ri_paged_decode_scratch_bytes(C.byref(layer))
    if size < 0:
        _lib.check(size, what)
    scratch = torch.empty((size,), dtype=torch.uint8, device=q.device)
    _lib.check(_lib.lib.ri_paged_decode(C.byref(layer), q.data_ptr(), strides[0] if b > 1 else hq * DIM, out.data_ptr(),
                                        None if lse is None else lse.data_ptr(), _SCALE if scale is None else scale,
                                        scratch.data_ptr(), _lib.current_stream()), what)
    torch.autograd.graph.increment_version([x for x in (out, lse, weight) if x is not None])
    _status.report(status)
    return out


def paged_observe(q, key_pages, page_table, lengths, weight, *, scale=None):
    """Add to every slot's ``weight`` the probabilities that the last queries of its request give it: ``q`` dense ``[batch, window,
    q_heads, 128]``, the rows of the last ``window`` tokens in use, each of which sees the slots up to its own; summed over queries
    and over the query heads of a KV head.  What ``paged_evict`` goes by after a prompt.  Requests shorter than the window are
    padded in front, with anything.  Slots must be in the order of their tokens (no eviction before)."""
    what = "paged_observe"
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return paged_observe(q, key_pages, page_table, lengths, weight, scale=scale)
    if q.dim() != 4 or key_pages.dim() != 4 or weight is None:
        _fail(what, "expected q [batch, window, q_heads, 128], pages [pages, kv_heads, page_size, 128] and weights")
    b, window, hq, d = q.shape
    hk = key_pages.shape[1]
    if d != DIM or window < 1 or hk < 1 or hq < hk or hq % hk or page_table.shape[0] != b or not q.is_contiguous():
        _fail(what, "expected dense q [batch, window, q_heads, 128], q_heads a multiple of kv_heads, one page table row per request")
    if q.dtype != key_pages.dtype or q.device != key_pages.device or q.requires_grad:
        _fail(what, "expected q and the pages of one type on one GPU, without gradients")
    layer, status = _layer(what, key_pages, None, page_table, lengths, weight, None, hq // hk)
    size = _lib.lib.ri_paged_observe_scratch_bytes(C.byref(layer))
    if size < 0:
        _lib.check(size, what)
    scratch = torch.empty((size,), dtype=torch.uint8, device=q.device)
    _lib.check(_lib.lib.ri_paged_observe(C.byref(layer), q.data_ptr(), window, _SCALE if scale is None else scale, scratch.data_ptr(),
                                         _lib.current_stream()), what)
    torch.autograd.graph.increment_version(weight)
    _status.report(status)


def paged_evict(key_pages, value_pages, weight, token, page_table, lengths, seen, keep, n_sink=0, n_recent=0):
    """Requests of more than ``keep`` slots keep ``keep`` for every KV head: the slots of the first ``n_sink`` and the last
    ``n_recent`` of their ``seen[b]`` tokens (int32 ``[batch]``; together at most ``keep``), then those of largest weight, the lower
    slot first among equals.  In place: the i-th slot in front of ``keep`` that goes takes the key, value, weight and token number
    of the i-th one behind it that stays, so slots are no longer in the order of their tokens.  ``lengths`` and the page tables are
    left alone: clamp the lengths to ``keep`` when the last layer is done, and the pages behind are free.  Requests must not share
    pages."""
    what = "paged_evict"
    if _elsewhere(key_pages):
        with torch.cuda.device(key_pages.device):
            return paged_evict(key_pages, value_pages, weight, token, page_table, lengths, seen, keep, n_sink, n_recent)
    if value_pages is None or weight is None or token is None:
        _fail(what, "keys, values, weights and token numbers move together: none may be missing")
    layer, status = _layer(what, key_pages, value_pages, page_table, lengths, weight, token, 1)
    if seen.shape != (layer.batch,) or seen.dtype != torch.int32 or seen.device != key_pages.device or not seen.is_contiguous():
        _fail(what, "expected dense int32 seen [batch]")
    size = _lib.lib.ri_paged_evict_scratch_bytes(C.byref(layer), keep)
    if size < 0:
        _lib.check(size, what)
    scratch = torch.empty((size,), dtype=torch.uint8, device=key_pages.device)
    _lib.check(_lib.lib.ri_paged_evict(C.byref(layer), seen.data_ptr(), keep, n_sink, n_recent, scratch.data_ptr(),
                                       _lib.current_stream()), what)
    torch.autograd.graph.increment_version((key_pages, value_pages, weight, token))
    _status.report(status)
