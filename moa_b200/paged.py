"""Paged key/value cache: append with the rotary embedding on the way, and attention of one new token.

The ring cache (``cache.py``) holds one token count for the whole batch and one ring per head.  A server
that answers many requests at once has sequences of different lengths that come and go, and models whose
query heads share key/value heads; its cache is a pool of pages that sequences take from and give back.
The kernels are ``csrc/paged.cu``; there is no CPU path and no gradient, as in the rest of the package.
"""
from __future__ import annotations

import struct
from typing import Dict, Optional, Tuple

import torch
from torch import Tensor

from . import _lib
from ._lib import lib

# fields of moa_paged_append_args and moa_paged_decode_args (include/moa_b200.h), all 8 bytes wide
_APPEND = struct.Struct("=12Q30q")
_DECODE = struct.Struct("=13Q30qd")
_COUNTER_BYTES = 8192
_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_NO_ROPE = (0, 0, 0, 0, 0, 0)

# the stream's handle without a Stream object around it, as torch's own generated code asks for it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or _lib.current_stream
_capturing = torch.cuda.is_current_stream_capturing

_workspaces: Dict = {}
_touched = set()      # devices that a paged call has run on


def _workspace(index: int, stream: int) -> Tensor:
    """Scratch of ``paged_decode``: kept per device and stream; a call that is being captured gets one of its own,
    from the graph's memory, so that two graphs never share one."""
    if _capturing():
        ws = torch.empty(lib.moa_paged_decode_workspace_bytes(), dtype=torch.uint8, device=index)
        ws[:_COUNTER_BYTES].zero_()
        return ws
    ws = _workspaces.get((index, stream))
    if ws is None:
        ws = _workspaces[index, stream] = torch.zeros(lib.moa_paged_decode_workspace_bytes(), dtype=torch.uint8,
                                                      device=index)
    return ws


# The checks below run on every call, and at decode sizes the host's share of a call is larger than the
# kernel's: they ask a tensor for each property once, and for the cheapest form of it (get_device() instead of
# device, all strides at once), and they are few functions.

def _pool_arguments(key_pages: Tensor, value_pages: Tensor, page_table: Tensor, lengths: Tensor, B: int, D: int, dtype,
                    device: int):
    assert dtype in _DTYPES, f"the paged cache supports float16 and bfloat16 only, got {dtype}"
    shape = key_pages.shape
    assert len(shape) == 4 and value_pages.shape == shape and shape[3] == D, "pages must be (num_pages, KV, page_size, D)"
    assert key_pages.dtype is dtype and value_pages.dtype is dtype, "pages and tokens must have the same dtype"
    ka, kb, kc, kd = key_pages.stride()
    va, vb, vc, vd = value_pages.stride()
    assert kd == 1 and vd == 1, "rows of the pages must be contiguous"
    width = page_table.shape
    assert len(width) == 2 and width[0] == B and page_table.dtype is torch.int32, "page_table must be int32 (B, max_pages)"
    width = width[1]
    ta, tb = page_table.stride()
    assert tb == 1 or width == 1, "rows of page_table must be contiguous"
    assert lengths.dtype is torch.int32 and lengths.shape == (B,) and lengths.is_contiguous(), \
        "lengths must be contiguous int32 (B,)"
    assert device == key_pages.get_device() == value_pages.get_device() == page_table.get_device() == \
        lengths.get_device(), "all tensors must be on the same device"
    return ka, kb, kc, va, vb, vc, ta, width, shape[0], shape[2], shape[1]


def _rope_arguments(rope: Tuple[Tensor, Tensor], B: int, N: int, D: int, dtype, device: int):
    cos, sin = rope
    shape, stride = cos.shape, cos.stride()
    assert sin.shape == shape and sin.stride() == stride and stride[-1] == 1 and shape[-1] == D, \
        "rope tables must be two tensors of one shape and layout with rows of D"
    kind = cos.dtype
    assert sin.dtype is kind and (kind is dtype or kind is torch.float32), \
        "rope tables must have the tensors' dtype or be float32"
    assert device == cos.get_device() == sin.get_device(), "all tensors must be on the same device"
    if len(shape) == 2:
        assert shape[0] > 0, "a rope table by position needs rows"
        return cos.data_ptr(), sin.data_ptr(), 0, stride[0], shape[0], kind is torch.float32
    assert len(shape) == 3 and (shape[0] == 1 or shape[0] == B) and shape[1] == N, \
        "rope tables must be (positions, D), (B, N, D) or (1, N, D)"
    return cos.data_ptr(), sin.data_ptr(), 0 if shape[0] == 1 else stride[0], stride[1], 0, kind is torch.float32


def _rows(t: Tensor, N: int):
    """``t`` (.., .., N, D), or a copy of it whose rows the kernels can read, with its address and first three strides
    (that of a dimension of one is of no interest)."""
    a, b, n, d = t.stride()
    ptr = t.data_ptr()
    if N == 1:
        n = 0
    if d != 1 or (a | b | n) & 7 or ptr & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        a, b, n, d = t.stride()
        ptr = t.data_ptr()
    return t, ptr, a, b, n


def _refuse(device: int, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise NotImplementedError(
                    "the paged cache has no gradient (inference only): call it under torch.no_grad()")
    if device < 0:
        raise RuntimeError("moa_b200 runs on CUDA tensors only (there is no CPU path)")


def _launch(name: str, entry, arguments, device: int) -> None:
    """``entry(arguments(stream), stream)`` on the device's current stream, with the device current; ``arguments``
    packs the struct once the stream is known (the scratch belongs to it)."""
    if _lib.NVTX or torch.cuda.current_device() != device:
        with torch.cuda.device(device), _lib.nvtx_range("moa_b200." + name):
            stream = _raw_stream(device)
            status = entry(arguments(stream), stream)
    else:
        stream = _raw_stream(device)
        status = entry(arguments(stream), stream)
    if status:
        _lib.check("moa_" + name, status)
    _touched.add(device)


def paged_append(key: Tensor, value: Tensor, key_pages: Tensor, value_pages: Tensor, page_table: Tensor,
                 lengths: Tensor, counts: Optional[Tensor] = None, rope: Optional[Tuple[Tensor, Tensor]] = None,
                 query: Optional[Tensor] = None, advance: bool = False) -> Optional[Tuple[Tensor, Tensor]]:
    """Puts the keys and values of new tokens into the pages of their sequences, in one launch.

    ``key, value``: ``(B, KV, N, D)``, read through their strides (last dim contiguous).  Token ``i`` of
    sequence ``b``, for ``i < min(counts[b], N)`` (``counts`` int32 ``(B,)``; none: all ``N``), goes to position
    ``p = lengths[b] + i``: slot ``p % page_size`` of page ``page_table[b, p // page_size]``.  The rows behind a
    count are padding.  ``lengths[b] < 0`` marks a row without a sequence; nothing of it is stored.

    ``key_pages, value_pages``: ``(num_pages, KV, page_size, D)``, any strides with a contiguous last dim (a pool
    that is ``(num_pages, page_size, KV, D)`` in memory is passed transposed); ``page_size`` a power of two.
    ``page_table``: int32 ``(B, max_pages)``; entries without a token may hold anything.  ``lengths``: int32
    ``(B,)``, tokens in the pages before the call; ``advance=True`` adds the appended ones (a second launch).

    ``rope=(cos, sin)``: the keys are rotated on the way (Llama ``rotate_half`` convention, fp32, rounded once).
    Tables are ``(positions, D)``, a row for every position, or ``(B, N, D)`` / ``(1, N, D)``, a row for every new
    token; in the tokens' dtype or float32.  With ``query`` ``(B, H, N, D)`` the rotated query and key are also
    returned, as contiguous ``(B, H, N, D)`` and ``(B, KV, N, D)`` (what a prompt's attention reads next); padding
    rows are zero there.  Otherwise nothing is returned.

    A token whose page (or row of a table by position) does not exist is not stored, and
    ``check_device_status()`` raises for it.  Two tokens of one call must not have the same place."""
    shape = key.shape
    assert len(shape) == 4 and value.shape == shape, "key and value must be (B, KV, N, D)"
    B, KV, N, D = shape
    dtype, device = key.dtype, key.get_device()
    pool = _pool_arguments(key_pages, value_pages, page_table, lengths, B, D, dtype, device)
    assert pool[10] == KV, "pages must be (num_pages, KV, page_size, D)"
    assert value.dtype is dtype and value.get_device() == device, "key and value must be alike"
    H = KV
    if query is not None:
        assert rope is not None, "a query is given to be rotated: rope is needed"
        shape = query.shape
        assert len(shape) == 4 and shape[0] == B and shape[2] == N and shape[3] == D, "query must be (B, H, N, D)"
        assert query.dtype is dtype and query.get_device() == device, "query and key must be alike"
        H = shape[1]
    counts_ptr = 0
    if counts is not None:
        assert counts.dtype is torch.int32 and counts.shape == (B,) and counts.is_contiguous(), \
            "counts must be contiguous int32 (B,)"
        assert counts.get_device() == device, "all tensors must be on the same device"
        counts_ptr = counts.data_ptr()
    r = _NO_ROPE if rope is None else _rope_arguments(rope, B, N, D, dtype, device)
    _refuse(device, key, value, query)
    result, qo, ko, q_ptr, qa, qb, qn = None, 0, 0, 0, 0, 0, 0
    if query is not None:
        result = query.new_empty((B, H, N, D)), query.new_empty((B, KV, N, D))
        qo, ko = result[0].data_ptr(), result[1].data_ptr()
        query, q_ptr, qa, qb, qn = _rows(query, N)
    if B == 0 or N == 0 or KV == 0:
        return result
    key, k_ptr, ka, kb, kn = _rows(key, N)
    value, v_ptr, va, vb, vn = _rows(value, N)
    _launch("paged_append", lib.moa_paged_append, lambda stream: _APPEND.pack(
        k_ptr, v_ptr, q_ptr, key_pages.data_ptr(), value_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
        counts_ptr, r[0], r[1], qo, ko, ka, kb, kn, va, vb, vn, qa, qb, qn, *pool[:10], *r[2:], B, H, KV, N, D,
        _DTYPES[dtype], advance), device)
    return result


def paged_decode(query: Tensor, key_pages: Tensor, value_pages: Tensor, page_table: Tensor, lengths: Tensor,
                 sm_scale: float, key: Optional[Tensor] = None, value: Optional[Tensor] = None,
                 rope: Optional[Tuple[Tensor, Tensor]] = None, sink_size: Optional[Tensor] = None,
                 local_size: Optional[Tensor] = None, out: Optional[Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None, advance: bool = False) -> Tensor:
    """Attention of one query token per sequence over the sequence's pages, in one launch.

    ``query``: ``(B, H, 1, D)``; ``H`` is a multiple of the pool's ``KV`` heads and query head ``h`` reads key head
    ``h // (H // KV)``.  Pool, ``page_table`` and ``lengths`` as in ``paged_append``.  Returns ``(B, 1, H, D)`` (into
    ``out`` if given, whose rows must be 16-byte aligned) in the query's dtype, or float32 with ``out_dtype=torch.float32`` (the unrounded result).

    ``sink_size, local_size``: int64 ``(KV,)`` in tokens, both or none; a head then attends only the first
    ``sink_size`` and last ``local_size`` tokens of a sequence (what a ring cache of that size holds), and only
    pages that hold some of them are read.  A head with nothing to attend gets zeros.

    Without ``key`` and ``value`` the first ``lengths[b]`` tokens are attended.  With them, ``(B, KV, 1, D)``, the new
    token is appended at position ``lengths[b]`` and attended too: the result of ``paged_append`` followed by this
    function with ``lengths + 1``, except that the rotated query is not rounded to its dtype in between.
    ``rope=(cos, sin)`` (tables as there, ``N = 1``) rotates query and key; ``advance=True`` adds one to the length
    of every sequence; ``lengths[b] < 0`` marks a row without a sequence: nothing is stored and its output is zero.

    Tokens whose page does not exist are left out, and ``check_device_status()`` raises for them."""
    shape = query.shape
    assert len(shape) == 4 and shape[2] == 1, "query must be (B, H, 1, D)"
    B, H, _, D = shape
    dtype, device = query.dtype, query.get_device()
    pool = _pool_arguments(key_pages, value_pages, page_table, lengths, B, D, dtype, device)
    KV = pool[10]
    assert KV > 0 and H % KV == 0, "the query heads must be a multiple of the pool's key/value heads"
    k_ptr = v_ptr = ka = kb = va = vb = 0
    r = _NO_ROPE
    if key is not None:
        assert value is not None, "key and value go together"
        shape = key.shape
        assert shape == (B, KV, 1, D) and value.shape == shape, "key and value must be (B, KV, 1, D)"
        assert key.dtype is dtype and value.dtype is dtype and device == key.get_device() == value.get_device(), \
            "query, key and value must be alike"
        if rope is not None:
            r = _rope_arguments(rope, B, 1, D, dtype, device)
        key, k_ptr, ka, kb, _ = _rows(key, 1)
        value, v_ptr, va, vb, _ = _rows(value, 1)
    else:
        assert value is None, "key and value go together"
        assert rope is None, "rope is for the step with a new token"
        assert not advance, "advance is for the step with a new token"
    assert (sink_size is None) == (local_size is None), "sink_size and local_size go together"
    sink_ptr = local_ptr = 0
    if sink_size is not None:
        for t in (sink_size, local_size):
            assert t.dtype is torch.int64 and t.shape == (KV,) and t.is_contiguous(), \
                "sink_size and local_size must be contiguous int64 (KV,)"
            assert t.get_device() == device, "all tensors must be on the same device"
        sink_ptr, local_ptr = sink_size.data_ptr(), local_size.data_ptr()
    _refuse(device, query, key, value)
    if out is None:
        if out_dtype is None or out_dtype is dtype:
            out = query.new_empty((B, 1, H, D))
        else:
            assert out_dtype is torch.float32, "out_dtype must be the query's dtype or float32"
            out = torch.empty((B, 1, H, D), dtype=torch.float32, device=query.device)
        oa, ob = H * D, D
    else:
        assert out.shape == (B, 1, H, D) and out.get_device() == device, "out must be (B, 1, H, D)"
        assert out.dtype is dtype or out.dtype is torch.float32, "out must have the query's dtype or be float32"
        assert out_dtype is None or out_dtype is out.dtype
        oa, _, ob, od = out.stride()
        assert od == 1, "rows of out must be contiguous"
    if B == 0 or H == 0:
        return out
    query, q_ptr, qa, qb, _ = _rows(query, 1)

    def arguments(stream):
        ws = _workspace(device, stream)
        return _DECODE.pack(
            q_ptr, k_ptr, v_ptr, key_pages.data_ptr(), value_pages.data_ptr(), out.data_ptr(), page_table.data_ptr(),
            lengths.data_ptr(), sink_ptr, local_ptr, r[0], r[1], ws.data_ptr(), qa, qb, ka, kb, va, vb, oa, ob,
            *pool[:10], *r[2:], B, H, KV, D, _DTYPES[dtype], out.dtype is torch.float32, advance, ws.numel(), sm_scale)

    _launch("paged_decode", lib.moa_paged_decode, arguments, device)
    return out


_STATUS = {31: ("moa_paged_append", "no page for a new token of sequence {0} at position {1}: it was not stored"),
           32: ("moa_paged_decode", "no page for position {1} of sequence {0} (head {2}): it was not attended"),
           33: ("moa_paged_append", "no rope row for a new token of sequence {0} at position {1}: it was not stored"),
           34: ("moa_paged_decode", "sequence {0} has {1} tokens, more than its row of the page table holds"),
           35: ("moa_paged_decode", "a load did not arrive (block {0}, thread {1}): the output is invalid")}


def check_status(device=None) -> None:
    """Raises ``MoaError`` when a paged call on ``device`` (none: on any) left a token out since the last look.
    Waits for the device; ``check_device_status`` calls it."""
    for index in sorted(_touched):
        if device is not None and device.index not in (None, index):
            continue
        words = torch.zeros(4, dtype=torch.int32)
        with torch.cuda.device(index):
            _lib.check("moa_paged_status", lib.moa_paged_status(words.data_ptr()))
        code, *where = words.tolist()
        if code:
            name, text = _STATUS.get(code, ("moa_paged_decode", "status {0} {1} {2}"))
            raise _lib.MoaError(name, 1, lib.moa_strerror(1).decode(), text.format(*where))
