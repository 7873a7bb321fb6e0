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

_workspaces: Dict = {}
_touched = set()      # devices that a paged call has run on


def _workspace(index: int, stream: int) -> Tensor:
    """Scratch of ``paged_decode``: kept per device and stream; a call that is being captured gets one of its own,
    from the graph's memory, so that two graphs never share one."""
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(lib.moa_paged_decode_workspace_bytes(), dtype=torch.uint8, device=index)
        ws[:_COUNTER_BYTES].zero_()
        return ws
    ws = _workspaces.get((index, stream))
    if ws is None:
        ws = _workspaces[index, stream] = torch.zeros(lib.moa_paged_decode_workspace_bytes(), dtype=torch.uint8,
                                                      device=index)
    return ws


# The checks below run on every call, and at decode sizes the host's share of a call is larger than the
# kernel's: they ask a tensor for each property once (get_device() instead of device, all strides at once).

def _pool_arguments(key_pages: Tensor, value_pages: Tensor, page_table: Tensor, lengths: Tensor, B: int, KV: int,
                    D: int, dtype, device: int):
    assert dtype in _DTYPES, f"the paged cache supports float16 and bfloat16 only, got {dtype}"
    shape = key_pages.shape
    assert len(shape) == 4 and value_pages.shape == shape and shape[1] == KV and shape[3] == D, \
        "pages must be (num_pages, KV, page_size, D)"
    assert key_pages.dtype is dtype and value_pages.dtype is dtype, "pages and tokens must have the same dtype"
    ks, vs = key_pages.stride(), value_pages.stride()
    assert ks[3] == 1 and vs[3] == 1, "rows of the pages must be contiguous"
    ts, width = page_table.stride(), page_table.shape
    assert len(width) == 2 and width[0] == B and page_table.dtype is torch.int32, "page_table must be int32 (B, max_pages)"
    assert ts[1] == 1 or width[1] == 1, "rows of page_table must be contiguous"
    _check_row_of_ints(lengths, B, device, torch.int32, "lengths must be contiguous int32 (B,)")
    assert key_pages.get_device() == device and value_pages.get_device() == device and \
        page_table.get_device() == device, "all tensors must be on the same device"
    return (ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], ts[0], width[1], shape[0], shape[2])


def _check_row_of_ints(t: Tensor, n: int, device: int, dtype, what: str) -> None:
    assert t.dtype is dtype and t.dim() == 1 and t.numel() == n and t.is_contiguous(), what
    assert t.get_device() == device, "all tensors must be on the same device"


def _rope_arguments(rope: Tuple[Tensor, Tensor], B: int, N: int, D: int, dtype, device: int):
    cos, sin = rope
    shape, stride = cos.shape, cos.stride()
    assert sin.shape == shape and sin.stride() == stride and stride[-1] == 1 and shape[-1] == D, \
        "rope tables must be two tensors of one shape and layout with rows of D"
    kind = cos.dtype
    assert sin.dtype is kind and (kind is dtype or kind is torch.float32), \
        "rope tables must have the tensors' dtype or be float32"
    assert cos.get_device() == device and sin.get_device() == device, "all tensors must be on the same device"
    if len(shape) == 2:
        assert shape[0] > 0, "a rope table by position needs rows"
        return (cos.data_ptr(), sin.data_ptr(), 0, stride[0], shape[0], kind is torch.float32)
    assert len(shape) == 3 and (shape[0] == 1 or shape[0] == B) and shape[1] == N, \
        "rope tables must be (positions, D), (B, N, D) or (1, N, D)"
    return (cos.data_ptr(), sin.data_ptr(), 0 if shape[0] == 1 else stride[0], stride[1], 0, kind is torch.float32)


def _rows(t: Tensor):
    """``t`` (.., .., N, D), or a copy of it whose rows the kernels can read, with its address and first three strides
    (that of a dimension of one is of no interest)."""
    a, b, n, d = t.stride()
    if t.shape[2] == 1:
        n = 0
    if d != 1 or (a | b | n) & 7 or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        a, b, n, d = t.stride()
    return t, t.data_ptr(), (a, b, n)


def _inference_only(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError("the paged cache has no gradient (inference only): call it under torch.no_grad()")


def _cuda_only(device: int) -> None:
    if device < 0:
        raise RuntimeError("moa_b200 runs on CUDA tensors only (there is no CPU path)")


def _launch(name: str, entry, arguments, device: int) -> None:
    """``entry(arguments(stream), stream)`` on the device's current stream, with the device current; ``arguments``
    packs the struct once the stream is known (the scratch belongs to it)."""
    if _lib.NVTX or torch.cuda.current_device() != device:
        with torch.cuda.device(device), _lib.nvtx_range("moa_b200." + name):
            stream = torch.cuda.current_stream(device).cuda_stream
            status = entry(arguments(stream), stream)
    else:
        stream = torch.cuda.current_stream(device).cuda_stream
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
    pool = _pool_arguments(key_pages, value_pages, page_table, lengths, B, KV, D, dtype, device)
    assert value.dtype is dtype and value.get_device() == device, "key and value must be alike"
    H = KV
    if query is not None:
        assert rope is not None, "a query is given to be rotated: rope is needed"
        shape = query.shape
        assert len(shape) == 4 and shape[0] == B and shape[2] == N and shape[3] == D, "query must be (B, H, N, D)"
        assert query.dtype is dtype and query.get_device() == device, "query and key must be alike"
        H = shape[1]
    if counts is not None:
        _check_row_of_ints(counts, B, device, torch.int32, "counts must be contiguous int32 (B,)")
    r = _NO_ROPE if rope is None else _rope_arguments(rope, B, N, D, dtype, device)
    _inference_only(key, value, query)
    _cuda_only(device)
    result, q_ptr, q_strides, out_ptrs = None, 0, (0, 0, 0), (0, 0)
    if query is not None:
        result = (torch.empty((B, H, N, D), dtype=dtype, device=query.device),
                  torch.empty((B, KV, N, D), dtype=dtype, device=query.device))
        query, q_ptr, q_strides = _rows(query)
        out_ptrs = result[0].data_ptr(), result[1].data_ptr()
    if B == 0 or N == 0 or KV == 0:
        return result
    key, k_ptr, k_strides = _rows(key)
    value, v_ptr, v_strides = _rows(value)
    _launch("paged_append", lib.moa_paged_append, lambda stream: _APPEND.pack(
        k_ptr, v_ptr, q_ptr, key_pages.data_ptr(), value_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
        0 if counts is None else counts.data_ptr(), r[0], r[1], *out_ptrs, *k_strides, *v_strides, *q_strides, *pool,
        *r[2:], B, H, KV, N, D, _DTYPES[dtype], advance), device)
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
    KV = key_pages.shape[1]
    pool = _pool_arguments(key_pages, value_pages, page_table, lengths, B, KV, D, dtype, device)
    assert KV > 0 and H % KV == 0, "the query heads must be a multiple of the pool's key/value heads"
    k_ptr = v_ptr = 0
    k_strides = v_strides = (0, 0, 0)
    r = _NO_ROPE
    if key is not None:
        assert value is not None, "key and value go together"
        assert key.shape == (B, KV, 1, D) and value.shape == (B, KV, 1, D), "key and value must be (B, KV, 1, D)"
        assert key.dtype is dtype and value.dtype is dtype and key.get_device() == device and \
            value.get_device() == device, "query, key and value must be alike"
        if rope is not None:
            r = _rope_arguments(rope, B, 1, D, dtype, device)
        key, k_ptr, k_strides = _rows(key)
        value, v_ptr, v_strides = _rows(value)
    else:
        assert value is None, "key and value go together"
        assert rope is None, "rope is for the step with a new token"
        assert not advance, "advance is for the step with a new token"
    assert (sink_size is None) == (local_size is None), "sink_size and local_size go together"
    sink_ptr = local_ptr = 0
    if sink_size is not None:
        for t in (sink_size, local_size):
            _check_row_of_ints(t, KV, device, torch.int64, "sink_size and local_size must be contiguous int64 (KV,)")
        sink_ptr, local_ptr = sink_size.data_ptr(), local_size.data_ptr()
    _inference_only(query, key, value)
    _cuda_only(device)
    if out is None:
        assert out_dtype is None or out_dtype is dtype or out_dtype is torch.float32
        out = torch.empty((B, 1, H, D), dtype=out_dtype or dtype, device=query.device)
    else:
        assert out.shape == (B, 1, H, D) and out.stride(3) == 1 and out.get_device() == device, "out must be (B, 1, H, D)"
        assert out.dtype is dtype or out.dtype is torch.float32, "out must have the query's dtype or be float32"
        assert out_dtype is None or out_dtype is out.dtype
    if B == 0 or H == 0:
        return out
    query, q_ptr, q_strides = _rows(query)
    o_strides = out.stride()

    def arguments(stream):
        ws = _workspace(device, stream)
        return _DECODE.pack(
            q_ptr, k_ptr, v_ptr, key_pages.data_ptr(), value_pages.data_ptr(), out.data_ptr(), page_table.data_ptr(),
            lengths.data_ptr(), sink_ptr, local_ptr, r[0], r[1], ws.data_ptr(), q_strides[0], q_strides[1],
            k_strides[0], k_strides[1], v_strides[0], v_strides[1], o_strides[0], o_strides[2], *pool, *r[2:],
            B, H, KV, D, _DTYPES[dtype], out.dtype is torch.float32, advance, ws.numel(), sm_scale)

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
