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


def _workspace(device, stream: int) -> Tensor:
    """Scratch of ``paged_decode``: kept per device and stream; a call that is being captured gets one of its own,
    from the graph's memory, so that two graphs never share one."""
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(lib.moa_paged_decode_workspace_bytes(), dtype=torch.uint8, device=device)
        ws[:_COUNTER_BYTES].zero_()
        return ws
    key = (device.index, stream)
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = torch.zeros(lib.moa_paged_decode_workspace_bytes(), dtype=torch.uint8, device=device)
    return ws


def _pool_arguments(key_pages: Tensor, value_pages: Tensor, page_table: Tensor, lengths: Tensor, B: int, KV: int,
                    D: int, dtype, device):
    assert dtype in _DTYPES, f"the paged cache supports float16 and bfloat16 only, got {dtype}"
    assert key_pages.dim() == 4 and key_pages.shape == value_pages.shape, "pages must be (num_pages, KV, page_size, D)"
    num_pages, kv, page_size, d = key_pages.shape
    assert kv == KV and d == D, "pages must be (num_pages, KV, page_size, D)"
    assert key_pages.dtype == dtype and value_pages.dtype == dtype, "pages and tokens must have the same dtype"
    ks, vs = key_pages.stride(), value_pages.stride()
    assert ks[3] == 1 and vs[3] == 1, "rows of the pages must be contiguous"
    assert page_table.dim() == 2 and page_table.shape[0] == B and page_table.dtype == torch.int32, \
        "page_table must be int32 (B, max_pages)"
    assert page_table.stride(1) == 1 or page_table.shape[1] == 1, "rows of page_table must be contiguous"
    assert lengths.shape == (B,) and lengths.dtype == torch.int32 and lengths.is_contiguous(), \
        "lengths must be contiguous int32 (B,)"
    assert key_pages.device == device and value_pages.device == device and page_table.device == device and \
        lengths.device == device, "all tensors must be on the same device"
    return (ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], page_table.stride(0), page_table.shape[1], num_pages, page_size)


def _rope_arguments(rope: Tuple[Tensor, Tensor], B: int, N: int, D: int, dtype, device):
    cos, sin = rope
    assert cos.shape == sin.shape and cos.stride() == sin.stride() and cos.stride(-1) == 1 and cos.shape[-1] == D, \
        "rope tables must be two tensors of one shape and layout with rows of D"
    assert cos.dtype == sin.dtype and (cos.dtype == dtype or cos.dtype == torch.float32), \
        "rope tables must have the tensors' dtype or be float32"
    assert cos.device == device and sin.device == device, "all tensors must be on the same device"
    if cos.dim() == 2:
        assert cos.shape[0] > 0, "a rope table by position needs rows"
        where = (0, cos.stride(0), cos.shape[0])
    else:
        assert cos.dim() == 3 and cos.shape[0] in (1, B) and cos.shape[1] == N, \
            "rope tables must be (positions, D), (B, N, D) or (1, N, D)"
        where = (0 if cos.shape[0] == 1 else cos.stride(0), cos.stride(1), 0)
    return (cos.data_ptr(), sin.data_ptr(), *where, int(cos.dtype == torch.float32))


def _rows(t: Tensor) -> Tensor:
    """``t``, or a copy of it in rows that the kernels can read."""
    return t if _lib.rows_ok(t) else t.clone(memory_format=torch.contiguous_format)


def _inference_only(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError("the paged cache has no gradient (inference only): call it under torch.no_grad()")


def _on(device):
    """The device guard of a launch; nothing to do when it is the current device already."""
    return _lib.NO_RANGE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


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
    assert key.dim() == 4 and key.shape == value.shape, "key and value must be (B, KV, N, D)"
    B, KV, N, D = key.shape
    dtype, device = key.dtype, key.device
    pool = _pool_arguments(key_pages, value_pages, page_table, lengths, B, KV, D, dtype, device)
    assert value.dtype == dtype and value.device == device
    key, value = _rows(key), _rows(value)
    H, q_ptr, q_strides = KV, 0, (0, 0, 0)
    if query is not None:
        assert rope is not None, "a query is given to be rotated: rope is needed"
        assert query.dim() == 4 and query.shape[0] == B and query.shape[2:] == (N, D), "query must be (B, H, N, D)"
        assert query.dtype == dtype and query.device == device
        query = _rows(query)
        H, q_ptr, q_strides = query.shape[1], query.data_ptr(), query.stride()[:3]
    if counts is not None:
        assert counts.shape == (B,) and counts.dtype == torch.int32 and counts.is_contiguous(), \
            "counts must be contiguous int32 (B,)"
        assert counts.device == device, "all tensors must be on the same device"
    r = _NO_ROPE if rope is None else _rope_arguments(rope, B, N, D, dtype, device)
    _inference_only(key, value, query)
    if device.type != "cuda":
        raise RuntimeError("moa_b200 runs on CUDA tensors only (there is no CPU path)")
    result = None
    if query is not None:
        result = (torch.empty(B, H, N, D, dtype=dtype, device=device),
                  torch.empty(B, KV, N, D, dtype=dtype, device=device))
    if B == 0 or N == 0 or KV == 0:
        return result
    args = _APPEND.pack(
        key.data_ptr(), value.data_ptr(), q_ptr, key_pages.data_ptr(), value_pages.data_ptr(), page_table.data_ptr(),
        lengths.data_ptr(), _lib.ptr(counts), r[0], r[1], 0 if result is None else result[0].data_ptr(),
        0 if result is None else result[1].data_ptr(),
        *key.stride()[:3], *value.stride()[:3], *q_strides, *pool, *r[2:], B, H, KV, N, D, _DTYPES[dtype], advance)
    _touched.add(device.index)
    with _on(device), _lib.nvtx_range("moa_b200.paged_append"):
        status = lib.moa_paged_append(args, _lib.current_stream(device))
    if status:
        _lib.check("moa_paged_append", status)
    return result


def paged_decode(query: Tensor, key_pages: Tensor, value_pages: Tensor, page_table: Tensor, lengths: Tensor,
                 sm_scale: float, key: Optional[Tensor] = None, value: Optional[Tensor] = None,
                 rope: Optional[Tuple[Tensor, Tensor]] = None, sink_size: Optional[Tensor] = None,
                 local_size: Optional[Tensor] = None, out: Optional[Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None, advance: bool = False) -> Tensor:
    """Attention of one query token per sequence over the sequence's pages, in one launch.

    ``query``: ``(B, H, 1, D)``; ``H`` is a multiple of the pool's ``KV`` heads and query head ``h`` reads key head
    ``h // (H // KV)``.  Pool, ``page_table`` and ``lengths`` as in ``paged_append``.  Returns ``(B, 1, H, D)`` (into
    ``out`` if given) in the query's dtype, or float32 with ``out_dtype=torch.float32`` (the unrounded result).

    ``sink_size, local_size``: int64 ``(KV,)`` in tokens, both or none; a head then attends only the first
    ``sink_size`` and last ``local_size`` tokens of a sequence (what a ring cache of that size holds), and only
    pages that hold some of them are read.  A head with nothing to attend gets zeros.

    Without ``key`` and ``value`` the first ``lengths[b]`` tokens are attended.  With them, ``(B, KV, 1, D)``, the new
    token is appended at position ``lengths[b]`` and attended too: the result of ``paged_append`` followed by this
    function with ``lengths + 1``, except that the rotated query is not rounded to its dtype in between.
    ``rope=(cos, sin)`` (tables as there, ``N = 1``) rotates query and key; ``advance=True`` adds one to the length
    of every sequence; ``lengths[b] < 0`` marks a row without a sequence: nothing is stored and its output is zero.

    Tokens whose page does not exist are left out, and ``check_device_status()`` raises for them."""
    assert query.dim() == 4 and query.shape[2] == 1, "query must be (B, H, 1, D)"
    B, H, _, D = query.shape
    dtype, device = query.dtype, query.device
    KV = key_pages.shape[1]
    pool = _pool_arguments(key_pages, value_pages, page_table, lengths, B, KV, D, dtype, device)
    assert KV > 0 and H % KV == 0, "the query heads must be a multiple of the pool's key/value heads"
    q = _rows(query.select(2, 0))
    k_ptr = v_ptr = 0
    k_strides = v_strides = (0, 0)
    assert (key is None) == (value is None), "key and value go together"
    assert rope is None or key is not None, "rope is for the step with a new token"
    assert not advance or key is not None, "advance is for the step with a new token"
    if key is not None:
        assert key.shape == (B, KV, 1, D) and value.shape == (B, KV, 1, D), "key and value must be (B, KV, 1, D)"
        assert key.dtype == dtype and value.dtype == dtype and key.device == device and value.device == device
        k, v = _rows(key.select(2, 0)), _rows(value.select(2, 0))
        k_ptr, v_ptr, k_strides, v_strides = k.data_ptr(), v.data_ptr(), k.stride()[:2], v.stride()[:2]
    r = _NO_ROPE if rope is None else _rope_arguments(rope, B, 1, D, dtype, device)
    assert (sink_size is None) == (local_size is None), "sink_size and local_size go together"
    if sink_size is not None:
        for t in (sink_size, local_size):
            assert t.shape == (KV,) and t.dtype == torch.int64 and t.is_contiguous(), \
                "sink_size and local_size must be contiguous int64 (KV,)"
            assert t.device == device, "all tensors must be on the same device"
    _inference_only(query, key, value)
    if device.type != "cuda":
        raise RuntimeError("moa_b200 runs on CUDA tensors only (there is no CPU path)")
    if out is None:
        assert out_dtype is None or out_dtype == dtype or out_dtype == torch.float32
        out = torch.empty(B, 1, H, D, dtype=out_dtype or dtype, device=device)
    else:
        assert out.shape == (B, 1, H, D) and out.stride(3) == 1 and out.device == device
        assert out.dtype == dtype or out.dtype == torch.float32, "out must have the query's dtype or be float32"
        assert out_dtype is None or out_dtype == out.dtype
    if B == 0 or H == 0:
        return out
    o_strides = out.stride()
    _touched.add(device.index)
    with _on(device), _lib.nvtx_range("moa_b200.paged_decode"):
        stream = _lib.current_stream(device)
        ws = _workspace(device, stream)
        args = _DECODE.pack(
            q.data_ptr(), k_ptr, v_ptr, key_pages.data_ptr(), value_pages.data_ptr(), out.data_ptr(),
            page_table.data_ptr(), lengths.data_ptr(), _lib.ptr(sink_size), _lib.ptr(local_size), r[0], r[1],
            ws.data_ptr(), *q.stride()[:2], *k_strides, *v_strides, o_strides[0], o_strides[2], *pool, *r[2:],
            B, H, KV, D, _DTYPES[dtype], out.dtype == torch.float32, advance, ws.numel(), sm_scale)
        status = lib.moa_paged_decode(args, stream)
    if status:
        _lib.check("moa_paged_decode", status)
    return out


_STATUS = {31: ("moa_paged_append", "no page for a new token of sequence {0} at position {1}: it was not stored"),
           32: ("moa_paged_decode", "no page for position {1} of sequence {0} (head {2}): it was not attended"),
           33: ("moa_paged_append", "no rope row for a new token of sequence {0} at position {1}: it was not stored"),
           34: ("moa_paged_decode", "sequence {0} has {1} tokens, more than its row of the page table holds")}


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
