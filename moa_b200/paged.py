"""Paged key/value cache: append with the rotary embedding on the way, and attention of one new token.

The ring cache (``cache.py``) holds one token count for the whole batch and one ring per head.  A server
that answers many requests at once has sequences of different lengths that come and go, and models whose
query heads share key/value heads; its cache is a pool of pages that sequences take from and give back.
The kernels are ``csrc/paged.cu``; there is no CPU path and no gradient, as in the rest of the package.
"""
from __future__ import annotations

import copy
import ctypes
import importlib.util
import os
import struct
import sys
from typing import Dict, List, Optional, Sequence, Tuple

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
# paged_decode takes (sequence, key head) pairs a warp each when there are more than blocks (two per SM) and the page
# table reaches this many tokens at most
_MANY, _SHORT = 296, 256

# the stream's handle without a Stream object around it, as torch's own generated code asks for it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or _lib.current_stream
_capturing = torch.cuda.is_current_stream_capturing

#: the common case of both calls, compiled (csrc/paged_host.cpp) for one Python and one torch, as its name says
HOST_PATH = os.path.join(_lib.HERE, f"_paged_host.{sys.implementation.cache_tag}-torch{torch.__version__}.so")


def _load_host():
    """The compiled part, or None where there is none for this Python, torch and library: the same calls are then made
    from Python alone."""
    if not os.path.exists(HOST_PATH):
        return None
    spec = importlib.util.spec_from_file_location("moa_b200._paged_host", HOST_PATH)
    try:
        host = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(host)
    except ImportError:
        return None
    if getattr(host, "abi", None) != _lib.ABI_VERSION:
        return None
    host.init(ctypes.cast(lib.moa_paged_append, ctypes.c_void_p).value,
              ctypes.cast(lib.moa_paged_decode, ctypes.c_void_p).value)
    return host


_host = None if _lib.NVTX else _load_host()      # (ranges are marked from Python)

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
        if _host is not None:
            _host.seen(index, stream, ws.data_ptr(), ws.numel())
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
    if device not in _touched:
        _touched.add(device)
        if _host is not None:
            _host.seen(device, 0, 0, 0)


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
    if _host is not None:
        got = _host.append(key, value, key_pages, value_pages, page_table, lengths, counts, rope, query, advance)
        if got is not None:
            if got is True:
                return None
            if got.__class__ is int:
                _lib.check("moa_paged_append", got)
            return got
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
    ``out`` if given, whose rows must be 16-byte aligned) in the query's dtype, or float32 with ``out_dtype=torch.float32`` (the
    result before that rounding).  Scores, maxima and sums are fp32; a weight is held to 2^-22 of itself in fp16 (and 2^-39
    of the largest) and to 2^-17 of itself in bf16, the coordinates of a rotated query to 2^-22 (and 2^-25) and to 2^-16.
    Infinite values and keys give what the formula gives.

    ``sink_size, local_size``: int64 ``(KV,)`` in tokens, both or none; a head then attends only the first
    ``sink_size`` and last ``local_size`` tokens of a sequence (what a ring cache of that size holds), and only
    pages that hold some of them are read.  A head with nothing to attend gets zeros.

    Without ``key`` and ``value`` the first ``lengths[b]`` tokens are attended.  With them, ``(B, KV, 1, D)``, the new
    token is appended at position ``lengths[b]`` and attended too: the result of ``paged_append`` followed by this
    function with ``lengths + 1``, except that the rotated query is not rounded to its dtype in between.
    ``rope=(cos, sin)`` (tables as there, ``N = 1``) rotates query and key; ``advance=True`` adds one to the length
    of every sequence; ``lengths[b] < 0`` marks a row without a sequence: nothing is stored and its output is zero.

    Tokens whose page does not exist are left out, and ``check_device_status()`` raises for them."""
    if _host is not None:
        got = _host.decode(query, key_pages, value_pages, page_table, lengths, sm_scale, key, value, rope, sink_size,
                           local_size, out, out_dtype, advance)
        if got is not None:
            if got.__class__ is int:
                _lib.check("moa_paged_decode", got)
            return got
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


class PagedCache:
    """Keys and values of a batch of sequences that grow, end and begin independently, in a pool of pages.

    Beside ``StaticCircularCache``: a slot of the batch has its own length and takes pages as it grows; query
    heads may share ``num_kv_heads`` key/value heads; ``update`` and ``decode_attention`` are called the same way, so
    that ``MoAAttention`` and ``MoALlamaModel`` take either cache.  With ``static_size`` and ``circular_size``
    (``[layer][head]``, in tokens) a head attends the first and the last of its sequence's tokens only, as a
    ring of that size would; without them every token.

    Host and device keep the lengths side by side: the kernels advance ``lengths`` ``(num_layers, batch_size)``,
    the host counts along to hand out pages.  ``page_table`` ``(batch_size, max_length / page_size)`` and ``lengths``
    stay where they are, so a captured decode step can be replayed while ``reserve`` hands out pages between
    replays.  All calls of one cache belong on one stream."""

    def __init__(self, num_layers: int, num_kv_heads: int, num_pages: int, batch_size: int = 1, max_length: int = 4096,
                 head_dim: int = 128, page_size: int = 64, static_size: Optional[List[List[int]]] = None,
                 circular_size: Optional[List[List[int]]] = None, device="cuda",
                 dtype: torch.dtype = torch.float16) -> None:
        assert dtype in _DTYPES, f"the paged cache supports float16 and bfloat16 only, got {dtype}"
        assert head_dim in (64, 128), "head_dim must be 64 or 128"
        assert page_size > 0 and page_size & (page_size - 1) == 0, "page_size must be a power of two"
        assert num_layers > 0 and num_kv_heads > 0 and num_pages > 0 and batch_size > 0 and max_length > 0
        assert (static_size is None) == (circular_size is None), "static_size and circular_size go together"
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.num_layers, self.num_kv_heads, self.head_dim, self.page_size = num_layers, num_kv_heads, head_dim, page_size
        self.batch_size, self.device, self.dtype = batch_size, device, dtype
        self.static_cache_size = self.circular_cache_size = [None] * num_layers
        if static_size is not None:
            for sizes in (static_size, circular_size):
                assert len(sizes) == num_layers and all(len(row) == num_kv_heads for row in sizes), \
                    "static_size and circular_size must be [layer][key/value head]"
            self.static_cache_size = [torch.tensor(row, dtype=torch.int64, device=device) for row in static_size]
            self.circular_cache_size = [torch.tensor(row, dtype=torch.int64, device=device) for row in circular_size]
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        self.key_pages = [torch.empty(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.value_pages = [torch.empty(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        width = -(-max_length // page_size)
        self.page_table = torch.full((batch_size, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(num_layers, batch_size, dtype=torch.int32, device=device)
        # shared by the views that slots() makes
        self._first = 0
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(batch_size)]
        self._tokens: List[List[int]] = [[0] * batch_size for _ in range(num_layers)]     # -1: no sequence

    # ------------------------------------------------------------------ slots and pages
    def slots(self, first: int, last: int) -> "PagedCache":
        """This cache's slots ``first .. last - 1`` as a cache of their own, on the same pages: a prompt can be taken
        in there while the other slots wait."""
        if not 0 <= first < last <= self.batch_size:
            raise IndexError(f"slots {first} .. {last - 1} of {self.batch_size}")
        view = copy.copy(self)
        view.batch_size, view._first = last - first, self._first + first
        view.page_table, view.lengths = self.page_table[first:last], self.lengths[:, first:last]
        return view

    def free_pages(self) -> int:
        return len(self._free)

    def get_seq_length(self, layer_idx: Optional[int] = 0) -> int:
        """Tokens of the longest sequence."""
        return max(max(n, 0) for n in self.sequence_lengths(layer_idx))

    def sequence_lengths(self, layer_idx: int = 0) -> List[int]:
        """Tokens in every slot as the host counts them, -1 for a slot without a sequence."""
        return self._tokens[layer_idx][self._first:self._first + self.batch_size]

    def positions(self, q_len: int) -> Tensor:
        """``(batch_size, q_len)`` positions of the next ``q_len`` tokens, from the lengths on the device."""
        at = torch.arange(q_len, device=self.device)
        return self.lengths[0].clamp(min=0).long()[:, None] + at

    def release(self, slot: int) -> None:
        """Ends the sequence in ``slot``: its pages go back to the pool, and the slot is idle until ``admit``."""
        self._set(slot, -1)

    def admit(self, slot: int) -> None:
        """Begins a new, empty sequence in ``slot`` (whatever was there is released)."""
        self._set(slot, 0)

    def _set(self, slot: int, tokens: int) -> None:
        if not 0 <= slot < self.batch_size:
            raise IndexError(f"slot {slot} of {self.batch_size}")
        self._free.extend(reversed(self._pages[self._first + slot]))
        self._pages[self._first + slot] = []
        for row in self._tokens:
            row[self._first + slot] = tokens
        self.page_table[slot].fill_(-1)
        self.lengths[:, slot].fill_(tokens)

    def reserve(self, tokens) -> None:
        """Pages for ``tokens`` more tokens (a number, or one per slot) in every slot that has a sequence.  All or
        nothing: raises without taking any page when the pool or a row of the page table is too small."""
        tokens = [tokens] * self.batch_size if isinstance(tokens, int) else [int(n) for n in tokens]
        assert len(tokens) == self.batch_size, "one number of tokens per slot"
        wanted = []
        for slot, more in enumerate(tokens):
            at = self._first + slot
            longest = max(row[at] for row in self._tokens)
            missing = -(-(longest + more) // self.page_size) - len(self._pages[at]) if longest >= 0 and more > 0 else 0
            if missing > 0:
                if len(self._pages[at]) + missing > self.page_table.shape[1]:
                    raise ValueError(f"slot {slot} would hold {longest + more} tokens: more than the cache's max_length")
                wanted.append((slot, missing))
        if not wanted:
            return
        if sum(missing for _, missing in wanted) > len(self._free):
            raise RuntimeError(f"out of pages: {sum(m for _, m in wanted)} wanted, {len(self._free)} free")
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("pages cannot be handed out while a graph is captured: reserve() them before")
        for slot, missing in wanted:
            pages = self._pages[self._first + slot]
            new = [self._free.pop() for _ in range(missing)]
            self.page_table[slot, len(pages):len(pages) + missing] = torch.tensor(new, dtype=torch.int32).to(self.device)
            pages.extend(new)

    def _room(self, layer_idx: int, counts: List[int]) -> None:
        """Pages for ``counts`` more tokens in the slots, if they are not there yet."""
        row = self._tokens[layer_idx]
        for slot, more in enumerate(counts):
            at = self._first + slot
            if row[at] >= 0 and row[at] + more > len(self._pages[at]) * self.page_size:
                longest = [max(r[self._first + s] for r in self._tokens) for s in range(self.batch_size)]
                self.reserve([max(row[self._first + s] + n - longest[s], 0) if row[self._first + s] >= 0 else 0
                              for s, n in enumerate(counts)])
                return

    def _count(self, layer_idx: int, counts: List[int]) -> None:
        row = self._tokens[layer_idx]
        for slot, more in enumerate(counts):
            if row[self._first + slot] >= 0:
                row[self._first + slot] += more

    # ------------------------------------------------------------------ the calls a layer makes
    def update(self, key_states: Tensor, value_states: Tensor, layer_idx: int, attention_mask: Optional[Tensor] = None,
               cache_kwargs: Optional[Dict] = None, counts: Optional[Sequence[int]] = None,
               rope: Optional[Tuple[Tensor, Tensor]] = None, query: Optional[Tensor] = None):
        """Appends ``(B, KV, q_len, D)`` states to the slots' sequences, of slot ``b`` the first ``counts[b]`` tokens (none:
        all); rows of idle slots are left alone, and it is an error when no slot can take what it is given.  ``rope`` and
        ``query`` as in ``paged_append``.  Returns the rotated query and key when a query is given, else the states it
        was given."""
        if attention_mask is not None:
            raise NotImplementedError("PagedCache.update: padding is told by counts, on the right")
        assert layer_idx < self.num_layers
        B, KV, N, D = key_states.shape
        assert (B, KV, D) == (self.batch_size, self.num_kv_heads, self.head_dim), "states must be (B, KV, q_len, D)"
        assert key_states.dtype == self.dtype and key_states.device == self.device, "states and cache must be alike"
        each = [N] * B if counts is None else [min(max(int(n), 0), N) for n in counts]
        assert len(each) == B, "one count per slot"
        given = [held for more, held in zip(each, self.sequence_lengths(layer_idx)) if more > 0]
        if given and max(given) < 0:
            raise RuntimeError("no slot that tokens are given for has a sequence: admit one first")
        self._room(layer_idx, each)
        on_device = None if counts is None else torch.tensor(each, dtype=torch.int32).to(self.device)
        got = paged_append(key_states, value_states, self.key_pages[layer_idx], self.value_pages[layer_idx],
                           self.page_table, self.lengths[layer_idx], counts=on_device, rope=rope, query=query, advance=True)
        self._count(layer_idx, each)
        return (key_states, value_states) if got is None else got

    def decode_attention(self, query_states: Tensor, key_states: Tensor, value_states: Tensor, layer_idx: int,
                         sm_scale: float, out: Optional[Tensor] = None, rope: Optional[Tuple[Tensor, Tensor]] = None,
                         out_dtype: Optional[torch.dtype] = None) -> Tensor:
        """One decode step of one layer in one launch, as ``StaticCircularCache.decode_attention``: rotate, append and
        attend over every slot's sequence with its new token.  ``rope``: this step's tables, ``(B, 1, D)`` or
        ``(B, D)``.  Rows of idle slots are zero; it is an error when every slot is idle.  A captured call replays on any lengths for which pages are
        reserved; the host's count is then the replayer's to keep (``DecodeGraph`` does)."""
        assert layer_idx < self.num_layers
        B = self.batch_size
        assert query_states.dtype == self.dtype and query_states.device == self.device, "states and cache must be alike"
        # (the first slot is looked at alone; a captured step is for the lengths that its replays find)
        if self._tokens[layer_idx][self._first] < 0 and max(self.sequence_lengths(layer_idx)) < 0 and \
                not (self.device.type == "cuda" and _capturing()):
            raise RuntimeError("no slot has a sequence to append to: admit one first")
        self._room(layer_idx, [1] * B)
        if rope is not None:
            rope = tuple(t.reshape(B, 1, self.head_dim) for t in rope)
        table = self.page_table
        if B * self.num_kv_heads > _MANY and self.page_size <= _SHORT < table.shape[1] * self.page_size and \
                max(self.sequence_lengths(layer_idx)) < _SHORT and not _capturing():
            # the kernel for many short sequences goes by the table's width (a captured step keeps all of it)
            table = table[:, :_SHORT // self.page_size]
        out = paged_decode(query_states, self.key_pages[layer_idx], self.value_pages[layer_idx], table,
                           self.lengths[layer_idx], sm_scale, key=key_states, value=value_states, rope=rope,
                           sink_size=self.static_cache_size[layer_idx], local_size=self.circular_cache_size[layer_idx],
                           out=out, out_dtype=out_dtype, advance=True)
        self._count(layer_idx, [1] * B)
        return out
