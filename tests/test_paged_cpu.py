"""Paged cache without a GPU: what the entry points refuse, and the layout of the argument structs."""
import ctypes
import os
import re

import pytest
import torch

import moa_b200
from moa_b200 import _lib, paged

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "moa_b200.h")


def _fields(name):
    """Field names of a struct of the header, in order."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    got = []
    for line in body.split(";"):
        line = re.sub(r"\b(const|void|int32_t|int64_t|double)\b", " ", line).replace("*", " ")
        got += [f.strip() for f in line.split(",") if f.strip()]
    return got


def test_packed_arguments_have_the_header_structs_size():
    assert paged._APPEND.size == 8 * len(_fields("moa_paged_append_args"))
    assert paged._DECODE.size == 8 * len(_fields("moa_paged_decode_args"))
    text = open(HEADER).read()
    assert int(re.search(r"MOA_PAGED_COUNTER_BYTES (\d+)", text).group(1)) == paged._COUNTER_BYTES


def _inputs(B=2, H=4, KV=2, N=1, D=64, page=16, dtype=torch.float16):
    return dict(query=torch.zeros(B, H, N, D, dtype=dtype), key=torch.zeros(B, KV, N, D, dtype=dtype),
                value=torch.zeros(B, KV, N, D, dtype=dtype), key_pages=torch.zeros(6, KV, page, D, dtype=dtype),
                value_pages=torch.zeros(6, KV, page, D, dtype=dtype), page_table=torch.zeros(B, 3, dtype=torch.int32),
                lengths=torch.zeros(B, dtype=torch.int32))


def _append(**changes):
    t = _inputs()
    t.update(changes)
    t.pop("query") if "query" not in changes else None
    return moa_b200.paged_append(**t)


def _decode(step=False, **changes):
    t = _inputs()
    if not step:
        t.pop("key"), t.pop("value")
    t.update(changes)
    return moa_b200.paged_decode(**t, sm_scale=0.1)


def test_cpu_tensors_are_rejected_not_silently_computed():
    for call in (_append, _decode, lambda: _decode(step=True)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


TABLE2 = torch.zeros(48, 64, dtype=torch.float16)
APPEND_BAD = {
    "key and value differ": dict(value=torch.zeros(2, 2, 2, 64).half()),
    "fp32": dict(key=torch.zeros(2, 2, 1, 64), value=torch.zeros(2, 2, 1, 64)),
    "value of another type": dict(value=torch.zeros(2, 2, 1, 64).bfloat16()),
    "pages of another type": dict(key_pages=torch.zeros(6, 2, 16, 64).bfloat16()),
    "other heads": dict(key_pages=torch.zeros(6, 3, 16, 64).half(), value_pages=torch.zeros(6, 3, 16, 64).half()),
    "pages differ": dict(value_pages=torch.zeros(7, 2, 16, 64).half()),
    "pages with rows that are not contiguous": dict(key_pages=torch.zeros(6, 2, 64, 16).half().transpose(2, 3)),
    "int64 page table": dict(page_table=torch.zeros(2, 3, dtype=torch.int64)),
    "page table of another batch": dict(page_table=torch.zeros(3, 3, dtype=torch.int32)),
    "page table by columns": dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t()),
    "int64 lengths": dict(lengths=torch.zeros(2, dtype=torch.int64)),
    "lengths of another batch": dict(lengths=torch.zeros(3, dtype=torch.int32)),
    "lengths apart": dict(lengths=torch.zeros(4, dtype=torch.int32)[::2]),
    "int64 counts": dict(counts=torch.zeros(2, dtype=torch.int64)),
    "counts of another batch": dict(counts=torch.zeros(1, dtype=torch.int32)),
    "query without tables": dict(query=torch.zeros(2, 4, 1, 64).half()),
    "query of another length": dict(query=torch.zeros(2, 4, 2, 64).half(), rope=(TABLE2, TABLE2)),
    "tables of another width": dict(rope=(TABLE2[:, :32], TABLE2[:, :32])),
    "tables of another type": dict(rope=(TABLE2.bfloat16(), TABLE2.bfloat16())),
    "tables of two shapes": dict(rope=(TABLE2, TABLE2[:5])),
    "tables of another batch": dict(rope=(torch.zeros(3, 1, 64).half(), torch.zeros(3, 1, 64).half())),
    "tables of another length": dict(rope=(torch.zeros(2, 2, 64).half(), torch.zeros(2, 2, 64).half())),
    "an empty table": dict(rope=(TABLE2[:0], TABLE2[:0])),
}
DECODE_BAD = {
    "two query tokens": dict(query=torch.zeros(2, 4, 2, 64).half()),
    "heads that do not divide": dict(query=torch.zeros(2, 5, 1, 64).half()),
    "another head size": dict(query=torch.zeros(2, 4, 1, 128).half()),
    "key without value": dict(key=torch.zeros(2, 2, 1, 64).half()),
    "tables without a new token": dict(rope=(TABLE2, TABLE2)),
    "advance without a new token": dict(advance=True),
    "sink without local": dict(sink_size=torch.zeros(2, dtype=torch.int64)),
    "int32 spans": dict(sink_size=torch.zeros(2, dtype=torch.int32), local_size=torch.zeros(2, dtype=torch.int32)),
    "spans by query head": dict(sink_size=torch.zeros(4, dtype=torch.int64), local_size=torch.zeros(4, dtype=torch.int64)),
    "int64 page table": dict(page_table=torch.zeros(2, 3, dtype=torch.int64)),
    "int64 lengths": dict(lengths=torch.zeros(2, dtype=torch.int64)),
    "pages of another type": dict(value_pages=torch.zeros(6, 2, 16, 64).bfloat16()),
}
STEP_BAD = {
    "key of another batch": dict(key=torch.zeros(1, 2, 1, 64).half(), value=torch.zeros(1, 2, 1, 64).half()),
    "two new tokens": dict(key=torch.zeros(2, 2, 2, 64).half(), value=torch.zeros(2, 2, 2, 64).half()),
    "key by query head": dict(key=torch.zeros(2, 4, 1, 64).half(), value=torch.zeros(2, 4, 1, 64).half()),
    "value of another type": dict(value=torch.zeros(2, 2, 1, 64).bfloat16()),
    "tables of another length": dict(rope=(torch.zeros(2, 2, 64).half(), torch.zeros(2, 2, 64).half())),
}


@pytest.mark.parametrize("what", APPEND_BAD)
def test_append_refuses(what):
    with pytest.raises(AssertionError):
        _append(**APPEND_BAD[what])


@pytest.mark.parametrize("what", DECODE_BAD)
def test_decode_refuses(what):
    with pytest.raises(AssertionError):
        _decode(**DECODE_BAD[what])


@pytest.mark.parametrize("what", STEP_BAD)
def test_step_refuses(what):
    with pytest.raises(AssertionError):
        _decode(step=True, **STEP_BAD[what])


def test_gradients_are_refused():
    key = torch.zeros(2, 2, 1, 64).half().requires_grad_()
    with pytest.raises(NotImplementedError, match="inference"):
        _append(key=key)
    with pytest.raises(NotImplementedError, match="inference"):
        _decode(query=torch.zeros(2, 4, 1, 64).half().requires_grad_())
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):     # and nothing else is wrong with the call
        _append(key=key)


# The C entry points check what they are given before anything is launched, so that the checks can be
# exercised with made-up (aligned, never read) addresses.
A = 4096
APPEND_OK = dict(k=A, v=A, k_pages=A, v_pages=A, page_table=A, lengths=A, k_sb=128, k_sh=64, k_sn=64, v_sb=128, v_sh=64,
                 v_sn=64, kp_page=2048, kp_head=1024, kp_slot=64, vp_page=2048, vp_head=1024, vp_slot=64, table_stride=3,
                 max_pages=3, num_pages=6, page_size=16, B=2, H=4, KV=2, N=1, D=64)
DECODE_OK = dict(q=A, k_pages=A, v_pages=A, out=A, page_table=A, lengths=A, workspace=A, q_sb=256, q_sh=64, o_sb=256,
                 o_sh=64, kp_page=2048, kp_head=1024, kp_slot=64, vp_page=2048, vp_head=1024, vp_slot=64, table_stride=3,
                 max_pages=3, num_pages=6, page_size=16, B=2, H=4, KV=2, D=64, workspace_bytes=1 << 40, sm_scale=0.1)


def _call_c(entry, packer, good, **changes):
    values = dict(good)
    values.update(changes)
    names = _fields("moa_%s_args" % entry)
    assert set(values) <= set(names)
    packed = packer.pack(*[values.get(n, 0) for n in names])
    return getattr(_lib.lib, "moa_" + entry)(packed, 0)


@pytest.mark.parametrize("changes,status,text", [
    (dict(k=0), 1, b"null"), (dict(k_pages=0), 1, b"null"), (dict(lengths=0), 1, b"null"), (dict(B=0), 1, b"shape"),
    (dict(B=65536), 1, b"shape"), (dict(N=0), 1, b"number of tokens"), (dict(num_pages=0), 1, b"page table"),
    (dict(max_pages=0), 1, b"page table"), (dict(page_size=24), 1, b"power of two"), (dict(page_size=1 << 17), 1, b"power of two"),
    (dict(k_pages=A + 8), 1, b"aligned"), (dict(kp_slot=68), 1, b"aligned"), (dict(v=A + 2), 1, b"aligned"),
    (dict(k_sn=-64), 1, b"aligned"), (dict(rope_cos=A), 1, b"go together"), (dict(rope_cos=A, rope_sin=A, rope_sn=60), 1, b"rope"),
    (dict(q=A), 1, b"go together"), (dict(q=A, q_out=A, k_out=A), 1, b"tables"), (dict(D=96), 2, b"head_dim"),
    (dict(dtype=7), 2, b"dtype"),
])
def test_append_entry_checks_its_arguments(changes, status, text):
    assert _call_c("paged_append", paged._APPEND, APPEND_OK, **changes) == status
    assert text in _lib.lib.moa_last_error_detail()


@pytest.mark.parametrize("changes,status,text", [
    (dict(q=0), 1, b"null"), (dict(out=0), 1, b"null"), (dict(page_table=0), 1, b"null"), (dict(KV=0), 1, b"shape"),
    (dict(H=5), 1, b"multiple"), (dict(k_new=A), 1, b"go together"), (dict(sink_size=A), 1, b"go together"),
    (dict(advance=1), 1, b"new token"), (dict(rope_cos=A, rope_sin=A), 1, b"new token"), (dict(q=A + 2), 1, b"aligned"),
    (dict(out=A + 8), 1, b"rows of out"), (dict(o_sh=68), 1, b"rows of out"), (dict(page_size=0), 1, b"power of two"), (dict(workspace=0), 4, b"workspace"), (dict(workspace_bytes=100), 4, b"workspace"),
    (dict(D=80), 2, b"head_dim"), (dict(dtype=2), 2, b"dtype"),
])
def test_decode_entry_checks_its_arguments(changes, status, text):
    assert _call_c("paged_decode", paged._DECODE, DECODE_OK, **changes) == status
    assert text in _lib.lib.moa_last_error_detail()


def test_null_arguments_are_an_error_not_a_crash():
    assert _lib.lib.moa_paged_append(None, 0) == 1
    assert _lib.lib.moa_paged_decode(None, 0) == 1
    assert _lib.lib.moa_paged_status(0) == 1
    assert ctypes.sizeof(ctypes.c_void_p) == 8


# ------------------------------------------------------------------------------------------- PagedCache, host side
def _cache(**changes):
    args = dict(num_layers=2, num_kv_heads=2, num_pages=6, batch_size=3, max_length=64, head_dim=64, page_size=16, device="cpu")
    args.update(changes)
    return moa_b200.PagedCache(**args)


def _held(cache):
    return [[p for p in row if p >= 0] for row in cache.page_table.tolist()]


def test_cache_hands_out_pages_once_and_takes_them_back():
    cache = _cache()
    assert cache.free_pages() == 6 and cache.page_table.shape == (3, 4) and cache.get_seq_length() == 0
    cache.reserve([16, 17, 0])
    held = _held(cache)
    assert [len(h) for h in held] == [1, 2, 0] and len(set(sum(held, []))) == 3 and cache.free_pages() == 3
    cache.reserve(1)                                  # the third slot has none yet, the others have room
    assert [len(h) for h in _held(cache)] == [1, 2, 1]
    assert _held(cache)[:2] == held[:2]
    cache.release(1)
    assert _held(cache)[1] == [] and cache.free_pages() == 4 and cache.sequence_lengths() == [0, -1, 0]
    assert cache.lengths[:, 1].tolist() == [-1, -1]
    cache.reserve(10)                                 # nothing for the idle slot
    assert _held(cache)[1] == []
    cache.admit(1)
    cache.reserve([0, 64, 0])
    assert cache.free_pages() == 0 and len(set(sum(_held(cache), []))) == 6


def test_cache_refuses_without_taking_anything():
    cache = _cache()
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.reserve([64, 33, 1])                    # 4 + 3 + 1 of 6
    with pytest.raises(ValueError, match="max_length"):
        cache.reserve([0, 65, 0])
    assert cache.free_pages() == 6 and _held(cache) == [[], [], []]
    with pytest.raises(IndexError):
        cache.release(3)
    with pytest.raises(IndexError):
        cache.slots(1, 4)
    with pytest.raises(AssertionError):
        cache.reserve([1, 1])
    for bad in (dict(page_size=48), dict(head_dim=96), dict(dtype=torch.float32), dict(static_size=[[1, 1], [1, 1]]),
                dict(static_size=[[1, 1]], circular_size=[[1, 1]]), dict(num_pages=0)):
        with pytest.raises(AssertionError):
            _cache(**bad)


def test_slots_are_a_view_with_shared_pages():
    cache = _cache()
    view = cache.slots(1, 3)
    view.reserve([20, 0])
    assert [len(h) for h in _held(cache)] == [0, 2, 0] and view.free_pages() == cache.free_pages() == 4
    view._count(0, [20, 5])
    assert cache.sequence_lengths(0) == [0, 20, 5] and view.get_seq_length() == 20 and view.slots(1, 2).sequence_lengths() == [5]
    view.release(0)
    assert cache.sequence_lengths(1) == [0, -1, 0] and cache.free_pages() == 6
    assert view.page_table.data_ptr() == cache.page_table[1].data_ptr()


def test_room_counts_layers_that_lag_behind():
    cache = _cache()
    cache._room(0, [16, 16, 16])
    cache._count(0, [16, 16, 16])
    cache._room(1, [16, 16, 16])                      # the second layer of the same step: no further pages
    assert cache.free_pages() == 3
    cache._count(1, [16, 16, 16])
    cache._room(0, [1, 1, 1])
    assert cache.free_pages() == 0


def test_cache_calls_check_their_states():
    cache = _cache()
    k = torch.zeros(3, 2, 5, 64).half()
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.update(k, k, 0)
    with pytest.raises(NotImplementedError):
        cache.update(k, k, 0, attention_mask=torch.ones(3, 5))
    with pytest.raises(AssertionError):
        cache.update(k[:2], k[:2], 0)
    with pytest.raises(AssertionError):
        cache.update(k.bfloat16(), k.bfloat16(), 0)
    with pytest.raises(AssertionError):
        cache.update(k, k, 0, counts=[1, 2])
    with pytest.raises(AssertionError):
        cache.update(k, k, 2)


def test_compiled_checks_leave_everything_else_to_python():
    """On tensors without a device, on things that are no tensors, and with too few arguments they answer None."""
    assert paged._host is not None, "moa_b200/_paged_host.so is not built"
    t = _inputs()
    pools = (t["key_pages"], t["value_pages"], t["page_table"], t["lengths"])
    assert paged._host.decode(t["query"], *pools, 0.1, None, None, None, None, None, None, None, False) is None
    assert paged._host.append(t["key"], t["value"], *pools, None, None, None, False) is None
    assert paged._host.decode(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14) is None
    assert paged._host.decode() is None and paged._host.append(None) is None
