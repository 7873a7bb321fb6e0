"""Calls with a paged cache that must be refused before anything is written or handed out.  No GPU."""
import pytest
import torch

import moa_b200


def _attention(**changes):
    torch.manual_seed(0)
    attention = moa_b200.MoAAttention(128, 2, 0, dtype=torch.float16).eval()
    for name, value in changes.items():
        setattr(attention, name, value)
    return attention


def _cache(batch_size=2):
    return moa_b200.PagedCache(num_layers=1, num_kv_heads=2, num_pages=8, batch_size=batch_size, max_length=64, head_dim=64,
                               page_size=16, device="cpu")


def _attend(attention, cache, tokens):
    hidden = torch.zeros(cache.batch_size, tokens, 128, dtype=torch.float16)
    tables = tuple(torch.zeros(cache.batch_size, tokens, 64, dtype=torch.float16) for _ in range(2))
    return attention.attend(hidden, cache, tables)


def _state(cache):
    return cache.free_pages(), cache.sequence_lengths(), cache.lengths.tolist(), cache.page_table.tolist()


@pytest.mark.parametrize("idle", [[0], [1], [0, 1]])
def test_a_prompt_into_a_slot_without_a_sequence_is_refused(idle):
    cache = _cache()
    for slot in idle:
        cache.release(slot)
    before = _state(cache)
    with pytest.raises(RuntimeError, match="admit"):
        _attend(_attention(), cache, 5)
    assert _state(cache) == before
    one = cache.slots(idle[0], idle[0] + 1)
    with pytest.raises(RuntimeError, match="admit"):
        _attend(_attention(), one, 5)
    assert _state(cache) == before
    for slot in idle:
        cache.admit(slot)
    with pytest.raises(RuntimeError, match="CUDA"):       # and nothing else is wrong with the call
        _attend(_attention(), cache, 5)


def test_update_refuses_tokens_that_no_slot_can_take():
    cache = _cache()
    k = torch.zeros(2, 2, 5, 64).half()
    cache.release(0), cache.release(1)
    before = _state(cache)
    for counts in (None, [5, 0], [0, 3]):
        with pytest.raises(RuntimeError, match="admit"):
            cache.update(k, k, 0, counts=counts)
    assert _state(cache) == before
    cache.admit(1)
    with pytest.raises(RuntimeError, match="admit"):
        cache.update(k, k, 0, counts=[5, 0])
    # one of them can: rows of idle slots are left alone
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.update(k, k, 0)


@pytest.mark.parametrize("tokens", [1, 5])
def test_the_fused_gather_refuses_pages_before_anything_is_stored(tokens):
    cache = _cache()
    before = _state(cache)
    with pytest.raises(NotImplementedError, match="ring caches"):
        _attend(_attention(peer_gather=object()), cache, tokens)
    assert _state(cache) == before


def test_a_graph_over_pages_is_refused_with_the_fused_gather_before_pages_are_taken():
    model = moa_b200.MoALlamaModel(num_layers=2, hidden_size=128, num_heads=2, intermediate_size=64, vocab_size=11, device="cpu")
    model.layers[1].self_attn.peer_gather = object()
    cache = _cache()
    before = _state(cache)
    with pytest.raises(NotImplementedError, match="ring caches"):
        moa_b200.DecodeGraph(model, cache)
    assert _state(cache) == before


def test_a_capture_that_fails_leaves_the_lengths_as_they_were(monkeypatch):
    """The host counts a captured step's tokens and takes them back; also when the step raises half way."""
    import contextlib

    class Stream:
        def __init__(self, device=None):
            pass

        def wait_stream(self, other):
            pass

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", object)
    monkeypatch.setattr(torch.cuda, "graph", lambda graph, stream=None: contextlib.nullcontext())
    cache = moa_b200.PagedCache(2, 2, 8, 2, 64, 64, 16, device="cpu")
    cache.reserve([3, 16])
    for layer in range(2):
        cache._count(layer, [3, 16])

    class Model:
        device, layers, fails = torch.device("cpu"), [], True

        def __call__(self, ids, past_key_values):
            past_key_values._count(0, [1, 1])
            if self.fails:
                raise ValueError("layer 1")
            past_key_values._count(1, [1, 1])
            return ids, past_key_values

    model = Model()
    with pytest.raises(ValueError, match="layer 1"):
        moa_b200.DecodeGraph(model, cache)
    assert [cache.sequence_lengths(layer) for layer in range(2)] == [[3, 16]] * 2
    model.fails = False
    moa_b200.DecodeGraph(model, cache)
    assert [cache.sequence_lengths(layer) for layer in range(2)] == [[3, 16]] * 2


@pytest.mark.parametrize("entry,changes", [
    ("append", dict(page_table=2)), ("append", dict(lengths=2)), ("append", dict(counts=2)),
    ("decode", dict(page_table=2)), ("decode", dict(lengths=1)), ("decode", dict(sink_size=4, local_size=0)),
    ("decode", dict(sink_size=0, local_size=4)), ("decode", dict(workspace=8)),
])
def test_the_c_entries_refuse_addresses_that_a_kernel_cannot_read_at(entry, changes):
    from moa_b200 import _lib, paged
    from test_paged_cpu import A, APPEND_OK, DECODE_OK, _call_c

    good, packer = (APPEND_OK, paged._APPEND) if entry == "append" else (DECODE_OK, paged._DECODE)
    at = {name: A + off for name, off in changes.items()}
    assert _call_c("paged_" + entry, packer, good, **at) == 1
    assert b"aligned" in _lib.lib.moa_last_error_detail()


def test_a_token_for_a_cache_without_any_sequence_is_refused():
    """A prompt of one token takes the decode step's way."""
    cache = _cache()
    cache.release(1)
    before = _state(cache)
    with pytest.raises(RuntimeError, match="admit"):
        _attend(_attention(), cache.slots(1, 2), 1)
    assert _state(cache) == before
    with pytest.raises(RuntimeError, match="CUDA"):       # an idle slot beside another one: its row is zero
        _attend(_attention(), cache, 1)
    cache.release(0)
    with pytest.raises(RuntimeError, match="admit"):
        _attend(_attention(), cache, 1)
