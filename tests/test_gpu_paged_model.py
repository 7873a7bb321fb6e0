"""PagedCache through the model: the ring cache's results, and sequences that come and go.

Tolerance of the comparisons of two runs of a model: both round to fp16 at the same places of a layer (norm,
projection, rotation, attention, o_proj, two sums, norm, gate, up, product, down: 12), each rounding is off by 2^-11 at
most, and the runs' errors may point opposite ways: 2 * 12 * 2^-11 per layer of the norm of the result, with two layers
and the two roundings around them (embedding's norm, lm_head) 52 * 2^-11."""
import pytest
import torch

import moa_b200

pytestmark = pytest.mark.gpu
REL = 52 * 2.0 ** -11
PLAN = {"alphas": [[128, 64, 192, 128], [64, 128, 128, 256]], "betas": [[0.1, 0.0, 0.3, 0.5], [0.2, 0.0, 0.1, 0.4]]}


def _model(plan=PLAN):
    torch.manual_seed(3)
    model = moa_b200.MoALlamaForCausalLM(num_layers=2, hidden_size=512, num_heads=4, intermediate_size=1024,
                                         vocab_size=101, dtype=torch.float16, device="cuda")
    for p in model.parameters():
        if p.dim() > 1:
            p.data.normal_(0, 0.04)
    if plan is not None:
        model.set_mixture_of_attention(plan, moa_max_new_token=128)
    return model


def _near(a, b):
    a, b = a.double(), b.double()
    assert torch.isfinite(a).all()
    off = ((a - b).norm() / b.norm()).item()
    assert off <= REL, off


def _ids(*shape, seed=0):
    return torch.randint(0, 101, shape, generator=torch.Generator().manual_seed(seed)).cuda()


def test_paged_and_ring_cache_agree_through_the_model():
    model = _model()
    prompt = _ids(2, 300)
    a, ring = model(prompt)
    paged = model.model.new_paged_cache(2, 300, page_size=16)
    b, same = model(prompt, past_key_values=paged)
    assert same is paged and paged.sequence_lengths(1) == [300, 300] and paged.lengths.tolist() == [[300, 300]] * 2
    _near(b, a)
    for step in range(40):                    # far enough for the rings to drop tokens of the prompt
        ids = _ids(2, 1, seed=step)
        a, _ = model(ids, past_key_values=ring)
        b, _ = model(ids, past_key_values=paged)
        _near(b, a)
    assert paged.get_seq_length() == ring.get_seq_length() == 340
    moa_b200.check_device_status()


def test_graph_of_the_paged_step_equals_the_eager_step():
    model = _model()
    prompt = _ids(3, 70)
    one, two = model.model.new_paged_cache(3, 70, page_size=16), model.model.new_paged_cache(3, 70, page_size=16)
    for cache in (one, two):
        model(prompt, past_key_values=cache)
        model(_ids(3, 1, seed=9), past_key_values=cache)
    graph = moa_b200.DecodeGraph(model, two)
    assert two.sequence_lengths() == [71] * 3 and two.lengths.tolist() == [[71] * 3] * 2
    for step in range(40):                    # over page ends: pages are handed out between replays
        ids = _ids(3, 1, seed=step)
        a, _ = model(ids, past_key_values=one)
        b = graph.step(ids)
        assert torch.equal(a, b), step
    assert two.sequence_lengths() == [111] * 3 and two.lengths.tolist() == [[111] * 3] * 2
    moa_b200.check_device_status()


@pytest.mark.parametrize("plan", [PLAN, None])
def test_sequences_come_and_go(plan):
    """Four slots, prompts of different lengths taken in one by one, one released and its slot used again, an idle slot
    in between; every slot's logits are those of its sequence alone."""
    model = _model(plan)
    cache = model.model.new_paged_cache(4, 400, num_pages=40, page_size=16, max_length=256)
    prompts = {0: _ids(1, 33, seed=1), 1: _ids(1, 150, seed=2), 3: _ids(1, 2, seed=3)}
    cache.release(2)
    alone = {}

    def take(slot, prompt):
        view = cache.slots(slot, slot + 1)
        got, _ = model(prompt, past_key_values=view)
        alone[slot] = model.model.new_paged_cache(1, 400, max_length=256)
        want, _ = model(prompt, past_key_values=alone[slot])
        _near(got, want)

    for slot, prompt in prompts.items():
        take(slot, prompt)
    graph = None
    for step in range(30):
        if step == 6:
            graph = moa_b200.DecodeGraph(model, cache)
        if step == 10:
            cache.release(1)
            alone.pop(1)
        if step == 15:
            cache.admit(1)
            take(1, _ids(1, 90, seed=4))
        if step == 20:
            cache.admit(2)
            take(2, _ids(1, 1, seed=5))
        ids = _ids(4, 1, seed=100 + step)
        got = graph.step(ids) if graph is not None else model(ids, past_key_values=cache)[0]
        for slot in alone:
            want, _ = model(ids[slot:slot + 1], past_key_values=alone[slot])
            _near(got[slot:slot + 1], want)
    assert cache.sequence_lengths() == [63, 105, 11, 32]
    assert cache.lengths.tolist() == [[63, 105, 11, 32]] * 2
    assert cache.free_pages() == 40 - (4 + 7 + 1 + 2)
    moa_b200.check_device_status()


def test_prompt_into_a_used_slot_is_refused():
    model = _model()
    cache = model.model.new_paged_cache(1, 50)
    model(_ids(1, 20), past_key_values=cache)
    with pytest.raises(NotImplementedError, match="empty slots"):
        model(_ids(1, 20), past_key_values=cache)


def test_pages_run_out_before_anything_is_written():
    model = _model()
    cache = model.model.new_paged_cache(2, 50, num_pages=3, page_size=16, max_length=64)
    with pytest.raises(RuntimeError, match="out of pages"):
        model(_ids(2, 40), past_key_values=cache)
    assert cache.sequence_lengths() == [0, 0] and cache.free_pages() == 3 and cache.lengths.tolist() == [[0, 0]] * 2
    with pytest.raises(ValueError, match="max_length"):
        model(_ids(2, 65), past_key_values=cache)


def test_shared_key_heads_and_ragged_prompts_through_the_cache():
    """Grouped heads: padded prompts with counts, then steps; against attention in 64 bits over what the pages hold."""
    from test_gpu_paged import attention64, close, rotated64, tables

    class Held:
        pass

    B, H, KV, D = 3, 8, 2, 64
    cache = moa_b200.PagedCache(1, KV, 64, B, 200, D, 16, [[4, 0]], [[50, 90]], dtype=torch.bfloat16)
    gen = torch.Generator().manual_seed(1)
    normal = lambda *s: torch.randn(*s, generator=gen).bfloat16().cuda()
    cos, sin = tables(D, torch.arange(200), torch.float32)
    k, v = normal(B, KV, 60, D), normal(B, KV, 60, D)
    cache.update(k, v, 0, counts=[60, 7, 0], rope=(cos, sin))
    assert cache.sequence_lengths() == [60, 7, 0] and cache.lengths.tolist() == [[60, 7, 0]]
    for step in range(30):
        q, k, v = normal(B, H, 1, D), normal(B, KV, 1, D), normal(B, KV, 1, D)
        at = cache.lengths[0].long()
        rope = (cos[at], sin[at])             # (B, D), as the ring cache takes them
        out = cache.decode_attention(q, k, v, 0, 0.125, rope=rope, out_dtype=torch.float32)
    c = Held()
    c.B, c.H, c.KV, c.D, c.kp, c.vp = B, H, KV, D, cache.key_pages[0], cache.value_pages[0]
    c.places = lambda b, pos: (cache.page_table[b, pos // 16].long(), pos % 16)
    qr = rotated64(q, rope[0][:, None, None], rope[1][:, None, None])[0]
    ref, tol = attention64(c, qr, cache.lengths[0], 0.125, [4, 0], [50, 90])
    close(out, ref, tol)
    moa_b200.check_device_status()


def test_many_short_sequences_through_the_cache():
    """160 slots of two key heads each, grown over 256 tokens: the same as the pages hold, whichever kernel it takes."""
    from test_gpu_paged import attention64, close

    class Held:
        pass

    B, H, KV, D = 160, 4, 2, 64
    cache = moa_b200.PagedCache(1, KV, B * 5, B, 320, D, 64, dtype=torch.float16)
    gen = torch.Generator().manual_seed(2)
    normal = lambda *s: torch.randn(*s, generator=gen).half().cuda()
    counts = [int(n) for n in torch.randint(1, 254, (B,), generator=gen)]
    counts[5] = 253
    cache.update(normal(B, KV, 253, D), normal(B, KV, 253, D), 0, counts=counts)
    c = Held()
    c.B, c.H, c.KV, c.D, c.kp, c.vp = B, H, KV, D, cache.key_pages[0], cache.value_pages[0]
    c.places = lambda b, pos: (cache.page_table[b, pos // 64].long(), pos % 64)
    for step in range(6):                     # the longest sequence: 254 .. 259 tokens
        q, k, v = normal(B, H, 1, D), normal(B, KV, 1, D), normal(B, KV, 1, D)
        out = cache.decode_attention(q, k, v, 0, 0.125, out_dtype=torch.float32)
        ref, tol = attention64(c, q, cache.lengths[0], 0.125)
        close(out, ref, tol)
    assert cache.sequence_lengths() == [n + 6 for n in counts]
    moa_b200.check_device_status()
