"""Slots without a sequence, through the model: what is refused, and that a captured step is not."""
import pytest
import torch

import moa_b200
from test_gpu_paged_model import _ids, _model

pytestmark = pytest.mark.gpu


def test_a_step_captured_while_every_slot_is_idle():
    model = _model()
    cache = model.model.new_paged_cache(2, 70, page_size=16)
    model(_ids(2, 40), past_key_values=cache)
    model(_ids(2, 1), past_key_values=cache)              # libraries initialise lazily
    cache.release(0), cache.release(1)
    with pytest.raises(RuntimeError, match="admit"):
        model(_ids(2, 1), past_key_values=cache)
    with pytest.raises(RuntimeError, match="admit"):
        model(_ids(1, 9), past_key_values=cache.slots(1, 2))
    graph = moa_b200.DecodeGraph(model, cache)
    assert cache.free_pages() == cache.page_table.numel() and cache.lengths.tolist() == [[-1, -1]] * 2
    graph.step(_ids(2, 1))                                # nothing to do, nothing done
    assert cache.lengths.tolist() == [[-1, -1]] * 2 and cache.sequence_lengths() == [-1, -1]
    cache.admit(1)
    model(_ids(1, 30, seed=4), past_key_values=cache.slots(1, 2))
    alone = model.model.new_paged_cache(1, 70, page_size=16)
    model(_ids(1, 30, seed=4), past_key_values=alone)
    for step in range(3):
        ids = _ids(2, 1, seed=10 + step)
        got = graph.step(ids)
        want, _ = model(ids[1:], past_key_values=alone)
        off = (got[1:].double() - want.double()).norm() / want.double().norm()
        assert off <= 52 * 2.0 ** -11                     # test_gpu_paged_model: two runs of a model
    assert cache.sequence_lengths() == [-1, 33] and cache.lengths.tolist() == [[-1, 33]] * 2
    moa_b200.check_device_status()
