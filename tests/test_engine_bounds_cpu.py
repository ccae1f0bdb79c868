"""The decode engine stays within its slots: a step or a prompt that would write
into another slot's part of the cache, or past the history, is refused on the
host (the steps themselves are graph replays; here they are counted)."""

import pytest
import torch

from harness import engine as E
from harness import model as H


class Replay:
    def __init__(self):
        self.count = 0

    def replay(self):
        self.count += 1


def make(max_slots=4, max_len=20, max_steps=12, kv_cache=""):
    m = H.build_model(H.TINY, dtype=torch.float32)
    H.init_dense(m, 3)
    eng = E.DecodeEngine(m, max_slots, max_len, max_steps, kv_cache=kv_cache, page_size=8)
    eng.graphs = {b: Replay() for b in eng.buckets}
    return eng


def prompts(*lens):
    return [torch.arange(n) % H.TINY.vocab_size for n in lens]


def test_steps_past_the_slot_are_refused():
    eng = make()
    eng.prefill(prompts(12, 15))
    with pytest.raises(ValueError, match="max_len"):
        eng.decode_steps([2] * 6)
    assert eng.graphs[2].count == 0  # none of them ran
    eng.decode_steps([2] * 5)
    assert eng.graphs[2].count == 5
    with pytest.raises(ValueError, match="max_len"):
        eng.decode_steps([2])
    eng.decode_steps([1] * 3)  # slot 0 alone has room for three more
    with pytest.raises(ValueError, match="max_len"):
        eng.decode_steps([1])
    eng.prefill(prompts(3))
    eng.decode_steps([1] * 12)
    assert eng.graphs[1].count == 15


def test_a_bucket_takes_its_other_slots_along():
    """Three requests run in the bucket of four; a slot left over from an
    earlier batch starts empty."""
    eng = make()
    eng.prefill(prompts(5, 5, 5, 19))
    with pytest.raises(ValueError, match="max_len"):
        eng.decode_steps([3, 3])
    eng.prefill(prompts(5, 5, 5))
    assert eng.positions.tolist() == [5, 5, 5, 0]
    eng.decode_steps([3] * 12)
    assert eng.graphs[4].count == 12


def test_steps_past_the_history_are_refused():
    eng = make(max_len=40)
    eng.prefill(prompts(2))
    eng.decode_steps([1] * 12)
    with pytest.raises(ValueError, match="max_steps"):
        eng.decode_steps([1])


@pytest.mark.parametrize("kv_cache", ["", "int8"])
def test_prompts_past_the_slot_are_refused(kv_cache):
    eng = make(kv_cache=kv_cache)
    with pytest.raises(ValueError, match="slots"):
        eng.prefill(prompts(21))
    with pytest.raises(ValueError, match="slots"):
        eng.prefill(prompts(1, 1, 1, 1, 1))


@pytest.mark.parametrize("kv_cache", ["", "int8"])
def test_capture_past_the_slot_is_refused(kv_cache):
    """A capture runs two steps first; behind a slot that is nearly full they
    would write into the next one."""
    eng = make(kv_cache=kv_cache)
    eng.held = [3, 19, 0, 0]
    with pytest.raises(ValueError, match="capture"):
        eng.capture()
    eng.held, eng.rows = [3, 18, 0, 0], 12
    with pytest.raises(ValueError, match="capture"):
        eng.capture()
