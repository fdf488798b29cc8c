"""Several answers to one prompt, what the host decides of them: ``LLMEngine``'s own requests, prefixes, grammars and steps, without a device."""
import pytest

from host_engine import HostEngine
from mini_inference_engine_b200 import SamplingParams


class Upto:
    """Allows everything, then nothing (or fails) from ``length`` tokens on."""

    def __init__(self, length, fails=False):
        self.length, self.fails = length, fails

    def allowed(self, ids):
        if len(ids) < self.length:
            return None
        if self.fails:
            raise KeyError("no rule")
        return []


def whole(eng):
    """Nothing is held any more."""
    assert eng.cache.num_free() == eng.cache.pools[0].num_usable and eng.cache.pinned == [0] and not eng.prefixes and not eng.rules._held
    eng.cache.check()


@pytest.mark.parametrize("overlap", [True, False])
@pytest.mark.parametrize("first", ["count", "grammar"])
def test_a_grammar_that_fails_hides_nobody_else(overlap, first):
    """A request that ends where another's grammar fails -- by count in the step that is read for the grammars, or because its own allows nothing -- is returned by the next step."""
    eng = HostEngine(40, overlap_steps=overlap)
    params = dict(max_tokens=3) if first == "count" else dict(max_tokens=9, grammar=Upto(3))
    good = eng.add_request([5, 6, 7], SamplingParams(ignore_eos=True, **params))
    bad = eng.add_request([5, 6, 7], SamplingParams(max_tokens=9, ignore_eos=True, grammar=Upto(3, fails=True)))
    got, raised = [], 0
    while eng.has_work():
        try:
            got += eng.step()
        except KeyError:
            raised += 1
    assert raised == 1 and got == [good] and len(good.output_ids) == 3 and len(bad.output_ids) == 3 and bad.finish_time is not None
    assert good.output_ids == [3, 4, 5]
    whole(eng)


@pytest.mark.parametrize("when", ["waiting", "running"])
def test_a_request_that_is_ended_early_gives_everything_back(when):
    """``scheduler.finish`` ends a request wherever it is: its prefix and its rules' slot go back too."""
    eng = HostEngine(40, overlap_steps=False)
    p = eng.add_prefix(list(range(40)))
    assert eng.computed == [32]
    s = eng.add_request(list(range(40)), SamplingParams(max_tokens=9, repetition_penalty=1.2), prefix=p)
    if when == "running":
        eng.step()
        eng.rules._held[s.seq_id] = 0
        eng.rules._free.clear()
    eng.scheduler.finish(s)
    assert p.users == 0 and not eng.has_work() and eng.rules._free == ([0] if when == "running" else [])
    eng.scheduler.finish(s)                                   # once more: nothing happens
    assert p.users == 0
    eng.release_prefix(p)
    whole(eng)
