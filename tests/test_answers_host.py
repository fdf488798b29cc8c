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


def prompts_of(count, tokens):
    return [[(i * 31 + k) % 4096 for k in range(tokens)] for i in range(count)]


def check_outputs(outs, prompts, n, tokens):
    assert [o.prompt_len for o in outs] == [len(p) for p in prompts for _ in range(n)]
    assert all(o.output_ids == list(range(o.prompt_len, o.prompt_len + tokens)) for o in outs)        # (the model's answers)


@pytest.mark.parametrize("overlap", [True, False])
@pytest.mark.parametrize("blocks,count", [(100, 12), (60, 5), (42, 3)])
def test_more_prompts_than_the_cache_holds_prefixes_for(overlap, blocks, count):
    """Requests of 40 pages, ten of them their prompt's: they fit one after another, and so do their prefixes."""
    prompts = prompts_of(count, 165)
    eng = HostEngine(blocks, overlap_steps=overlap, max_model_len=1024)
    outs = eng.generate(prompts, SamplingParams(max_tokens=475, ignore_eos=True), n=2)
    check_outputs(outs, prompts, 2, 475)
    assert eng.computed == [160] * count and all(o.ttft >= 0 and o.latency >= o.ttft for o in outs)
    whole(eng)


def test_every_place_is_filled():
    """Prompts are taken up to the most requests that run at once, short ones (no whole page) among them."""
    prompts = [p[:t] for p, t in zip(prompts_of(12, 40), (40, 16, 17, 3, 40, 33, 40, 40, 1, 40, 18, 40))]
    eng = HostEngine(200, max_num_seqs=9)
    outs = eng.generate(prompts, SamplingParams(max_tokens=6, ignore_eos=True), n=3)
    check_outputs(outs, prompts, 3, 6)
    assert len(eng.ran[0]) == 9 and eng.computed == [32, 16, 32, 32, 32, 32, 32, 16, 32]
    whole(eng)


def test_answers_beside_a_prefix_that_is_held():
    """Pages that a user's prefix holds are not the answers'."""
    eng = HostEngine(60, max_model_len=1024)
    p = eng.add_prefix(list(range(160)))
    prompts = prompts_of(4, 165)
    outs = eng.generate(prompts, SamplingParams(max_tokens=475, ignore_eos=True), n=2)
    check_outputs(outs, prompts, 2, 475)
    with pytest.raises(ValueError, match="never fit"):
        eng.generate(prompts_of(2, 165) + prompts_of(1, 320), SamplingParams(max_tokens=600, ignore_eos=True), n=2)
    eng.release_prefix(p)
    whole(eng)


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("bad,match", [([], "empty"), ([5000], "vocabulary"), ([1] * 2000, "max_model_len"), ([1] * 990, "never fit")])
def test_nothing_is_added_when_a_prompt_is_refused(n, bad, match):
    eng = HostEngine(50, max_model_len=1024)
    with pytest.raises(ValueError, match=match):
        eng.generate(prompts_of(2, 40) + [bad], SamplingParams(max_tokens=4), n=n)
    assert not eng.has_work() and eng.computed == []
    whole(eng)


@pytest.mark.parametrize("given", [dict(repetition_penalty=1e-46), dict(repetition_penalty=1e39), dict(presence_penalty=-1e39), dict(frequency_penalty=1e300),
                                   dict(logit_bias={3: 1e39})])
def test_numbers_that_float32_does_not_hold_are_refused(given):
    """The kernels' numbers are float32: a repetition penalty of 0 or infinity there makes NaN of some logits."""
    with pytest.raises(ValueError, match="float32"):
        SamplingParams(**given)


def test_numbers_at_the_ends_of_float32_are_taken():
    most, least = 3.4028234e38, 1e-45
    SamplingParams(repetition_penalty=most, presence_penalty=-most, frequency_penalty=most, logit_bias={3: most, 4: -most, 5: -1e300})
    SamplingParams(repetition_penalty=least)


def test_a_request_keeps_the_biases_that_it_was_added_with():
    """What the caller does to its dictionary afterwards does not reach a request: its list is on the device by then, as long as it was."""
    eng = HostEngine(40)
    given = SamplingParams(max_tokens=3, logit_bias={3: 1.0})
    s = eng.add_request([1, 2], given)
    given.logit_bias.update({4: 2.0, 10 ** 6: 1.0})
    assert s.params.logit_bias == {3: 1.0}
    given.logit_bias = {3: float("nan")}
    with pytest.raises(ValueError, match="logit_bias"):
        eng.add_request([1, 2], given)


def test_a_step_without_grammars_looks_at_no_request_for_them():
    """However many wait: a step's host work goes by the rows it runs."""
    eng = HostEngine(40, max_num_seqs=2, overlap_steps=False)
    for _ in range(50):
        eng.add_request([1, 2], SamplingParams(max_tokens=3))
    asked = []

    class Params:
        def __getattribute__(self, name):
            asked.append(name)
            return getattr(SamplingParams(max_tokens=3), name)

    for s in list(eng.scheduler.waiting)[2:]:
        s.params = Params()
    eng.step()
    assert asked == []


def test_grammars_are_asked_for_as_long_as_their_requests_live():
    eng = HostEngine(40)
    first, second = eng.add_request([1, 2], SamplingParams(max_tokens=3, grammar=Upto(9))), eng.add_request([1, 2], SamplingParams(max_tokens=9, grammar=Upto(5)))
    early = eng.add_request([1, 2], SamplingParams(max_tokens=9, grammar=Upto(9)))
    eng.scheduler.finish(early)
    assert list(eng._under_grammar) == [first.seq_id, second.seq_id]
    while eng.has_work():
        eng.step()
    assert not eng._under_grammar and len(first.output_ids) == 3 and len(second.output_ids) == 5 and early.mask_at == -1
    whole(eng)


def test_an_engine_ends_with_its_last_reference():
    """Nothing waits for the garbage collector, which may run while another engine captures its graphs: graphs that end then break that capture."""
    import gc
    import weakref
    gc.collect()
    gc.disable()
    try:
        eng = HostEngine(40)
        eng.generate(prompts_of(2, 40), SamplingParams(max_tokens=3, grammar=Upto(2)), n=2)
        p = eng.add_prefix(list(range(40)))
        s = eng.add_request(list(range(40)), prefix=p)
        eng.step()
        gone, scheduler = weakref.ref(eng), eng.scheduler
        del eng
        assert gone() is None and s.prefix is p
        scheduler.finish(s)                                   # nobody is left to hear of it
    finally:
        gc.enable()


def test_a_grammar_that_allows_only_what_is_banned_allows_nothing():
    """Else the choice, with nothing left to choose from, would return a token that the grammar forbids."""
    class Only:
        def allowed(self, ids):
            return [5, 7] if len(ids) < 2 else [5]

    eng = HostEngine(40)
    out, = eng.generate([[1, 2]], SamplingParams(max_tokens=9, grammar=Only(), logit_bias={5: -1e300, 7: -2.0}))
    assert len(out.output_ids) == 2
    eng.add_request([1, 2], SamplingParams(max_tokens=9, grammar=Only(), logit_bias={5: float("-inf")}))
    eng.step()
    s, = eng.scheduler.running
    assert s.mask.tolist()[0] == 1 << 7 and not s.mask[1:].any()


def test_options_of_a_class_of_the_callers_own():
    """A copy of a request's options is of their own class."""
    from dataclasses import dataclass

    @dataclass
    class Named(SamplingParams):
        name: str = ""

        def __post_init__(self):
            super().__post_init__()
            self.seen = True

    eng = HostEngine(400, max_model_len=64)
    s = eng.add_request([1] * 60, Named(max_tokens=50, logit_bias={3: 1.0}, name="a"))
    assert isinstance(s.params, Named) and s.params.name == "a" and s.params.max_tokens == 4 and s.params.seen
