"""Requests with and without prefixes, rules, grammars, noise and seeds of their own that come, go and are ended early in a random order, on caches that are too small for all of
them: each answers as it would alone, is returned once, and gives back everything it held."""
import itertools
import random

import pytest
import torch

import plain_llama as pl
from test_answers_engine_gpu import always_share, check_answer, engines, plain  # noqa: F401

pytestmark = pytest.mark.gpu


class Third:
    """Every third token is even, or odd."""

    def __init__(self, odd):
        self.odd = odd

    def allowed(self, ids):
        return None if len(ids) % 3 else range(self.odd, 256, 2)


def options(rng):
    from mini_inference_engine_b200 import SamplingParams
    return SamplingParams(max_tokens=rng.randint(1, 30), ignore_eos=rng.random() < 0.8, temperature=rng.choice([0, 0, 0.9]), seed=rng.choice([None, None, 7]),
                          repetition_penalty=rng.choice([1, 1, 1.4]), presence_penalty=rng.choice([0, 0, 0.4]), frequency_penalty=rng.choice([0, 0, 0.3]),
                          logit_bias=rng.choice([None, None, {5: 2.0, 9: -float("inf")}]), logprobs=rng.random() < 0.3,
                          grammar=Third(rng.randint(0, 1)) if rng.random() < 0.15 else None)


def live_through(eng, rng, count):
    """Runs ``count`` requests; returns those that ended by themselves as (request, prompt, options)."""
    prefixes, live, returned, early = [], [], set(), set()

    def report(ended):
        for s in ended:
            assert s.seq_id not in returned
            returned.add(s.seq_id)

    while len(live) < count or eng.has_work():
        dice = rng.random()
        if len(live) < count and dice < 0.35:
            base = rng.choice(prefixes + [None])
            ids = [] if base is None else list(base.token_ids) if rng.random() < 0.9 else list(base.token_ids[:rng.randint(1, len(base.token_ids))])
            ids += [rng.randrange(256) for _ in range(rng.randint(1, 25))]
            if base is not None and ids[:len(base.token_ids)] != base.token_ids[:len(ids)]:
                base = None
            sp = options(rng)
            try:
                live.append((eng.add_request(ids, sp, prefix=base), ids, sp))
            except ValueError as e:
                assert "never fit" in str(e) or "max_model_len" in str(e)
        elif len(live) < count and dice < 0.42:
            try:
                prefixes.append(eng.add_prefix([rng.randrange(256) for _ in range(rng.randint(16, 60))]))
            except ValueError as e:
                assert "pages" in str(e)
        elif dice < 0.47 and prefixes:
            eng.release_prefix(prefixes.pop(rng.randrange(len(prefixes))))
        elif dice < 0.5 and len(live) > 5:
            report(eng.drain())
            s = rng.choice(live)[0]
            if s.finish_time is None and s.status.name != "FINISHED":
                eng.scheduler.finish(s)
                early.add(s.seq_id)
        else:
            report(eng.step())
    for p in prefixes:
        eng.release_prefix(p)
    assert eng.cache.num_free() == eng.cache.pools[0].num_usable and eng.cache.pinned == [0] and not eng.rules._held and not eng._under_grammar
    eng.cache.check()
    whole = [entry for entry in live if entry[0].seq_id not in early]
    assert all(s.seq_id in returned for s, _, _ in whole)
    return whole


WAYS = [dict(), dict(overlap_steps=False), dict(use_cuda_graphs=False), dict(max_num_batched_tokens=24), dict(max_num_seqs=3)]


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("way", WAYS)
def test_float32(engines, monkeypatch, way, seed):  # noqa: F811
    """The same tokens as alone, drawn ones too: their noise goes by the request's number."""
    from mini_inference_engine_b200.engine import sequence
    rng = random.Random(seed)
    whole = live_through(engines(num_blocks=rng.choice([22, 40, 80]), **way), rng, 25)
    ref = engines()
    for s, ids, sp in whole:
        monkeypatch.setattr(sequence, "_ids", itertools.count(s.seq_id))
        o = ref.generate([ids], sp)[0]
        assert o.output_ids == s.output_ids, (sp, len(ids), s.num_preemptions, s.prefix_pages)
        if sp.logprobs:
            assert len(s.logprobs) == len(s.output_ids) and max((abs(a - b) for a, b in zip(o.logprobs, s.logprobs)), default=0) < 1e-3


@pytest.mark.parametrize("way", WAYS)
def test_bfloat16(engines, plain, always_share, way):  # noqa: F811
    rng = random.Random(9)
    for s, ids, sp in live_through(engines("tiny_a", torch.bfloat16, num_blocks=40, **way), rng, 20):
        if sp.temperature == 0:
            check_answer(plain, "tiny_a", ids, s, sp, 2e-2, pl.round_bf16, sp.grammar)
