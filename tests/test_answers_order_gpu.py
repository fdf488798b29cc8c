"""Steps in which a prompt's portion runs beside requests that decode, in every order that the batch may have: each request gets its own token and log-probability."""
import random

import pytest
import torch

from test_answers_engine_gpu import engines  # noqa: F401

pytestmark = pytest.mark.gpu

WAYS = [dict(), dict(overlap_steps=False), dict(use_cuda_graphs=False), dict(graph_prompt_portions=0), dict(max_num_batched_tokens=24), dict(split_step_max_tokens=4)]


def prompts_of(seed, lengths):
    rng = random.Random(seed)
    return [[rng.randrange(256) for _ in range(n)] for n in lengths]


def alone(engines, prompts, params):  # noqa: F811
    ref = engines()
    return [ref.generate([p], sp)[0] for p, sp in zip(prompts, params)]


def check(seqs, want):
    for s, o in zip(seqs, want):
        assert s.output_ids == o.output_ids
        if s.params.logprobs:
            assert max(abs(a - b) for a, b in zip(s.logprobs, o.logprobs)) < 1e-3


def options(rules):
    from mini_inference_engine_b200 import SamplingParams
    more = [dict(logprobs=True), dict(repetition_penalty=1.4), dict(), dict(logit_bias={5: 2.0}, logprobs=True)] if rules else [dict()] * 4
    return [SamplingParams(max_tokens=14, ignore_eos=True, **more[i % 4]) for i in range(12)]


@pytest.mark.parametrize("rules", [False, True])
@pytest.mark.parametrize("way", WAYS)
def test_a_portion_behind_a_prefix_beside_requests_without(engines, way, rules):  # noqa: F811
    """Rows of one prefix lie side by side, in front: a prompt behind a prefix comes before requests that decode and have none."""
    system = prompts_of(1, [33])[0]
    tails = prompts_of(2, [9, 1, 20, 5, 7, 16])
    prompts = [t if i % 2 else system + t for i, t in enumerate(tails)]
    params = options(rules)
    want = alone(engines, prompts, params)
    eng = engines(**way)
    prefix = eng.add_prefix(system)
    seqs = []
    for i, p in enumerate(prompts):                           # each joins those that decode already
        seqs.append(eng.add_request(p, params[i], prefix=None if i % 2 else prefix))
        for _ in range(2):
            eng.step()
    while eng.has_work():
        eng.step()
    check(seqs, want)
    eng.release_prefix(prefix)


@pytest.mark.parametrize("rules", [False, True])
@pytest.mark.parametrize("way", WAYS)
def test_a_prompt_of_one_token_behind_a_longer_one(engines, way, rules):  # noqa: F811
    """It runs as a decoding row does, and in front of the portion that it lies behind in the batch."""
    prompts = prompts_of(3, [12, 20, 1, 1, 15, 1])
    params = options(rules)
    want = alone(engines, prompts, params)
    eng = engines(**way)
    seqs = [eng.add_request(prompts[0], params[0])]
    eng.step()
    for i in range(1, 6):
        seqs.append(eng.add_request(prompts[i], params[i]))
        if i in (3, 5):
            eng.step()
    while eng.has_work():
        eng.step()
    check(seqs, want)


@pytest.mark.parametrize("way", WAYS)
def test_answers_whose_prompts_end_one_token_behind_a_page(engines, way):  # noqa: F811
    prompts = prompts_of(4, [33, 17, 40, 49, 65])
    params = options(True)[:5]
    want = alone(engines, prompts, params)
    outs = engines(**way).generate(prompts, params, n=2)
    assert [o.output_ids for o in outs] == [want[i // 2].output_ids for i in range(10)]
