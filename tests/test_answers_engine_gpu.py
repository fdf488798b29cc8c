"""Several answers to one prompt through the engine: shared prefixes, rules on the logits, grammars, log-probabilities, each alone and together, against
the plain implementation token by token."""
import math
import random

import pytest
import torch

import plain_llama as pl
from plain_rules import ruled

pytestmark = pytest.mark.gpu


@pytest.fixture()
def engines(model_folders):
    from mini_inference_engine_b200 import EngineConfig, LLMEngine

    def make(name="tiny_a", dtype=torch.float32, **cfg):
        cfg.setdefault("max_num_seqs", 8)
        cfg.setdefault("num_blocks", 120)
        cfg.setdefault("cuda_graph_batch_sizes", (1, 4, 8))
        return LLMEngine(model_folders[name], EngineConfig(**cfg), dtype=dtype, load_tokenizer=False, verbose=False)

    return make


@pytest.fixture()
def plain(model_folders):
    from mini_inference_engine_b200.weights import read_model_folder
    kept = {}

    def logits(name, ids, rnd=pl.identity):
        if name not in kept:
            kept[name] = (pl.read_config(model_folders[name]), {k: v.float() for k, v in read_model_folder(model_folders[name]).items()})
        return pl.forward(*kept[name], list(ids), rnd)[-1]

    return logits


@pytest.fixture()
def always_share(monkeypatch):
    from mini_inference_engine_b200.kernels import attention
    monkeypatch.setattr(attention, "SHARE_MIN_BYTES", 1)


def words(bits):
    w = [0] * (-(-len(bits) // 32))
    for i, b in enumerate(bits):
        w[i // 32] |= int(b) << (i % 32)
    return w


def check_answer(plain, name, prompt, out, params, tol, rnd=pl.identity, grammar=None):
    """Every token is the best under the request's rules, within ``tol`` of the largest logit; its log-probability as well."""
    ids = list(prompt)
    for k, tok in enumerate(out.output_ids):
        raw = plain(name, ids, rnd)
        mask = None
        if grammar is not None:
            got = grammar.allowed(ids[len(prompt):])
            if got is not None:
                bits = [False] * raw.numel()
                for t in got:
                    bits[t] = True
                mask = words(bits)
        x, _ = ruled(raw, ids, len(prompt), params.repetition_penalty, params.presence_penalty, params.frequency_penalty,
                     [(t, b) for t, b in (params.logit_bias or {}).items()], mask)
        slack = tol * raw.abs().max().item() * max(1.0, params.repetition_penalty, 1 / params.repetition_penalty)
        assert x[tok] > -math.inf and (params.temperature > 0 or x[tok] >= x.max() - 2 * slack), (k, tok, float(x[tok]), float(x.max()))
        if params.logprobs:
            assert abs(out.logprobs[k] - float(torch.log_softmax(x, 0)[tok])) <= 2 * slack + 1e-4
        ids.append(tok)


WAYS = [dict(), dict(max_num_batched_tokens=16), dict(use_cuda_graphs=False), dict(overlap_steps=False), dict(num_blocks=10)]


def test_penalties_and_biases_every_way(engines, plain):
    from mini_inference_engine_b200 import SamplingParams
    rng = random.Random(0)
    prompts = [[rng.randrange(256) for _ in range(n)] for n in (5, 30, 17, 40)]
    params = [SamplingParams(max_tokens=24, ignore_eos=True, repetition_penalty=1.6, logprobs=True),
              SamplingParams(max_tokens=20, ignore_eos=True, presence_penalty=0.8, frequency_penalty=0.4),
              SamplingParams(max_tokens=24, ignore_eos=True),
              SamplingParams(max_tokens=16, ignore_eos=True, frequency_penalty=1.0, logit_bias={7: 3.0, 9: -math.inf, 200: 0.5}, logprobs=True)]
    first = None
    for way in WAYS:
        eng = engines(**way)
        free = [p.num_free for p in eng.cache.pools]
        outs = eng.generate(prompts, params)
        if "num_blocks" in way:
            assert eng.scheduler.num_preemptions > 0
        got = [(o.output_ids, o.logprobs) for o in outs]
        if first is None:
            first = got
            for p, o, sp in zip(prompts, outs, params):
                check_answer(plain, "tiny_a", p, o, sp, 1e-4)
            assert outs[2].logprobs is None and len(outs[0].logprobs) == 24
        else:
            assert [g[0] for g in got] == [g[0] for g in first], way
            for (_, a), (_, b) in zip(got, first):
                assert a is None or max(abs(x - y) for x, y in zip(a, b)) < 1e-3
        assert [p.num_free for p in eng.cache.pools] == free and not eng.rules._held
    # and a request without rules is what it is without the others
    alone = engines().generate([prompts[2]], params[2])[0]
    assert alone.output_ids == first[2][0]


class Alternate:
    """Even and odd tokens in turn, ``length`` of them."""

    def __init__(self, vocab, length=10 ** 9):
        self.vocab, self.length, self.asked = vocab, length, []

    def allowed(self, ids):
        self.asked.append(list(ids))
        return [] if len(ids) >= self.length else range(len(ids) % 2, self.vocab, 2)


def test_grammars(engines, plain):
    from mini_inference_engine_b200 import SamplingParams
    rng = random.Random(1)
    prompts = [[rng.randrange(256) for _ in range(n)] for n in (6, 33, 20)]
    for way in WAYS[:4]:
        grammars = [Alternate(256), Alternate(256, 5), None]
        params = [SamplingParams(max_tokens=12, ignore_eos=True, grammar=grammars[0], logprobs=True),
                  SamplingParams(max_tokens=12, ignore_eos=True, grammar=grammars[1], repetition_penalty=1.3), SamplingParams(max_tokens=12, ignore_eos=True)]
        eng = engines(**way)
        outs = eng.generate(prompts, params)
        assert [len(o.output_ids) for o in outs] == [12, 5, 12]
        assert all(t % 2 == i % 2 for o in outs[:2] for i, t in enumerate(o.output_ids))
        for p, o, sp, g in zip(prompts, outs, params, grammars):
            check_answer(plain, "tiny_a", p, o, sp, 1e-4, grammar=g)
        assert [outs[0].output_ids[:k] for k in range(12)] == grammars[0].asked[:12]
        assert not eng.rules._held and eng.cache.num_free() == eng.cache.pools[0].num_usable


def test_a_grammar_that_allows_nothing_or_fails(engines):
    from mini_inference_engine_b200 import SamplingParams

    class Fails:
        def allowed(self, ids):
            if len(ids) == 2:
                raise KeyError("no rule")
            return None

    eng = engines()
    out = eng.generate([[1, 2, 3]], SamplingParams(max_tokens=5, grammar=Alternate(256, 0)))[0]
    assert out.output_ids == [] and out.ttft is None
    good = eng.add_request([5, 6, 7], SamplingParams(max_tokens=6, ignore_eos=True))
    bad = eng.add_request([5, 6, 7], SamplingParams(max_tokens=6, ignore_eos=True, grammar=Fails()))
    with pytest.raises(KeyError):
        while eng.has_work():
            eng.step()
    while eng.has_work():
        eng.step()
    assert len(good.output_ids) == 6 and len(bad.output_ids) == 2 and eng.cache.num_free() == eng.cache.pools[0].num_usable


@pytest.mark.parametrize("name,dtype", [("tiny_a", torch.float32), ("tiny_a", torch.bfloat16), ("tiny_d", torch.bfloat16), ("tiny_b", torch.bfloat16)])
def test_answers_that_share_a_prompt(engines, plain, always_share, monkeypatch, name, dtype):
    from mini_inference_engine_b200 import SamplingParams
    from mini_inference_engine_b200.kernels import ops
    calls = []
    shared = ops.shared_prefix_attention
    monkeypatch.setattr(ops, "shared_prefix_attention", lambda *a, **k: (calls.append(1), shared(*a, **k))[1])
    rng = random.Random(2)
    prompts = [[rng.randrange(131) for _ in range(n)] for n in (37, 64, 10, 50)]
    sp = SamplingParams(max_tokens=20, ignore_eos=True)
    rnd, tol = (pl.identity, 1e-4) if dtype == torch.float32 else (pl.round_bf16, 2e-2)
    for way in (dict(), dict(use_cuda_graphs=False), dict(max_num_seqs=3), dict(num_blocks=24)):
        eng = engines(name, dtype, **way)
        calls.clear()
        outs = eng.generate(prompts, sp, n=3)
        assert len(outs) == 12 and all(len(o.output_ids) == 20 for o in outs)
        for i, o in enumerate(outs):
            check_answer(plain, name, prompts[i // 3], o, sp, tol, rnd)
        assert bool(calls) == (dtype == torch.bfloat16)
        if dtype == torch.float32:                            # greedy answers to one prompt are one answer, and the one without sharing
            alone = engines(name, dtype).generate(prompts, sp)
            assert [o.output_ids for o in outs] == [alone[i // 3].output_ids for i in range(12)]
        if dtype == torch.bfloat16 and not way:
            assert any(g is not None for g in eng._shared_graphs.values())
        assert eng.cache.num_free() == eng.cache.pools[0].num_usable and eng.cache.pinned == [0] and not eng.prefixes
        eng.cache.check()


def test_requests_behind_a_system_prompt(engines, plain, always_share):
    """A prefix that is kept, requests that come and go, one that is the prefix itself, one that ends inside it."""
    from mini_inference_engine_b200 import SamplingParams
    eng = engines("tiny_d", torch.bfloat16)
    system = [(i * 37) % 1031 for i in range(70)]
    p = eng.add_prefix(system)
    assert len(p.token_ids) == 64 and eng.cache.pinned == [4]
    sp = SamplingParams(max_tokens=12, ignore_eos=True)
    prompts = [system + [3, 4], system[:64], system[:64] + [9], system[:40], system + [5] * 20]
    seqs = [eng.add_request(q, sp, prefix=p) for q in prompts]
    assert [s.prefix_pages for s in seqs] == [4, 3, 4, 2, 4]
    other = eng.add_request([1, 2, 3], sp)
    while eng.has_work():
        eng.step()

    class Out:
        pass

    for q, s in zip(prompts + [[1, 2, 3]], seqs + [other]):
        o = Out()
        o.output_ids = s.output_ids
        check_answer(plain, "tiny_d", q, o, sp, 2e-2, pl.round_bf16)
    late = eng.add_request(system + [8], sp, prefix=p)
    eng.step()
    eng.release_prefix(p)
    assert eng.cache.pinned == [4]                            # held by the request that runs
    with pytest.raises(ValueError, match="released"):
        eng.add_request(system + [8], sp, prefix=p)
    with pytest.raises(ValueError, match="released"):
        eng.release_prefix(p)
    while eng.has_work():
        eng.step()
    assert len(late.output_ids) == 12 and eng.cache.pinned == [0] and eng.cache.num_free() == eng.cache.pools[0].num_usable
    eng.cache.check()


def test_prefixes_that_are_refused(engines):
    from mini_inference_engine_b200 import SamplingParams
    eng = engines(num_blocks=11)
    with pytest.raises(ValueError, match="fills no page"):
        eng.add_prefix([1] * 15)
    with pytest.raises(ValueError, match="empty"):
        eng.add_prefix([])
    with pytest.raises(ValueError, match="vocabulary"):
        eng.add_prefix([1] * 16 + [4096])
    p = eng.add_prefix([1] * 32)
    with pytest.raises(ValueError, match="does not begin"):
        eng.add_request([1] * 31 + [2, 3], prefix=p)
    with pytest.raises(ValueError, match="does not begin"):
        eng.add_request([2], prefix=p)
    with pytest.raises(ValueError, match="logit_bias"):
        eng.add_request([1], SamplingParams(logit_bias={256: 1.0}))
    s = eng.add_request([1] * 100, SamplingParams(max_tokens=20), prefix=p)         # 8 pages, two of them shared
    with pytest.raises(ValueError, match="too few"):
        eng.add_prefix([1] * 64)
    with pytest.raises(ValueError, match="never fit"):
        eng.add_request([2] * 120, SamplingParams(max_tokens=40))                   # eight pages of its own beside the prefix
    while eng.has_work():
        eng.step()
    assert len(s.output_ids) >= 1
    eng.release_prefix(p)
    eng.cache.check()
    with pytest.raises(ValueError, match="n must"):
        eng.generate([[1]], n=0)


def test_models_with_state_do_not_share(tmp_path):
    from mini_inference_engine_b200 import EngineConfig, LLMEngine, SamplingParams
    from mini_inference_engine_b200.config import load_preset
    from mini_inference_engine_b200.weights import write_model_folder
    d = str(tmp_path)
    write_model_folder(d, load_preset("tiny-getizen"), 0)
    eng = LLMEngine(d, EngineConfig(max_num_seqs=4, num_blocks=60, use_cuda_graphs=False, warm_up_prompt_step=False), load_tokenizer=False, verbose=False)
    with pytest.raises(ValueError, match="cannot share"):
        eng.add_prefix([1] * 32)
    outs = eng.generate([[1, 2, 3] * 10], SamplingParams(max_tokens=4, ignore_eos=True), n=2)          # every answer for itself
    assert len(outs) == 2 and outs[0].output_ids == outs[1].output_ids


def test_all_together(engines, plain, always_share):
    """Sampled answers to two prompts behind shared pages, under penalties, a bias and a grammar, with log-probabilities: the same with and without graphs
    where the kernels are the same, and each token allowed, with its probability."""
    from mini_inference_engine_b200 import SamplingParams
    rng = random.Random(5)
    prompts = [[rng.randrange(1031) for _ in range(n)] for n in (70, 49)]
    got = []
    for way in (dict(), dict(overlap_steps=False)):
        eng = engines("tiny_d", torch.bfloat16, **way)
        grammars = [Alternate(1031), Alternate(1031, 9)]
        params = [SamplingParams(max_tokens=15, temperature=0.9, seed=11, ignore_eos=True, repetition_penalty=1.2, frequency_penalty=0.3, grammar=grammars[0], logprobs=True),
                  SamplingParams(max_tokens=15, temperature=0.7, seed=11, ignore_eos=True, presence_penalty=0.5, logit_bias={4: 2.0}, grammar=grammars[1], logprobs=True)]
        outs = eng.generate(prompts, params, n=4)
        assert [len(o.output_ids) for o in outs] == [15] * 4 + [9] * 4
        assert len({tuple(o.output_ids) for o in outs[:4]}) > 1          # the answers differ: each has a noise of its own
        for i, o in enumerate(outs):
            check_answer(plain, "tiny_d", prompts[i // 4], o, params[i // 4], 2e-2, pl.round_bf16, grammars[i // 4])
        got.append([len(o.output_ids) for o in outs])
        assert not eng.rules._held and eng.cache.num_free() == eng.cache.pools[0].num_usable
    assert got[0] == got[1]


def test_requests_with_seeds_of_their_own(engines, plain):
    from mini_inference_engine_b200 import SamplingParams
    eng = engines()
    params = [SamplingParams(max_tokens=8, temperature=0.8, seed=s, ignore_eos=True, repetition_penalty=1.3, logprobs=True) for s in (1, 2, 1)]
    outs = eng.generate([[4, 5, 6]] * 3, params)
    for o, sp in zip(outs, params):
        check_answer(plain, "tiny_a", [4, 5, 6], o, sp, 1e-4)


def test_command_line(model_folders, capsys):
    import json

    from mini_inference_engine_b200.__main__ import main
    main(["generate", "--model", model_folders["tiny_a"], "--prompt-ids", ",".join(["3"] * 20), "--max-tokens", "5", "--ignore-eos", "--n", "2",
          "--repetition-penalty", "1.4", "--logprobs"])
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines() if x.startswith("{")]
    assert len(lines) == 2 and lines[0]["output_ids"] == lines[1]["output_ids"] and len(lines[0]["logprobs"]) == 5
