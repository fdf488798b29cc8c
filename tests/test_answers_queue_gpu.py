"""Several answers to more prompts than the cache holds at once, through the engine: the answers are those of each prompt alone."""
import random

import pytest
import torch

from test_answers_engine_gpu import always_share, engines  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("way", [dict(), dict(overlap_steps=False), dict(use_cuda_graphs=False), dict(max_num_batched_tokens=48)])
def test_prompts_that_do_not_fit_side_by_side(engines, always_share, way, dtype):  # noqa: F811
    from mini_inference_engine_b200 import SamplingParams
    rng = random.Random(3)
    prompts = [[rng.randrange(256) for _ in range(n)] for n in (100, 97, 64, 100, 9, 81)]
    sp = SamplingParams(max_tokens=40, ignore_eos=True, frequency_penalty=0.2, logprobs=True)
    eng = engines("tiny_a", dtype, num_blocks=20, **way)                # eight pages a request, six of them the prompt's, of nineteen
    outs = eng.generate(prompts, sp, n=3)
    assert [o.prompt_len for o in outs] == [len(p) for p in prompts for _ in range(3)]
    # (an answer ends with the longest sequence that the model takes)
    assert all(len(o.output_ids) == len(o.logprobs) == min(40, eng.cfg.max_model_len - o.prompt_len) and 0 <= o.ttft <= o.latency for o in outs)
    assert eng.cache.num_free() == eng.cache.pools[0].num_usable and not eng.prefixes and not eng.rules._held
    eng.cache.check()
    if dtype == torch.float32:                                # greedy, and no rounding that depends on what else runs
        alone = engines("tiny_a", dtype).generate(prompts, sp)
        assert [o.output_ids for o in outs] == [alone[i // 3].output_ids for i in range(18)]
