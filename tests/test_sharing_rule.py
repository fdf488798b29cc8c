"""When a decoding step reads shared prefixes once a group: the rule's answer for steps whose both forms were measured and lie well apart, and what the engine asks it with."""
import pytest
import torch

from host_engine import HostEngine
from mini_inference_engine_b200 import SamplingParams
from mini_inference_engine_b200.kernels.attention import sharing_pays, sharing_weight

# kv heads, head size, rows, groups, prefix, mean own keys; us a layer by ordinary attention and with the prefixes shared
MEASURED = [
    (32, 64, 256, 5, 112, 1507, 566, 2059), (4, 64, 256, 1, 400, 450, 58.3, 93.8), (4, 64, 128, 1, 784, 450, 38.8, 54.5), (4, 64, 16, 8, 12304, 450, 40.3, 67.8),
    (4, 64, 64, 1, 784, 50, 14.6, 19.9), (4, 64, 32, 1, 1600, 50, 13.4, 19.6), (4, 64, 256, 1, 208, 50, 21.2, 31.5), (32, 64, 192, 1, 368, 116, 164.9, 195.7),
    (8, 128, 256, 1, 112, 450, 115.7, 169.0), (8, 128, 128, 1, 208, 450, 75.1, 92.2), (32, 128, 128, 1, 64, 450, 198.5, 255.1), (32, 128, 64, 4, 112, 450, 115.8, 155.4),
    (8, 128, 8, 1, 1760, 50, 15.3, 19.7), (32, 128, 32, 1, 112, 50, 25.2, 31.4), (8, 80, 256, 1, 112, 6, 27.9, 39.3),
    (4, 64, 64, 1, 4688, 50, 55.0, 26.8), (4, 64, 256, 1, 1168, 50, 60.3, 35.9), (4, 64, 16, 1, 13120, 50, 38.4, 28.8), (4, 64, 64, 4, 2464, 50, 32.3, 24.3),
    (8, 128, 64, 1, 8000, 256, 376, 43), (8, 128, 16, 1, 2464, 50, 32.6, 19.1), (8, 128, 64, 1, 400, 50, 31.1, 23.7), (8, 128, 32, 4, 1328, 450, 54.0, 37.6),
    (32, 128, 16, 1, 832, 50, 47.3, 29.0), (32, 128, 64, 1, 208, 50, 63.2, 41.7), (4, 96, 32, 4, 2736, 50, 41.9, 25.7), (8, 80, 16, 1, 2624, 50, 35.0, 18.2),
]


@pytest.mark.parametrize("kv,dim,rows,groups,prefix,own,ordinary,shared", MEASURED)
def test_the_faster_form_is_taken(kv, dim, rows, groups, prefix, own, ordinary, shared):
    per_key = 4 * kv * dim
    assert sharing_pays([(rows // groups, 0, prefix)] * groups, per_key, sharing_weight(dim, kv, rows, rows * own * per_key, groups * prefix * per_key)) == (shared < ordinary)


def step_of(own, rows=128, pages=50, alone=0):
    """Requests of ``own`` tokens behind a prefix of ``pages`` pages, and ``alone`` without it, in front of a decoding step."""
    eng = HostEngine(60000, max_model_len=4096, max_num_batched_tokens=1 << 20)
    eng.dtype, eng._kv_shape = torch.bfloat16, (8, 128)
    system = [7] * (pages * 16)
    p = eng.add_prefix(system)
    seqs = [eng.add_request(system + [1] * own, SamplingParams(max_tokens=50), prefix=p) for _ in range(rows)]
    seqs += [eng.add_request([1] * 4000, SamplingParams(max_tokens=50)) for _ in range(alone)]
    eng.step()
    assert all(s.num_computed == s.prompt_len for s in seqs)
    return eng._shared_step(seqs)


def test_the_engine_counts_what_lies_behind_the_prefixes():
    assert step_of(20) == [(128, 0, 800)]
    assert step_of(1500) is None                              # twice as many keys of the rows' own
    assert step_of(20, alone=128) is None                     # and those of rows that share nothing
