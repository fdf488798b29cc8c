"""Several answers to one prompt, the parts that need no GPU: shared pages in the cache manager and the scheduler, groups in the batch, what the
sampling options refuse."""
import math

import numpy as np
import pytest
import torch

from mini_inference_engine_b200 import EngineConfig, SamplingParams
from mini_inference_engine_b200.cache.manager import CacheManager, GroupSpec, PageError, RequestCache
from mini_inference_engine_b200.engine.batch import BatchBuilder, BatchRow
from mini_inference_engine_b200.engine.prefix import Prefix, shared_groups
from mini_inference_engine_b200.engine.scheduler import Scheduler
from mini_inference_engine_b200.engine.sequence import Sequence
from mini_inference_engine_b200.kernels.attention import SHARE_MIN_BYTES, sharing_pays
from mini_inference_engine_b200.sampling.rules import mask_words


def manager(pages=40, groups=None, slots=0):
    return CacheManager(groups or [GroupSpec("full")], pages, 16, slots)


def made(m, tokens):
    p = Prefix(list(range(tokens)))
    assert m.reserve(p.cache, tokens)
    m.advance(p.cache, tokens)
    m.pin(p.cache)
    return p


def test_a_request_begins_with_a_prefix_and_leaves_it_alone():
    m = manager()
    p = made(m, 48)
    held = list(p.cache.tables[0])
    rc = RequestCache()
    m.adopt(rc, p.cache, 2)
    assert rc.num_computed == 32 and rc.tables == [held[:2]] and rc.table_arrays()[0].tolist() == held[:2]
    assert m.pages_needed(rc, 20) == [2] and m.reserve(rc, 20)
    assert rc.tables[0][:2] == held[:2] and not set(rc.tables[0][2:]) & set(held)
    m.advance(rc, 20)
    free = m.num_free()
    m.free(rc)
    assert m.num_free() == free + 2 and rc.shared == 0 and rc.num_computed == 0 and p.cache.tables[0] == held
    m.adopt(rc, p.cache, 3)                                   # after a preemption: once more
    assert rc.tables == [held]
    m.free(rc)
    m.pin(p.cache, False)
    m.free(p.cache)
    assert m.num_free() == 39 and m.pinned == [0]
    m.check()


def test_what_cannot_be_shared():
    m = manager()
    p = made(m, 32)
    rc = RequestCache()
    m.reserve(rc, 5)
    with pytest.raises(PageError):
        m.adopt(rc, p.cache, 1)
    with pytest.raises(PageError):
        m.adopt(RequestCache(), p.cache, 3)
    assert m.can_share()
    assert not manager(groups=[GroupSpec("full"), GroupSpec("window", window=8)]).can_share()
    assert not manager(groups=[GroupSpec("chunk", chunk=8)]).can_share()


def test_admission_counts_own_pages_only():
    m = manager(pages=12)                                     # 11 usable
    s = Scheduler(EngineConfig(max_num_seqs=8, max_num_batched_tokens=64), m)
    p = made(m, 64)                                           # 4 pages held
    assert not s.can_ever_fit(7 * 16) and s.can_ever_fit(6 * 16)              # 7 left, one in reserve
    assert s.can_ever_fit(10 * 16, shared=4) and not s.can_ever_fit(11 * 16, shared=4)
    assert not s.can_ever_fit(10 * 16, shared=4, pinned=1)
    seqs = []
    for i in range(3):
        q = Sequence(list(range(64)) + [7] * (3 + i), SamplingParams(max_tokens=4))
        q.prefix, q.prefix_pages = p, 4
        s.add(q)
        seqs.append(q)
    batch = s.schedule()
    assert [(q.seq_id, n) for q, n in batch] == [(q.seq_id, 3 + i) for i, q in enumerate(seqs)]        # the prefix counts as computed
    assert all(q.cache.tables[0][:4] == p.cache.tables[0] and len(q.cache.tables[0]) == 5 for q in seqs)
    s._push_out(seqs[2])
    assert seqs[2].cache.num_computed == 0 and m.num_free() == 5
    s.schedule()
    assert seqs[2].cache.shared == 4 and seqs[2].cache.tables[0][:4] == p.cache.tables[0]
    for q in seqs:
        s.finish(q)
    assert m.num_free() == 7
    m.check()


def test_groups_of_rows():
    a, b = Prefix([0] * 32), Prefix([0] * 16)

    def row(prefix, pages):
        q = Sequence([1], SamplingParams())
        q.prefix, q.cache.shared = prefix, pages
        return q

    rows = [row(a, 2), row(a, 2), row(a, 1), row(None, 0), row(b, 1), row(b, 0), row(b, 1), row(b, 1)]
    assert shared_groups(rows, 16) == [(2, 0, 32), (1, 2, 16), (1, 4, 16), (2, 6, 16)]
    assert shared_groups([row(None, 0)], 16) == [] and shared_groups([], 16) == []


def test_groups_travel_with_the_step():
    b = BatchBuilder(1, 16, "cpu")
    rows = [BatchRow([5], 40 + i, [np.arange(1, 5, dtype=np.int32)], 0, (0,)) for i in range(6)]
    buf, layout = b.pack(rows, pad_rows=8, table_width=4, shared=[(2, 1, 32), (2, 4, 16)], most_groups=3)
    ctx = b.to_device(buf, layout)
    assert ctx.prefix.start.tolist() == [1, 3, 4, 6, 6, 6, 6] and ctx.prefix.length.tolist() == [32, 0, 16, 0, 0, 0]
    plain, plain_layout = b.pack(rows, pad_rows=8, table_width=4)
    assert b.to_device(plain, plain_layout).prefix is None and plain_layout["size"] < layout["size"]
    for bad in ([(2, 1, 16), (2, 2, 16)], [(3, 4, 16)]):
        with pytest.raises(ValueError, match="groups"):
            b.pack(rows, shared=bad)


def test_when_sharing_pays():
    assert not sharing_pays([(1, 0, 10 ** 9)], 1024)          # alone with its prefix
    n = SHARE_MIN_BYTES // 1024
    assert sharing_pays([(2, 0, n)], 1024) and not sharing_pays([(2, 0, n - 1)], 1024) and sharing_pays([(2, 0, n // 2), (3, 2, n // 4)], 1024)


@pytest.mark.parametrize("given", [dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=math.inf), dict(presence_penalty=math.nan),
                                   dict(frequency_penalty=math.inf), dict(logit_bias={-1: 1.0}), dict(logit_bias={0.5: 1.0}), dict(logit_bias={3: math.nan}),
                                   dict(logit_bias={3: math.inf}), dict(grammar=object())])
def test_sampling_options_that_are_refused(given):
    with pytest.raises(ValueError):
        SamplingParams(**given)


def test_requests_with_rules():
    class G:
        def allowed(self, ids):
            return None

    assert not SamplingParams(temperature=0.7, seed=3).has_rules
    for given in (dict(repetition_penalty=1.1), dict(presence_penalty=-0.5), dict(frequency_penalty=0.1), dict(logit_bias={3: -math.inf}), dict(grammar=G()), dict(logprobs=True)):
        assert SamplingParams(**given).has_rules


def test_a_grammars_answer_as_words():
    assert mask_words(None, 40) is None
    assert mask_words([0, 33, 31], 40).tolist() == [1 - 2 ** 31, 2]
    assert mask_words({39}, 40).tolist() == [0, 128] and mask_words([], 40).tolist() == [0, 0] and mask_words(np.array([1, 1]), 40).tolist() == [2, 0]
    truth = np.zeros(40, dtype=bool)
    truth[32] = True
    assert mask_words(truth, 40).tolist() == [0, 1]
    for bad in ([40], [-1], np.ones(39, dtype=bool), [0.5], np.array([[1]])):
        with pytest.raises(ValueError):
            mask_words(bad, 40)
