"""Shared prefixes read row by row, through the block table of a group's first row: the plan says so, and what the other kernels are tested for holds."""
import pytest
import torch

import test_shared_prefix_walk_gpu as walk
from test_shared_prefix_gpu import DEV, Case, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def row_by_row(monkeypatch):
    """Rows are taken one by one however much they share."""
    from mini_inference_engine_b200.kernels import ops
    monkeypatch.setattr(ops, "PREFIX_ONE_BY_ONE_BYTES", (1 << 40, 1 << 40))
    monkeypatch.setattr(ops, "PREFIX_ONE_BY_ONE_KEYS", 1 << 40)
    ops._shared_plan.cache_clear()
    yield
    ops._shared_plan.cache_clear()


def one_by_one(ops, c, **hints):
    return ops._shared_plan(torch.cuda.current_device(), c.rows, c.group_prefix.numel(), c.H, c.G, c.D, c.page, hints["max_prefix"], hints["max_own"],
                            c.cache.shape[1], 0)[1] == 2


# few and many splits, both merges, pages from 1 to 256, prefixes that end inside a page
@pytest.mark.parametrize("groups,own", [([(2, 1)], 1), ([(2, 64)], 64), ([(3, 129)], 200), ([(2, 0), (3, 100), (2, 0)], 40), ([(0, 90), (3, 90), (0, 0), (1, 33)], 10),
                                        ([(33, 777)], 20), ([(4, 5000)], [1, 700, 64, 1]), ([(2, 3000), (2, 10), (2, 901), (2, 1), (2, 2001)], 500),
                                        ([(64, 600)], 900), ([(3, 333), (2, 96)], [0, 4, 0, 0, 1]), ([(3, 250)], [0, 0, 0])])
@pytest.mark.parametrize("D,page", [(64, 16), (64, 128), (128, 8), (128, 64), (96, 16), (80, 64)])
def test_groups(ops, groups, own, D, page):
    c = Case(groups, own, 8, 2, D, page, seed=len(groups) + D)
    assert one_by_one(ops, c, **c.hints)
    out = c.run(ops, **c.hints)
    c.check(out)
    c.check(c.run(ops, dtype=torch.float32, **c.hints))
    assert torch.equal(out, c.run(ops, **c.hints))            # run to run: the same bits


@pytest.mark.parametrize("groups,own", [([(2, 1)], 1), ([(3, 129)], 200), ([(0, 90), (3, 90), (0, 0), (1, 33)], 10), ([(3, 333), (2, 96)], [0, 4, 0, 0, 1])])
def test_pages_of_one_position(ops, groups, own):
    c = Case(groups, own, 8, 2, 16, 1, seed=5)
    assert one_by_one(ops, c, **c.hints)
    c.check(c.run(ops, **c.hints))


@pytest.mark.parametrize("H,G,D,rows", [(32, 2, 64, 3), (8, 2, 128, 3), (8, 2, 64, 9), (8, 2, 96, 3)])
def test_a_prefix_whose_last_key_the_step_writes(ops, H, G, D, rows):
    walk.test_a_prefix_whose_last_key_the_step_writes(ops, H, G, D, rows)


@pytest.mark.parametrize("H,G,D", [(32, 2, 64), (4, 2, 128), (4, 2, 80)])
def test_groups_and_lengths_out_of_range_are_reported(ops, H, G, D):
    walk.test_groups_and_lengths_out_of_range_are_reported(ops, H, G, D)


def test_calls_on_two_streams_at_once(ops):
    walk.test_calls_on_two_streams_at_once(ops)


@pytest.mark.parametrize("D,groups,own", [(64, [(2, 6000), (1, 0)], 900), (80, [(3, 5000)], 700), (128, [(2, 900), (1, 40)], 500), (64, [(3, 100)], 20)])
def test_a_query_that_is_no_number_stays_in_its_head(ops, D, groups, own):
    c = Case(groups, own, 8, 2, D, 16, seed=D)
    assert one_by_one(ops, c, **c.hints)
    c.qkv[1, 3 * D + 1] = float("nan")
    out = c.run(ops, **c.hints)
    assert torch.isnan(out[1, 3]).all()
    out[1, 3] = 0
    assert torch.isfinite(out).all()
    c.check(out, [0, 2])


@pytest.mark.parametrize("D", [64, 128, 80])
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_the_first_rows_own_values_stay_its_own(ops, D, what):
    """They lie in the page in which the prefix ends; a row without own keys reads that page too."""
    c = Case([(3, 133)], [20, 0, 5], 4, 2, D, 16, seed=D)
    c.cache[1, int(c.tables[0, 8]), 1, 9, 7] = what            # key 137 of the first row
    out = c.run(ops, **c.hints)
    assert not torch.isfinite(out[0, 2:, 7]).any()
    out[0, 2:, 7] = 0
    assert torch.isfinite(out).all()
    c.check(out, [1, 2])


def test_rows_with_more_tokens_and_captured_groups(ops):
    cases = [Case([(3, 400), (2, 0)], 30, 8, 2, 64, 16, seed=1), Case([(1, 90), (4, 250)], 60, 8, 2, 64, 16, seed=2), Case([(5, 37)], [1, 0, 3, 60, 2], 8, 2, 64, 16, seed=3)]
    pages, width = max(c.cache.shape[1] for c in cases), max(c.tables.shape[1] for c in cases)
    s = Case([(3, 400), (2, 0)], 30, 8, 2, 64, 16, seed=1)
    s.cache, s.tables = torch.zeros(2, pages, 2, 16, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(5, width, dtype=torch.int32, device=DEV)
    s.group_start, s.group_prefix = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)

    def fill(c):
        s.cache.zero_()
        s.cache[:, :c.cache.shape[1]].copy_(c.cache)
        s.tables.zero_()
        s.tables[:, :c.tables.shape[1]].copy_(c.tables)
        n = c.group_prefix.numel()
        s.group_start[:n + 1].copy_(c.group_start)
        s.group_start[n + 1:] = int(c.group_start[n])
        s.group_prefix.zero_()
        s.group_prefix[:n].copy_(c.group_prefix)
        for name in ("qkv", "q_start", "q_len", "ctx_len"):
            getattr(s, name).copy_(getattr(c, name))

    out = torch.empty(5, 8, 64, dtype=torch.bfloat16, device=DEV)
    hints = dict(max_prefix=512, max_own=128)
    assert one_by_one(ops, s, **hints)
    fill(cases[0])
    s.run(ops, out=out, **hints)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        s.run(ops, out=out, **hints)
    for c in (cases[1], cases[2], cases[0]):
        fill(c)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)
    fill(cases[1])
    s.q_len[1], s.q_len[4] = 3, 0
    out.fill_(77.0)
    graph.replay()
    torch.cuda.synchronize()
    cases[1].check(out, [0, 2, 3])
    assert (out[1] == 77.0).all() and (out[4] == 77.0).all()
