"""Attention over shared prefixes whose scratch memory is made while others already run, or inside a capture; against attention of every row over its whole sequence in 64 bits."""
import pytest
import torch

from test_shared_prefix_gpu import DEV, Case, ops  # noqa: F401  (the fixture)
from test_shared_prefix_walk_gpu import at_once  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture()
def bare(ops, monkeypatch):  # noqa: F811
    """No scratch memory has been made yet; the kernels have run."""
    for D in (64, 80):
        small(D).run(ops)
    torch.cuda.synchronize()
    monkeypatch.setattr(ops, "_workspaces", {})
    ops._shared_plan.cache_clear()
    return ops


def small(D):
    return Case([(3, 200)], 300, 32, 16, D, 16, seed=1)


def large(D, seed):
    """More rows and key heads than the smallest scratch tensors hold."""
    return Case([(40, 170), (30, 90)], [300] * 2 + [1] * 68, 32, 16, D, 16, seed=seed)


@pytest.mark.parametrize("D", [64, 80])
def test_first_on_a_busy_stream_then_on_another(bare, D):
    side = torch.cuda.Stream()
    a, b = large(D, 1), large(D, 2)
    with torch.cuda.stream(side):                             # what the allocator hands out on that stream holds no zeros
        junk = [torch.full((n,), 7, dtype=torch.int32, device=DEV) for n in (1024, 1120, 2240) for _ in range(6)]
        del junk
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(40_000_000)
        out = a.run(bare, **a.hints)
    other = b.run(bare, **b.hints)
    torch.cuda.synchronize()
    a.check(out)
    b.check(other)


@pytest.mark.parametrize("D", [64, 80])
def test_captured_before_any_call_of_its_sizes(bare, D):
    small(D).run(bare)                                        # (smaller scratch tensors are there)
    a, b = large(D, 3), large(D, 4)
    out = torch.empty(a.rows, a.H, D, dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        a.run(bare, out=out, **a.hints)
        a.run(bare, out=out, **a.hints)
    first = b.run(bare, **b.hints)                            # before the graph has run at all
    b.check(first)
    for _ in range(3):
        out.zero_()
        graph.replay()
        again = b.run(bare, **b.hints)
        torch.cuda.synchronize()
        a.check(out)
        assert torch.equal(again, first)
