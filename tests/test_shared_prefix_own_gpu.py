"""Rows of a group that have no keys of their own behind the shared prefix, where that ends inside a page: their block tables have no page for it.  Against attention of every row over
its whole sequence in 64 bits."""
import pytest
import torch

from test_shared_prefix_gpu import DEV, Case, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

OWN = [[0, 4, 0, 1, 0], [3, 0, 70, 0, 200], [0] * 5]


@pytest.fixture(params=["rule", "at once"])
def way(request, monkeypatch):
    from mini_inference_engine_b200.kernels import ops
    if request.param == "at once":
        monkeypatch.setattr(ops, "PREFIX_ONE_BY_ONE_BYTES", (-1, -1))
    ops._shared_plan.cache_clear()
    yield
    ops._shared_plan.cache_clear()


@pytest.mark.parametrize("H,G,D", [(8, 8, 32), (20, 1, 112), (7, 1, 64), (32, 8, 128), (64, 1, 64), (64, 1, 128), (6, 2, 80)])
@pytest.mark.parametrize("page", [1, 16, 64, 256])
@pytest.mark.parametrize("prefix", [1, 17, 63, 64, 65, 127, 129, 300])
def test_rows_without_own_keys(ops, way, H, G, D, page, prefix):  # noqa: F811
    for own in OWN:
        c = Case([(5, prefix)], own, H, G, D, page, seed=prefix + page, uncovered=0)
        for r in range(1, 5):
            if own[r] == 0:
                c.tables[r] = 10 ** 6                         # no entry of theirs may be followed
        out = c.run(ops, **c.hints)
        torch.cuda.synchronize()
        ops.check_range_errors()
        c.check(out)
        c.check(c.run(ops, dtype=torch.float32))
