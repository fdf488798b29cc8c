"""The two chains of the walk over shared prefixes, where they fall out of step: a prefix whose last step has no keys in its second half, and one tile of pairs that has its sums
to rescale where the other has not.  Against attention of every row over its whole sequence in 64 bits."""
import pytest
import torch

from test_shared_prefix_gpu import DEV, Case, ops  # noqa: F401  (the fixture)
from test_shared_prefix_walk_gpu import at_once, walks  # noqa: F401

pytestmark = pytest.mark.gpu


def hear(c, rows, keys):
    """Of the first group's prefix, ``keys`` (place, how loud): the rows in ``rows`` hear each, and nobody else does."""
    for r in range(c.rows):
        c.q[r, :, 0] = 30.0 if r in rows else 0.0
    c.qkv[:, :c.H * c.D] = c.q.view(c.rows, -1).to(DEV)
    for at, loud in keys:
        page, place = int(c.tables[0, at // c.page]), at % c.page
        c.cache[0, page, :, place, 0] = loud
        for k in c.keys[:c.groups[0][0]]:
            k[at, :, 0] = loud


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("more", [1, 2, 33, 63, 64, 65, 128])
@pytest.mark.parametrize("second", [False, True])
def test_a_prefix_that_ends_in_the_first_half_of_a_step(ops, D, more, second):
    """32 query heads on 2: sixteen rows are two tiles of 128 pairs, eight rows each."""
    rows, whole = 16, 5 * 128
    c = Case([(rows, whole + more)], 20, 32, 2, D, 16, seed=more + D)
    tile = range(8, 16) if second else range(8)
    hear(c, tile, [(whole - 128 + at, 3.0 + at / 16) for at in (3, 60, 70, 100, 127)] + [(whole, 20.0)])
    assert walks(ops, c, **c.hints)
    out = c.run(ops, **c.hints)
    c.check(out)
    assert torch.equal(out, c.run(ops, **c.hints))


@pytest.mark.parametrize("more", [1, 64])
@pytest.mark.parametrize("steps", [0, 1, 2, 39])
def test_every_length_of_an_item(ops, steps, more):
    """Many rows and key heads: the ranges of the walk are as long as the prefix, and the short step is an item's first, or behind many."""
    c = Case([(32, steps * 128 + more), (40, 128 + more)], 9, 64, 8, 128, 16, seed=steps)
    hear(c, range(16, 32), [(steps * 128 + more - 1, 25.0)])
    assert walks(ops, c, **c.hints)
    c.check(c.run(ops, **c.hints))
