"""Decode attention of rows that share a prefix, against attention of every row over its whole sequence in 64 bits."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture()
def ops():
    from mini_inference_engine_b200.kernels import ops
    torch.cuda.synchronize()
    ops.range_report().zero_()
    yield ops
    torch.cuda.synchronize()
    ops.check_range_errors()
    ops.check_tc_errors()


class Case:
    """Groups as (rows, prefix); ``own``: keys behind the prefix, a number a row or a bound to draw them from.  Pages lie scattered; what nobody may read
    holds NaN: other pages, a row's own page in front of its own keys; table entries that nobody may follow name a page of NaN."""

    def __init__(self, groups, own, H, G, D, page, seed=0, uncovered=0, loud=None, extra_pages=0, spread=1.5):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        rows = sum(n for n, _ in groups) + uncovered
        own = list(own) if isinstance(own, (list, tuple)) else [rng.randint(1, own) for _ in range(rows)]
        self.groups, self.H, self.G, self.D, self.page, self.rows = groups, H, G, D, page, rows
        start = [0]
        for n, _ in groups:
            start.append(start[-1] + n)
        prefix_of = [p for n, p in groups for _ in range(n)] + [0] * uncovered
        leader = [s for (n, _), s in zip(groups, start) for _ in range(n)] + list(range(start[-1], rows))
        self.ctx = [p + o for p, o in zip(prefix_of, own)]
        need = sum(-(-c // page) for c in self.ctx) + 2 + extra_pages
        ids = list(range(1, need - 1))
        rng.shuffle(ids)
        nan_page = need - 1
        width = max(-(-c // page) for c in self.ctx) + 1
        cache = torch.full((2, need, G, page, D), float("nan"), dtype=torch.bfloat16)
        cache[:, 0] = 0
        tables = torch.full((rows, width), nan_page, dtype=torch.int32)
        self.keys, self.values = [], []
        shared_kv = {}
        for r in range(rows):
            P, first = prefix_of[r], leader[r]
            k, v = torch.randn(2, self.ctx[r], G, D, generator=g).to(torch.bfloat16)
            if r != first and P:
                k[:P], v[:P] = shared_kv[first]
            if loud is not None:                              # one key that every row must hear
                at = min(loud, self.ctx[r] - 1)
                k[at], v[at] = 0, 5.0
                k[at, :, 0] = 30.0
            shared_kv[r] = (k[:P].clone(), v[:P].clone())
            self.keys.append(k)
            self.values.append(v)
            begin = 0 if r == first else P
            for i in range(begin // page, -(-self.ctx[r] // page)):
                pg = ids.pop()
                tables[r, i] = pg
                cache[:, pg] = 0 if (i + 1) * page > self.ctx[r] else cache[:, pg]      # behind the context: finite
                for at in range(max(begin, i * page), min(self.ctx[r], (i + 1) * page)):
                    cache[0, pg, :, at % page], cache[1, pg, :, at % page] = k[at], v[at]
                if i * page < begin:                          # in front of the own keys: NaN
                    cache[:, pg, :, :begin % page] = float("nan")
        q = torch.randn(rows, H, D, generator=g) * spread
        if loud is not None:
            q[:, :, :] = 0
            q[:, :, 0] = 30.0
        self.q = q.to(torch.bfloat16)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        stride = (H + 2 * G) * D
        stride += -stride % 8
        self.qkv = torch.full((rows, stride), float("nan"), dtype=torch.bfloat16)
        self.qkv[:, :H * D] = self.q.view(rows, -1)
        self.qkv = self.qkv.to(DEV)
        self.cache, self.tables = cache.to(DEV), tables.to(DEV)
        self.group_start, self.group_prefix = i32(start), i32([p for _, p in groups])
        self.q_start, self.q_len, self.ctx_len = i32(list(range(rows))), i32([1] * rows), i32(self.ctx)
        self.scale = 1.0 / math.sqrt(D)
        self.hints = dict(max_prefix=max([p for _, p in groups], default=0), max_own=max(c - p for c, p in zip(self.ctx, prefix_of)))

    def run(self, ops, out=None, dtype=torch.bfloat16, **hints):
        if out is None:
            out = torch.full((self.rows, self.H, self.D), 77.0, dtype=dtype, device=DEV)
        got = ops.shared_prefix_attention(self.qkv, self.qkv.shape[1], self.cache[0], self.cache[1], self.tables, self.q_start, self.q_len, self.ctx_len,
                                          self.group_start, self.group_prefix, out, self.H, self.G, self.D, self.page, self.scale, **hints)
        assert got is out
        return out

    def want(self, r):
        """The row's output in float64, and its bound: the weights are rounded to bfloat16 for their product with the values (half a step, 2^-8, of
        sum w |v|), the output once more (2^-8 of itself; a float32 output not); scores, exponentials and sums in float32 add less than a
        hundredth of that."""
        H, G, D = self.H, self.G, self.D
        q = self.q[r].double().view(G, H // G, D)
        k, v = self.keys[r].double(), self.values[r].double()
        w = torch.softmax(torch.einsum("ghd,kgd->ghk", q, k) * self.scale, -1)
        o = torch.einsum("ghk,kgd->ghd", w, v).reshape(H, D)
        return o, torch.einsum("ghk,kgd->ghd", w, v.abs()).reshape(H, D)

    def check(self, out, rows=None):
        got = out.cpu().double()
        for r in range(self.rows) if rows is None else rows:
            o, size = self.want(r)
            bound = 1.01 * 2.0 ** -8 * (size + (o.abs() if out.dtype == torch.bfloat16 else 0)) + 1e-6
            assert torch.isfinite(got[r]).all(), r
            off = (got[r] - o).abs() - bound
            assert (off <= 0).all(), (r, self.ctx[r], float(off.max()), float(size.max()))


HEADS = [(32, 4, 64, 16), (8, 8, 128, 16), (6, 2, 64, 8), (12, 1, 128, 32), (5, 5, 16, 16), (24, 4, 96, 16), (20, 1, 80, 16), (40, 2, 32, 4), (70, 1, 16, 16),
         (4, 2, 48, 1), (16, 4, 112, 64), (32, 8, 128, 128), (32, 4, 64, 256), (4, 4, 64, 2), (136, 1, 64, 16)]


@pytest.mark.parametrize("H,G,D,page", HEADS)
def test_head_shapes_and_pages(ops, H, G, D, page):
    c = Case([(3, 200), (1, 70), (4, 131)], 90, H, G, D, page, seed=H + D)
    c.check(c.run(ops, **c.hints))


@pytest.mark.parametrize("groups,own", [
    ([(2, 1)], 1),                                            # one shared key, one own
    ([(1, 500)], 3),                                          # a group of one row
    ([(2, 64)], 64), ([(2, 128)], 1), ([(2, 127)], 5), ([(3, 129)], 200), ([(2, 16)], 1),
    ([(5, 0)], 300), ([(2, 0), (3, 100), (2, 0)], 40),        # rows that share nothing
    ([(0, 90), (3, 90), (0, 0), (1, 33)], 10),                # groups without rows
    ([(33, 777)], 20), ([(70, 300), (1, 5)], 30),             # more rows than a tile holds
    ([(4, 5000)], [1, 700, 64, 1]),                           # a long prefix, unequal rests
    ([(2, 3000), (2, 10), (2, 900), (2, 1), (2, 2000)], 500)])
@pytest.mark.parametrize("D", [64, 128, 32])
def test_groups(ops, groups, own, D):
    c = Case(groups, own, 8, 2, D, 16, seed=len(groups) + D)
    out = c.run(ops, **c.hints)
    c.check(out)
    c.check(c.run(ops))                                       # without the hints: planned for the table's width
    assert torch.equal(out, c.run(ops, **c.hints))            # run to run: the same bits


def test_rows_of_no_group_share_nothing(ops):
    c = Case([(3, 150)], 60, 8, 2, 64, 16, uncovered=4)
    c.check(c.run(ops, **c.hints))


def test_rows_whose_context_ends_with_their_prefix(ops):
    """The newest key belongs to the prefix: the rows have no own keys."""
    for D in (64, 128, 80):
        c = Case([(3, 96), (2, 333)], [0, 4, 0, 0, 1], 8, 4, D, 16, seed=D)
        c.check(c.run(ops, **c.hints))


@pytest.mark.parametrize("loud", [0, 77, 1023, 1024, 1030])
@pytest.mark.parametrize("D", [64, 128, 48])
def test_one_key_that_every_row_hears(ops, loud, D):
    c = Case([(9, 1024)], [7, 8, 9, 10, 20, 30, 40, 100, 300], 8, 2, D, 16, loud=loud)
    out = c.run(ops, **c.hints)
    c.check(out)
    assert (out.float() - 5.0).abs().max() < 0.05


def test_float32_output(ops):
    for D in (64, 128, 96):
        c = Case([(6, 700), (1, 0)], 100, 12, 4, D, 16)
        c.check(c.run(ops, dtype=torch.float32, **c.hints))


def test_rows_with_more_tokens_are_left_alone(ops):
    c = Case([(5, 300), (2, 40)], 50, 8, 2, 64, 16)
    c.q_len[1] = 3
    c.q_len[6] = 2
    out = c.run(ops, **c.hints)
    c.check(out, [0, 2, 3, 4, 5])
    assert (out[1] == 77.0).all() and (out[6] == 77.0).all()


def test_no_groups_and_no_rows(ops):
    c = Case([], 200, 8, 2, 64, 16, uncovered=3)
    c.check(c.run(ops))
    c.check(c.run(ops, max_prefix=0))
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    out = torch.empty(0, 8, 64, dtype=torch.bfloat16, device=DEV)
    c.tables, c.q_start, c.q_len, c.ctx_len = c.tables[:0], empty, empty, empty
    assert c.run(ops, out=out) is out


@pytest.mark.parametrize("D", [64, 80])
def test_a_bad_page_is_reported(ops, D):
    c = Case([(3, 100), (1, 20)], 30, 4, 2, D, 16)
    c.tables[0, 2] = 10 ** 6                                  # the first group's prefix
    out = c.run(ops, **c.hints)
    torch.cuda.synchronize()
    got = ops.range_report().tolist()
    assert got[0] == 4 and got[1] == 16 and got[3] == 10 ** 6
    with pytest.raises(ops.KernelError, match="attention_prefix"):
        ops.check_range_errors()
    c.check(out, [3])                                         # the other group is as it should be


def test_a_context_inside_its_prefix_is_reported(ops):
    c = Case([(3, 100), (1, 20)], 30, 4, 2, 64, 16)
    c.ctx_len[1] = 60
    out = c.run(ops, **c.hints)
    torch.cuda.synchronize()
    assert ops.range_report().tolist()[:1] == [2]
    with pytest.raises(ops.KernelError, match="position"):
        ops.check_range_errors()
    c.check(out, [0, 2, 3])


def test_captured_step_follows_its_groups(ops):
    a = Case([(6, 400), (2, 0)], 30, 8, 2, 64, 16, seed=1, extra_pages=200)
    b = Case([(1, 90), (7, 250)], 60, 8, 2, 64, 16, seed=2, extra_pages=200)
    n = min(a.cache.shape[1], b.cache.shape[1])
    assert int(a.tables.max()) < a.cache.shape[1] and b.tables.max() < b.cache.shape[1]
    cache = torch.zeros(2, max(a.cache.shape[1], b.cache.shape[1]), 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    width = max(a.tables.shape[1], b.tables.shape[1])
    s = Case([(6, 400), (2, 0)], 30, 8, 2, 64, 16, seed=1, extra_pages=200)
    s.cache, s.tables = cache, torch.zeros(8, width, dtype=torch.int32, device=DEV)

    def fill(c):
        cache.zero_()
        cache[:, :c.cache.shape[1]].copy_(c.cache)
        s.tables.zero_()
        s.tables[:, :c.tables.shape[1]].copy_(c.tables)
        for name in ("qkv", "q_start", "q_len", "ctx_len", "group_start", "group_prefix"):
            getattr(s, name).copy_(getattr(c, name))

    assert n
    out = torch.empty(8, 8, 64, dtype=torch.bfloat16, device=DEV)
    fill(a)
    hints = dict(max_prefix=512, max_own=128)
    s.run(ops, out=out, **hints)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        s.run(ops, out=out, **hints)
    for c in (b, a, b):
        fill(c)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)


def test_follows_decode_attention_on_its_stream(ops):
    """On a stream of its own, one launch behind another, with workspaces that other sizes have used before."""
    side = torch.cuda.Stream()
    cases = [Case([(40, 600)], 200, 8, 2, 64, 16, seed=3), Case([(2, 64)], 5, 32, 4, 64, 16, seed=4), Case([(17, 2000), (3, 100)], 100, 8, 8, 128, 16, seed=5)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        outs = [c.run(ops, **c.hints) for c in cases for _ in range(2)]
    side.synchronize()
    for i, c in enumerate(cases):
        c.check(outs[2 * i])
        assert torch.equal(outs[2 * i], outs[2 * i + 1])


def test_a_cache_whose_offsets_pass_32_bits(ops):
    c = Case([(3, 100)], 40, 4, 2, 128, 16, extra_pages=2)
    pages = (1 << 31) // (2 * 16 * 128) + 64                  # elements before the last pages: more than 2^31
    big = torch.empty(2, pages, 2, 16, 128, dtype=torch.bfloat16, device=DEV)
    n = c.cache.shape[1]
    big[:, pages - n:] = c.cache
    big[:, 0] = 0
    c.cache, c.tables = big, c.tables + (pages - n)
    c.check(c.run(ops, **c.hints))


def test_an_infinite_value_reaches_the_rows_that_see_it_only(ops):
    for D in (64, 128, 80):
        c = Case([(3, 130), (3, 90)], [20] * 6, 4, 2, D, 16)
        pg = int(c.tables[0, 3])
        c.cache[1, pg, 1, 5, 7] = float("inf")                # key 53 of the first group, its second key head
        out = c.run(ops, **c.hints).cpu()
        assert torch.isinf(out[:3, 2:, 7]).all()
        out[:3, 2:, 7] = 0
        assert torch.isfinite(out).all()
        c.check(out.to(DEV), [3, 4, 5])


def test_refusals(ops):
    c = Case([(3, 100)], 30, 4, 2, 64, 16)
    ok = dict(c.__dict__)

    def refused(match, **change):
        c.__dict__.update(change)
        with pytest.raises(ops.KernelError, match=match):
            c.run(ops)
        c.__dict__.update(ok)

    refused("bfloat16", qkv=c.qkv.float())
    refused("int32", group_prefix=c.group_prefix.long())
    refused("one entry more", group_start=c.group_start[:1])
    refused("contiguous", cache=c.cache.transpose(2, 3))
    refused("power of two", page=12)
    refused("kv heads", G=3)
    refused("multiples of 16", D=72)
    refused("16 bytes", qkv=c.qkv[:, 1:])
    refused("every row", ctx_len=c.ctx_len[:2])
    c.check(c.run(ops))


@pytest.mark.parametrize("D", [64, 128, 80])
@pytest.mark.parametrize("groups,own", [([(3, 0), (2, 50)], [0, 5, 0, 0, 3]), ([(2, 0), (9, 0)], [0] * 11), ([(9, 0), (1, 0)], [0, 0, 0, 300, 0, 0, 1, 0, 0, 0])])
def test_rows_without_any_keys_give_zeros(ops, D, groups, own):
    c = Case(groups, own, 32, 2, D, 16, seed=D)
    other = Case([(20, 300)], 100, 32, 2, D, 16, seed=1)
    for hints in (c.hints, dict(max_prefix=64, max_own=c.hints["max_own"])):
        other.run(ops, **other.hints)                         # (other results in the scratch memory)
        out = c.run(ops, **hints)
        c.check(out, [r for r in range(c.rows) if c.ctx[r]])
        for r in range(c.rows):
            if not c.ctx[r]:
                assert (out[r] == 0).all(), r
