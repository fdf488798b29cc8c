"""Decode attention of rows that share a prefix, where prefix and own keys are one walk on the tensor cores (heads of 64 and 128, more than 128 pairs of a
row and a query head on a key head), against attention of every row over its whole sequence in 64 bits."""
import pytest
import torch

from test_shared_prefix_gpu import DEV, Case, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def at_once(monkeypatch):
    """Groups are taken at once however little they share."""
    from mini_inference_engine_b200.kernels import ops
    monkeypatch.setattr(ops, "PREFIX_ONE_BY_ONE_BYTES", (-1, -1))
    ops._shared_plan.cache_clear()
    yield
    ops._shared_plan.cache_clear()


def walks(ops, c, **hints):
    """The case, run by the walk: its plan says so."""
    return ops._shared_plan(torch.cuda.current_device(), c.rows, c.group_prefix.numel(), c.H, c.G, c.D, c.page, hints["max_prefix"], hints["max_own"],
                            c.cache.shape[1], 0)[1] == 1


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 32, 128, 256])
def test_pages(ops, D, page):
    c = Case([(5, 200), (1, 70), (4, 131)], 90, 32, 2, D, page, seed=D + page)
    assert walks(ops, c, **c.hints)
    out = c.run(ops, **c.hints)
    c.check(out)
    assert torch.equal(out, c.run(ops, **c.hints))            # run to run: the same bits


@pytest.mark.parametrize("H,G,rows", [(16, 16, 129), (17, 1, 8), (96, 2, 3), (136, 1, 2), (300, 1, 5), (40, 8, 27), (12, 4, 44)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_shapes(ops, H, G, rows, D):
    c = Case([(rows - 1, 150), (1, 20)], 40, H, G, D, 16, seed=H + D)
    assert walks(ops, c, **c.hints)
    c.check(c.run(ops, **c.hints))


@pytest.mark.parametrize("groups,own", [
    ([(9, 1)], 1), ([(9, 127)], 1), ([(9, 128)], 1), ([(9, 129)], 3), ([(9, 255)], 128), ([(9, 256)], 129), ([(10, 0)], 200),
    ([(2, 0), (9, 100), (2, 0)], 40), ([(0, 90), (9, 90), (0, 0), (1, 33), (0, 4)], 10),
    ([(1, 100)] * 12, 60),                                    # groups of one row
    ([(40, 777)], 20), ([(20, 300), (1, 5), (30, 129)], 150), # more pairs than a tile holds
    ([(9, 5000)], [1, 700, 64, 1, 129, 128, 127, 2, 333]),    # a long prefix, unequal rests
    ([(3, 3000), (2, 10), (2, 900), (2, 1), (2, 2000)], 500)])
@pytest.mark.parametrize("D", [64, 128])
def test_groups(ops, groups, own, D):
    c = Case(groups, own, 32, 2, D, 16, seed=len(groups) + D)
    assert walks(ops, c, **c.hints)
    out = c.run(ops, **c.hints)
    c.check(out)
    c.check(c.run(ops))                                       # without the hints: planned for the table's width
    assert torch.equal(out, c.run(ops, **c.hints))


@pytest.mark.parametrize("count", [30, 61, 64, 80])
def test_many_groups(ops, count):
    """More groups than the walk plans for: the kernel for any head size takes over, with the same results."""
    c = Case([(1 + i % 2, 10 + 7 * (i % 5)) for i in range(count)], 20, 32, 2, 64, 16, seed=count)
    c.check(c.run(ops, **c.hints))


@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_no_group_and_rows_without_own_keys(ops, D):
    c = Case([(6, 150), (4, 96)], [0, 4, 0, 0, 1, 9, 0, 0, 0, 128, 60, 1, 300], 32, 2, D, 16, uncovered=3, seed=D)
    assert walks(ops, c, **c.hints)
    c.check(c.run(ops, **c.hints))


@pytest.mark.parametrize("loud", [0, 77, 1023, 1024, 1030])
@pytest.mark.parametrize("D", [64, 128])
def test_one_key_that_every_row_hears(ops, loud, D):
    c = Case([(9, 1024)], [7, 8, 9, 10, 20, 30, 40, 100, 300], 32, 2, D, 16, loud=loud)
    assert walks(ops, c, **c.hints)
    out = c.run(ops, **c.hints)
    c.check(out)
    assert (out.float() - 5.0).abs().max() < 0.05


@pytest.mark.parametrize("D", [64, 128])
def test_float32_output(ops, D):
    c = Case([(8, 700), (2, 0)], 100, 32, 2, D, 16)
    assert walks(ops, c, **c.hints)
    c.check(c.run(ops, dtype=torch.float32, **c.hints))


@pytest.mark.parametrize("D", [64, 128])
def test_rows_with_more_tokens_are_left_alone(ops, D):
    """A row of several tokens, or of none, inside a group and outside: its output stays, and its neighbours do not see it."""
    c = Case([(8, 300), (3, 40)], 50, 32, 2, D, 16, uncovered=2)
    assert walks(ops, c, **c.hints)
    for row, n in ((1, 3), (5, 0), (8, 2), (11, 0)):
        c.q_len[row] = n
    out = c.run(ops, **c.hints)
    c.check(out, [0, 2, 3, 4, 6, 7, 9, 10, 12])
    for row in (1, 5, 8, 11):
        assert (out[row] == 77.0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_a_bad_page_is_reported(ops, D):
    """In a prefix: the other group is as it should be.  In own keys: the other rows are."""
    for row, entry, sound in ((0, 2, range(6, 10)), (3, 8, [0, 1, 2, 4, 5, 6, 7, 8, 9])):
        c = Case([(6, 100), (4, 20)], [40] * 10, 32, 2, D, 16)
        assert walks(ops, c, **c.hints)
        c.tables[row, entry] = 10 ** 6
        out = c.run(ops, **c.hints)
        torch.cuda.synchronize()
        got = ops.range_report().tolist()
        assert got[0] == 4 and got[3] == 10 ** 6
        with pytest.raises(ops.KernelError, match="page"):
            ops.check_range_errors()
        c.check(out, sound)


@pytest.mark.parametrize("D", [64, 128])
def test_a_context_inside_its_prefix_is_reported(ops, D):
    c = Case([(6, 100), (4, 20)], 30, 32, 2, D, 16)
    assert walks(ops, c, **c.hints)
    c.ctx_len[1] = 60
    out = c.run(ops, **c.hints)
    torch.cuda.synchronize()
    assert ops.range_report().tolist()[:1] == [2]
    with pytest.raises(ops.KernelError, match="position"):
        ops.check_range_errors()
    c.check(out, [0, 2, 3, 4, 5, 6, 7, 8, 9])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_what_is_no_number_stays_in_its_row(ops, D, what):
    """A value, a key and a query of one row's own, and a value of one group's prefix."""
    H, G = 32, 2

    def spoiled(row, prefix, cache, at):
        c = Case([(7, 130), (3, 90)], [30] * 10, H, G, D, 16, seed=D)
        assert walks(ops, c, **c.hints)
        key = 53 if prefix else c.ctx[row] - 9
        pg = int(c.tables[0 if prefix and row < 7 else row, key // 16])
        c.cache[cache, pg, 1, key % 16, at] = what
        return c, c.run(ops, **c.hints)

    c, out = spoiled(2, False, 1, 7)                          # an own value: one number of every head on that key head
    assert not torch.isfinite(out[2, H // G:, 7]).any()
    out[2, H // G:, 7] = 0
    assert torch.isfinite(out).all()
    c.check(out, [0, 1, 3, 4, 5, 6, 7, 8, 9])
    c, out = spoiled(4, True, 1, 7)                           # a prefix's value
    assert not torch.isfinite(out[:7, H // G:, 7]).any()
    out[:7, H // G:, 7] = 0
    assert torch.isfinite(out).all()
    c.check(out, [7, 8, 9])
    c, out = spoiled(5, False, 0, 3)                          # an own key
    assert torch.isfinite(out[:, :H // G]).all()
    c.check(out, [0, 1, 2, 3, 4, 6, 7, 8, 9])
    c = Case([(7, 130), (3, 90)], [30] * 10, H, G, D, 16, seed=D)
    c.qkv[6, 5] = what                                        # a query: one head
    out = c.run(ops, **c.hints)
    c.check(out, [0, 1, 2, 3, 4, 5, 7, 8, 9])
    assert torch.isfinite(out[6, 1:]).all()


@pytest.mark.parametrize("D", [64, 128])
def test_captured_step_follows_its_groups(ops, D):
    """One captured call, replayed for other groups, prefixes and lengths; between the replays another call uses the same workspaces."""
    cases = [Case([(9, 400), (3, 0)], 30, 32, 2, D, 16, seed=1), Case([(2, 90), (10, 250)], 60, 32, 2, D, 16, seed=2), Case([(1, 1), (11, 512)], [1] * 12, 32, 2, D, 16, seed=3)]
    pages, width = max(c.cache.shape[1] for c in cases), max(c.tables.shape[1] for c in cases)
    s = Case([(9, 400), (3, 0)], 30, 32, 2, D, 16, seed=1)
    s.cache, s.tables = torch.zeros(2, pages, 2, 16, D, dtype=torch.bfloat16, device=DEV), torch.zeros(12, width, dtype=torch.int32, device=DEV)

    def fill(c):
        s.cache.zero_()
        s.cache[:, :c.cache.shape[1]].copy_(c.cache)
        s.tables.zero_()
        s.tables[:, :c.tables.shape[1]].copy_(c.tables)
        for name in ("qkv", "q_start", "q_len", "ctx_len", "group_start", "group_prefix"):
            getattr(s, name).copy_(getattr(c, name))

    out = torch.empty(12, 32, D, dtype=torch.bfloat16, device=DEV)
    hints = dict(max_prefix=512, max_own=128)
    assert walks(ops, s, **hints)
    fill(cases[0])
    s.run(ops, out=out, **hints)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        s.run(ops, out=out, **hints)
    other = Case([(30, 700)], 100, 32, 2, D, 16, seed=9)
    for c in (cases[1], cases[0], cases[2], cases[1]):
        fill(c)
        out.zero_()
        graph.replay()
        other_out = other.run(ops, **other.hints)
        torch.cuda.synchronize()
        c.check(out)
        other.check(other_out)


@pytest.mark.parametrize("D", [64, 128])
def test_a_cache_whose_offsets_pass_32_bits(ops, D):
    c = Case([(9, 100)], 40, 32, 2, D, 16, extra_pages=2)
    assert walks(ops, c, **c.hints)
    pages = (1 << 31) // (2 * 16 * D) + 64                    # elements before the last pages: more than 2^31
    big = torch.empty(2, pages, 2, 16, D, dtype=torch.bfloat16, device=DEV)
    n = c.cache.shape[1]
    big[:, pages - n:] = c.cache
    big[:, 0] = 0
    c.cache, c.tables = big, c.tables + (pages - n)
    c.check(c.run(ops, **c.hints))


def test_rows_spread_over_the_packed_tokens(ops):
    """The rows' tokens lie anywhere, in any order, with others between them: what is no row's token keeps its output."""
    c = Case([(9, 200), (1, 30)], 50, 32, 2, 64, 16, seed=7)
    at = [17, 3, 8, 0, 21, 5, 11, 14, 2, 9]
    qkv = torch.full((24, c.qkv.shape[1]), float("nan"), dtype=torch.bfloat16, device=DEV)
    qkv[at] = c.qkv
    c.qkv, c.q_start = qkv, torch.tensor(at, dtype=torch.int32, device=DEV)
    out = torch.full((24, c.H, c.D), 77.0, dtype=torch.bfloat16, device=DEV)
    c.run(ops, out=out, **c.hints)
    c.check(out[at])
    out[at] = 77.0
    assert (out == 77.0).all()


@pytest.mark.parametrize("H,G,D,rows", [(32, 2, 64, 9), (32, 2, 128, 9), (8, 2, 64, 3), (8, 2, 96, 3)])
def test_a_prefix_whose_last_key_the_step_writes(ops, H, G, D, rows):
    """The launch in front writes the prefix's last key and value: the very next launch sees them, time after time."""
    c = Case([(rows, 128)], [0] * (rows - 1) + [5], H, G, D, 16, seed=D)
    page, cos, sin = int(c.tables[0, 7]), torch.ones(256, D // 2, device=DEV), torch.zeros(256, D // 2, device=DEV)
    positions, slots = torch.tensor([127], dtype=torch.int32, device=DEV), torch.tensor([page * 16 + 15], dtype=torch.int32, device=DEV)
    busy = torch.randn(2048, 2048, device=DEV)
    g = torch.Generator().manual_seed(D)
    for turn in range(8):
        k, v = torch.randn(2, G, D, generator=g).to(torch.bfloat16)
        k *= 4
        for r in range(rows):
            c.keys[r][127], c.values[r][127] = k, v
        c.qkv[0, H * D:(H + 2 * G) * D] = torch.cat([k.reshape(-1), v.reshape(-1)]).to(DEV)
        torch.cuda.synchronize()
        busy @ busy
        ops.rope_cache_write(c.qkv[:1], positions, slots, cos, sin, c.cache[0], c.cache[1], H, G, D, D, 16)
        c.check(c.run(ops, **c.hints))


@pytest.mark.parametrize("H,G,D", [(32, 2, 64), (32, 2, 128), (4, 2, 64), (4, 2, 80)])
def test_groups_and_lengths_out_of_range_are_reported(ops, H, G, D):
    """Groups that go back or reach beyond the rows, a prefix and a context longer than a block table: reported, and nothing outside is touched."""
    for name, at, value in (("group_start", 1, 99), ("group_start", 2, 3), ("group_start", 0, -1), ("group_prefix", 0, -5), ("group_prefix", 1, 10 ** 6),
                            ("ctx_len", 2, 10 ** 6), ("ctx_len", 7, 2 ** 31 - 1), ("ctx_len", 8, -4)):
        c = Case([(6, 100), (4, 20)], 30, H, G, D, 16, seed=D)
        c.tables = torch.where(c.tables == c.tables.max(), 0, c.tables)      # (entries nobody should follow: page 0)
        getattr(c, name)[at] = value
        c.run(ops, **c.hints)
        torch.cuda.synchronize()
        assert ops.range_report()[0].item() in (2, 5), (name, at)      # a position, or a row (whichever block comes first)
        with pytest.raises(ops.KernelError):
            ops.check_range_errors()
        ops.range_report().zero_()
        sound = Case([(6, 100), (4, 20)], 30, H, G, D, 16, seed=D)
        sound.check(sound.run(ops, **sound.hints))            # the call after it is as it should be


@pytest.mark.parametrize("D,groups,own", [(64, [(2, 6000), (1, 0)], 900), (80, [(3, 5000)], 700), (128, [(1, 9000), (2, 40)], 500)])
def test_few_rows_with_many_own_keys(ops, D, groups, own):
    """The kernel for any head size: a row's own keys in parts, behind a prefix in many ranges; a query that is no number shows in its row and head only."""
    c = Case(groups, own, 8, 2, D, 16, seed=D)
    assert not walks(ops, c, **c.hints)
    out = c.run(ops, **c.hints)
    c.check(out)
    assert torch.equal(out, c.run(ops, **c.hints))
    c.check(c.run(ops, dtype=torch.float32, **c.hints))
    c.qkv[1, 3 * D + 1] = float("nan")
    out = c.run(ops, **c.hints)
    assert torch.isnan(out[1, 3]).all()
    out[1, 3] = 0
    assert torch.isfinite(out).all()
    c.check(out, [0, 2])


def test_calls_on_two_streams_at_once(ops):
    """Each stream's calls use scratch memory of their own."""
    cases = [Case([(40, 900)], 200, 32, 2, 64, 16, seed=3), Case([(2, 3000)], 700, 8, 2, 64, 16, seed=4), Case([(17, 2000), (3, 100)], 100, 8, 8, 128, 16, seed=5)]
    want = [c.run(ops, **c.hints) for c in cases]
    for c, o in zip(cases, want):
        c.check(o)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for turn in range(10):
        got = []
        for k in range(9):
            i = (k + turn) % 3
            with torch.cuda.stream(streams[k % 3]):
                got.append((i, cases[i].run(ops, **cases[i].hints)))
        torch.cuda.synchronize()
        for i, o in got:
            assert torch.equal(o, want[i]), (turn, i)
