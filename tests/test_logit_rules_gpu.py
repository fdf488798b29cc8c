"""Rules on logits (penalties, biases, grammar masks) and the choice of a token under them, against the plain form in 64 bits."""
import math
import random

import pytest
import torch

from plain_rules import INF, logprob_bound, ruled

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


def words_of(allowed, words):
    """A list of allowed entries as int32 words."""
    w = [0] * words
    for i in allowed:
        w[i // 32] |= 1 << (i % 32)
    return [v - (1 << 32) if v >= 1 << 31 else v for v in w]


class Step:
    """Random rules for ``rows`` rows, as host lists and as the framework's tensors."""

    def __init__(self, ops, rows, vocab, seed=0, width=70, biases=5, masks=True, penalties=True, spare_words=0):
        rng = random.Random(seed)
        torch.manual_seed(seed)
        slots = rows + 2
        self.rows, self.vocab, self.ops = rows, vocab, ops
        self.logits = torch.randn(rows, vocab) * 3
        self.text = [[min(int(vocab * rng.random() ** 3), vocab - 1) for _ in range(width)] for _ in range(slots)]
        self.slot = rng.sample(range(slots), rows)
        self.total = [rng.choice([0, 1, width, rng.randint(0, width)]) for _ in range(rows)]
        self.prompt = [rng.choice([0, t, rng.randint(0, t)]) for t in self.total]
        self.rep = [rng.choice([1.0, 1.3, 0.8]) for _ in range(rows)]
        self.pres = [rng.choice([0.0, 0.7, -0.4]) for _ in range(rows)]
        self.freq = [rng.choice([0.0, 0.25]) for _ in range(rows)]
        # some tokens are named twice; some are banned
        self.bias = [[(rng.randrange(vocab), rng.choice([2.5, -1.25, 0.1, -INF])) for _ in range(biases)] for _ in range(slots)]
        for b in self.bias:
            if len(b) > 2:
                b[2] = (b[0][0], 0.3)
        self.bias_len = [rng.choice([biases, rng.randint(0, biases)]) for _ in range(rows)]
        words = -(-vocab // 32) + spare_words
        self.allowed = [sorted(rng.sample(range(vocab), min(vocab, n))) for n in (1, 7, max(1, vocab // 2))] + [list(range(vocab))]
        self.mask = [words_of(a, words) for a in self.allowed]
        if vocab % 32:
            for m in self.mask:                           # bits behind the vocabulary mean nothing
                m[vocab // 32] |= -1 << (vocab % 32) if m[vocab // 32] >= 0 else 0
        self.mask_row = [rng.choice([-1, 0, 1, 2, 3]) for _ in range(rows)]
        self.masks, self.penalties, self.biases = masks, penalties, biases
        self.build()

    def build(self):
        i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        f = lambda v: torch.tensor(v, dtype=torch.float32, device=DEV)
        some = dict(repetition=f(self.rep), presence=f(self.pres), frequency=f(self.freq)) if self.penalties else {}
        if self.biases:
            some.update(bias_tokens=i([[t for t, _ in b] for b in self.bias]), bias_values=f([[v for _, v in b] for b in self.bias]), bias_len=i(self.bias_len))
        if self.masks:
            some.update(mask=i(self.mask), mask_row=i(self.mask_row))
        self.t = dict(history=i(self.text), slot=i(self.slot), prompt_len=i(self.prompt), total_len=i(self.total), **some)
        self.rules = self.ops.LogitRules(**self.t)

    def row(self, r):
        s = self.slot[r]
        text = self.text[s][:self.total[r]] if self.penalties and s >= 0 else []
        rep, pres, freq = (torch.tensor(v[r], dtype=torch.float32).item() for v in (self.rep, self.pres, self.freq))
        biases = [(t, torch.tensor(b, dtype=torch.float32).item()) for t, b in (self.bias[s][:self.bias_len[r]] if self.biases and s >= 0 else [])]
        mask = self.mask[self.mask_row[r]] if self.masks and self.mask_row[r] >= 0 else None
        return ruled(self.logits[r], text, self.prompt[r], rep, pres, freq, biases, mask)

    def check(self, got):
        got = got.cpu().double()
        for r in range(self.rows):
            want, bound = self.row(r)
            inf = torch.isinf(want)
            assert torch.equal(torch.isinf(got[r]), inf) and torch.equal(got[r][inf], want[inf]), r
            assert ((got[r] - want).abs()[~inf] <= bound[~inf]).all(), (r, (got[r] - want).abs()[~inf].max())

    def arrays(self, temperature=0.0):
        return dict(temperature=torch.full((self.rows,), temperature, device=DEV), request=torch.arange(self.rows, device=DEV) * 11 + 5,
                    position=torch.arange(self.rows, dtype=torch.int32, device=DEV) % 3, out=torch.full((self.rows,), -7, dtype=torch.int32, device=DEV))

    def choose(self, logits=None, temperature=0.0, seed=3, **more):
        a = self.arrays(temperature)
        lp = torch.full((self.rows,), 5.0, device=DEV)
        x = self.logits.to(DEV) if logits is None else logits
        self.ops.sample(x, a["temperature"], a["request"], a["position"], seed, a["out"], rules=self.rules, logprob=lp, **more)
        return a["out"], lp


# entries: fewer than a group, not multiples of a group or a mask's word, several blocks a row, several turns a block
VOCABS = [1, 3, 33, 1031, 4095, 4096, 32000, 50001]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("rows", [1, 5])
def test_rules_against_64_bits(ops, rows, vocab):
    s = Step(ops, rows, vocab, seed=vocab + rows)
    x = s.logits.to(DEV)
    out = torch.full_like(x, 9.0)
    assert ops.apply_logit_rules(x, s.rules, out) is out
    s.check(out)
    assert torch.equal(x.cpu(), s.logits)
    ops.apply_logit_rules(x, s.rules, x)                     # in place: the same numbers
    assert torch.equal(x, out)


@pytest.mark.parametrize("vocab", VOCABS + [300001])
def test_choice_against_64_bits(ops, vocab):
    rows = 4 if vocab < 100000 else 2
    s = Step(ops, rows, vocab, seed=vocab)
    tokens, lp = s.choose()
    ruled_logits = torch.empty(rows, vocab, device=DEV)
    ops.apply_logit_rules(s.logits.to(DEV), s.rules, ruled_logits)
    s.check(ruled_logits)
    for r in range(rows):
        want, bound = s.row(r)
        x = ruled_logits[r].cpu()
        best = int((x == x.max()).nonzero()[0])              # the lowest entry of the largest ruled logit in float32
        assert int(tokens[r]) == best
        assert want[best] >= want.max() - 2 * float(bound.max())
        if want.max() == -INF:
            assert float(lp[r]) == -INF
        else:
            want_lp = float(torch.log_softmax(want, 0)[best])
            assert abs(float(lp[r]) - want_lp) <= logprob_bound(want) + float(bound.max()) * 2, (r, float(lp[r]), want_lp)


@pytest.mark.parametrize("parts", ["penalties", "biases", "masks"])
def test_each_rule_alone(ops, parts):
    s = Step(ops, 6, 5003, seed=4, penalties=parts == "penalties", biases=6 if parts == "biases" else 0, masks=parts == "masks", spare_words=3)
    out = torch.empty(6, 5003, device=DEV)
    ops.apply_logit_rules(s.logits.to(DEV), s.rules, out)
    s.check(out)


def test_masks_without_texts(ops):
    mask = torch.tensor([words_of([2, 31, 32, 39], 2)], dtype=torch.int32, device=DEV)
    rules = ops.LogitRules(mask=mask, mask_row=torch.tensor([0, -1], dtype=torch.int32, device=DEV))
    x = torch.randn(2, 40, device=DEV)
    out = ops.apply_logit_rules(x, rules, torch.empty_like(x))
    assert torch.isfinite(out[0]).nonzero().flatten().tolist() == [2, 31, 32, 39] and torch.equal(out[1], x[1])


def test_what_a_mask_hides_counts_for_nothing(ops):
    """NaN and infinities in masked places; a mask that leaves nothing; the type's lowest value as a logit."""
    V = 9001
    s = Step(ops, 4, V, seed=8, penalties=False, biases=0)
    keep = sorted({5, 77, 8000})
    s.mask[0], s.mask[1] = words_of(keep, -(-V // 32)), [0] * -(-V // 32)
    s.mask_row = [0, 1, 0, -1]
    s.logits[0, :] = float("nan")
    s.logits[0, keep] = torch.tensor([1.0, 3.0, 2.0])
    s.logits[2, :] = float("inf")
    s.logits[2, keep] = torch.finfo(torch.float32).min
    s.logits[3, :] = torch.finfo(torch.float32).min
    s.build()
    out = ops.apply_logit_rules(s.logits.to(DEV), s.rules, torch.empty(4, V, device=DEV)).cpu()
    assert torch.isfinite(out[0]).nonzero().flatten().tolist() == keep and (out[0][torch.isinf(out[0])] < 0).all()
    assert (out[1] == -INF).all()
    tokens, lp = s.choose()
    assert tokens.tolist() == [77, 0, 5, 0]
    want = torch.log_softmax(torch.tensor([1.0, 3.0, 2.0]).double(), 0)[1].item()
    assert abs(lp[0].item() - want) < 1e-5 and lp[1].item() == -INF
    assert abs(lp[2].item() + math.log(3)) < 1e-6 and abs(lp[3].item() + math.log(V)) < 1e-5      # equal logits, however low


def test_nan_outside_a_mask_shows(ops):
    s = Step(ops, 2, 6000, seed=1, penalties=False, biases=0, masks=True)
    s.mask_row = [-1, -1]
    s.logits[0, 17] = float("nan")
    s.build()
    tokens, lp = s.choose()
    others = s.logits[0].clone()
    others[17] = -INF
    assert int(tokens[0]) == int(others.argmax()) and torch.isnan(lp[0]) and torch.isfinite(lp[1])


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_rows_that_begin_anywhere(ops, shift):
    """Logits that are columns of a wider tensor: rows off the 16-byte groups, and an output that lies otherwise."""
    s = Step(ops, 3, 8191, seed=shift)
    wide = torch.full((3, 8191 + 5 + shift), float("nan"), device=DEV)
    x = wide[:, shift:shift + 8191]
    x.copy_(s.logits)
    for at in (shift, 0):
        out_wide = torch.full((3, 8300), 4.0, device=DEV)
        out = out_wide[:, at:at + 8191]
        ops.apply_logit_rules(x, s.rules, out)
        s.check(out)
        assert (out_wide[:, at + 8191:] == 4.0).all() and (at == 0 or (out_wide[:, :at] == 4.0).all())
    tokens, lp = s.choose(logits=x)
    again, lp2 = s.choose()
    assert torch.equal(tokens, again)
    assert (lp - lp2).abs().max() <= 2 * logprob_bound(s.logits)


def test_without_rules_the_choice_is_the_plain_one(ops):
    """With noise too: rules that say nothing change no token, and the log-probability needs no rules."""
    for vocab in (300, 32000):
        s = Step(ops, 9, vocab, seed=vocab, biases=0)
        s.rep, s.pres, s.freq, s.mask_row = [1.0] * 9, [0.0] * 9, [0.0] * 9, [3, -1] * 4 + [3]
        s.build()
        x = s.logits.to(DEV)
        for t in (0.0, 0.9):
            a = s.arrays(t)
            want = ops.sample(x, a["temperature"], a["request"], a["position"], 3, a["out"]).clone()
            got, lp = s.choose(temperature=t)
            assert torch.equal(got, want)
            lp2 = torch.empty(9, device=DEV)
            got2 = ops.sample(x, a["temperature"], a["request"], a["position"], 3, a["out"], logprob=lp2)
            assert torch.equal(got2, want) and torch.equal(lp, lp2)
            for r in range(9):
                exact = torch.log_softmax(s.logits[r].double(), 0)[int(want[r])].item()
                assert abs(lp[r].item() - exact) <= logprob_bound(s.logits[r].double())


def test_noise_under_rules_is_the_noise_of_the_ruled_logits(ops):
    s = Step(ops, 12, 7001, seed=2)
    x = ops.apply_logit_rules(s.logits.to(DEV), s.rules, torch.empty(12, 7001, device=DEV))
    a = s.arrays(0.7)
    want = ops.sample(x, a["temperature"], a["request"], a["position"], 3, a["out"]).clone()
    got, _ = s.choose(temperature=0.7)
    assert torch.equal(got, want)


def test_ties_go_to_the_lowest_entry(ops):
    x = torch.zeros(3, 40000, device=DEV)
    x[0, [39999, 20000, 7]] = 1.0
    x[1, [39999, 20000]] = 1.0
    rules = ops.LogitRules(mask=torch.full((1, 1250), -1, dtype=torch.int32, device=DEV), mask_row=torch.zeros(3, dtype=torch.int32, device=DEV))
    out = torch.empty(3, dtype=torch.int32, device=DEV)
    z = torch.zeros(3, device=DEV)
    ops.sample(x, z, torch.zeros(3, dtype=torch.int64, device=DEV), out.clone(), 0, out, rules=rules)
    assert out.tolist() == [7, 20000, 0]


def test_the_token_joins_the_text_and_reaches_the_host(ops):
    s = Step(ops, 4, 5000, seed=6, width=40)
    s.total = [40, 0, 13, 39]                                # the first has no room left
    s.prompt = [10, 0, 13, 2]
    s.build()
    before = s.t["history"].cpu().clone()
    host = torch.zeros(2, 8, dtype=torch.int32, pin_memory=True)
    tokens, _ = s.choose(append=True, host_out=host, host_turn=torch.tensor([1], dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    after = s.t["history"].cpu()
    for r in range(1, 4):
        before[s.slot[r], s.total[r]] = int(tokens[r])
    assert torch.equal(after, before)
    assert host[1, :4].tolist() == tokens.tolist() and host[0].eq(0).all()


def test_rows_without_a_slot_have_no_text_and_no_biases(ops):
    s = Step(ops, 4, 5000, seed=7)
    s.slot[1] = s.slot[3] = -1
    s.build()
    out = ops.apply_logit_rules(s.logits.to(DEV), s.rules, torch.empty(4, 5000, device=DEV))
    s.check(out)
    again = s.t["history"].clone()
    s.choose(append=True)
    changed = (s.t["history"] != again).any(1).nonzero().flatten().tolist()
    assert set(changed) <= {s.slot[0], s.slot[2]}


@pytest.mark.parametrize("what,code,value", [("slot", 5, 99), ("total_len", 2, 1000), ("total_len", 2, -3), ("bias_len", 2, 50), ("mask_row", 5, 4),
                                             ("history", 1, 5000), ("history", 1, -1), ("bias_tokens", 1, 70000)])
def test_numbers_out_of_range_are_reported(ops, what, code, value):
    s = Step(ops, 1, 5000, seed=7, width=30)
    s.rep, s.total, s.prompt, s.bias_len, s.mask_row = [1.3], [30], [4], [5], [-1]
    s.build()
    t = s.t[what]
    if t.dim() == 1:
        t[0] = value
    else:
        t[s.slot[0], 3] = value
    x = s.logits.to(DEV)
    for run in (lambda: ops.apply_logit_rules(x, s.rules, torch.empty_like(x)), s.choose):
        run()
        torch.cuda.synchronize()
        got = ops.range_report().tolist()
        assert got[0] == code and got[1] == 15 and got[3] == value
        with pytest.raises(ops.KernelError, match="skipped"):
            ops.check_range_errors()


def test_captured_rules_follow_their_contents(ops):
    s = Step(ops, 5, 20001, seed=9)
    x, out, lp = s.logits.to(DEV), torch.empty(5, 20001, device=DEV), torch.empty(5, device=DEV)
    a = s.arrays()

    def step():
        ops.apply_logit_rules(x, s.rules, out)
        ops.sample(x, a["temperature"], a["request"], a["position"], 3, a["out"], rules=s.rules, logprob=lp)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step()
    other = Step(ops, 5, 20001, seed=10)
    for name, t in s.t.items():
        t.copy_(other.t[name])
    x.copy_(other.logits)
    graph.replay()
    torch.cuda.synchronize()
    other.check(out)
    tokens, lp2 = other.choose()
    assert torch.equal(tokens, a["out"]) and torch.equal(lp, lp2)


def test_many_rows_and_a_second_stream(ops):
    s = Step(ops, 300, 1500, seed=11, width=200)
    x, out = s.logits.to(DEV), torch.empty(300, 1500, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.apply_logit_rules(x, s.rules, out)
    side.synchronize()
    s.check(out)


def test_no_rows(ops):
    rules = ops.LogitRules(mask=torch.zeros(1, 2, dtype=torch.int32, device=DEV), mask_row=torch.empty(0, dtype=torch.int32, device=DEV))
    x = torch.empty(0, 40, device=DEV)
    assert ops.apply_logit_rules(x, rules, torch.empty_like(x)).shape == (0, 40)


@pytest.mark.parametrize("rows,vocab,width", [(3, 1000, 6000), (9, 50001, 9000), (2, 70001, 17000)])
def test_the_same_call_gives_the_same_bits(ops, rows, vocab, width):
    """Texts that name the same tokens again and again: whichever thread comes to one first, the sums are the same."""
    s = Step(ops, rows, vocab, width=width, seed=vocab)
    s.total = [width - r for r in range(rows)]
    s.rep, s.pres = [1.3] * rows, [0.7] * rows
    s.build()
    logits, first = s.logits.to(DEV), None
    for _ in range(30):
        tokens, lp = s.choose(logits, temperature=0.8)
        now = (tokens.tolist(), lp.view(torch.int32).tolist())
        first = first or now
        assert now == first


@pytest.mark.parametrize("vocab,width", [(700, 300), (50001, 4000), (140001, 9000)])
@pytest.mark.parametrize("lift", [3.0, 4.5, 30.0, 500.0, None])
def test_texts_far_above_the_rest(ops, vocab, width, lift):
    """The text's tokens lead the others by ``lift`` (None: the mask leaves the text's alone): their sum is taken against their own greatest, and the same call
    gives the same bits."""
    rows = 3
    s = Step(ops, rows, vocab, width=width, biases=0, seed=vocab)
    s.total, s.rep, s.pres = [width, width - 7, width // 2], [1.0, 1.3, 0.8], [0.0, -0.4, 0.7]
    if lift is not None:
        for r in range(rows):
            at = torch.tensor(sorted(set(s.text[s.slot[r]][:s.total[r]])))
            s.logits[r, at] = s.logits[r, at].abs() + lift
        s.mask_row = [-1, -1, -1]
    else:
        s.allowed = [sorted(set(s.text[s.slot[r]][:s.total[r]])) for r in range(rows)]
        s.mask = [words_of(a, -(-vocab // 32)) for a in s.allowed]
        s.mask_row = list(range(rows))
    s.build()
    logits, first = s.logits.to(DEV), None
    for _ in range(10):
        tokens, lp = s.choose(logits)
        now = (tokens.tolist(), lp.view(torch.int32).tolist())
        first = first or now
        assert now == first
    for r in range(rows):
        want, bound = s.row(r)
        best = int(tokens[r])
        assert want[best] >= want.max() - 2 * float(bound.max())
        want_lp = float(torch.log_softmax(want, 0)[best])
        assert abs(float(lp[r]) - want_lp) <= logprob_bound(want) + float(bound.max()) * 2, (r, float(lp[r]), want_lp)
