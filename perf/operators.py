"""Operators of serving several answers to one prompt, as cases that can be timed and checked: decode attention of a batch whose rows
share a long prefix, rules on logits (penalties for repeated tokens, biases, grammar masks), and the choice of a token under such rules
with its log-probability.

A case is a dict of plain values; ``op`` says what runs.  ``own`` (set from outside) chooses between the framework's kernels and plain torch
operations in 32 bits."""
import math

import torch

own = False

DEV = "cuda"


# --------------------------------------------------------------------------- the cases

def _prefix(groups, own_keys, heads, kv_heads, dim, page=16, name=None):
    """``groups``: "rows:prefix" separated by blanks; every row has 1 to ``own_keys`` keys behind its group's prefix."""
    c = dict(op="prefix", groups=groups, own_keys=own_keys, heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    return c if name is None else dict(name=name, **c)


def _logits(op, rows, vocab, prompt, answer, bias, grammar, name=None):
    """Rows of up to ``prompt`` prompt and ``answer`` generated tokens, ``bias`` biased tokens each, one in ``grammar`` rows without a mask of
    its own (0: no masks at all)."""
    c = dict(op=op, rows=rows, vocab=vocab, prompt=prompt, answer=answer, bias=bias, grammar=grammar)
    return c if name is None else dict(name=name, **c)


def listed():
    return [
        # two answers to a short question, just begun: the smallest step that shares anything, all latency (TinyLlama's heads)
        _prefix("2:208", 5, 32, 4, 64, name="prefix-2-short"),
        # eight answers to one prompt of the benchmark's long size
        _prefix("8:2048", 120, 32, 4, 64, name="prefix-8"),
        # 64 users behind one long system prompt, in the middle of their own conversations (Llama-3-8B's heads)
        _prefix("64:8000", 512, 32, 8, 128, name="prefix-64"),
        # the largest: 256 samples of one long document
        _prefix("256:16384", 96, 32, 8, 128, name="prefix-256-long"),
        # a mixed batch: several prompts of odd lengths, some rows alone, one key head a query head (Llama-2-7B's heads)
        _prefix("17:3001 5:700 1:0 1:0 9:1537", 300, 32, 32, 128, name="prefix-groups"),
        # heads of another size, groups of six
        _prefix("12:999 3:50 20:2500", 77, 24, 4, 96, page=32, name="prefix-heads-96"),
        # one user's step: penalties over a short history
        _logits("rules", 1, 32000, 40, 24, 0, 0, name="rules-1"),
        # 64 users of a large vocabulary, every rule in use
        _logits("rules", 64, 128256, 1500, 500, 24, 2, name="rules-64"),
        # the largest: 256 users, long histories
        _logits("rules", 256, 128256, 6000, 2000, 100, 3, name="rules-256-long"),
        # the choice of a token: eight answers, penalties and a few biases
        _logits("choose", 8, 32000, 512, 100, 8, 0, name="choose-8"),
        # 64 answers that a grammar holds, large vocabulary
        _logits("choose", 64, 128256, 700, 300, 16, 4, name="choose-64"),
        # 200 rows, odd vocabulary
        _logits("choose", 200, 50001, 3000, 900, 50, 2, name="choose-200-odd"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _groups(case):
    return [tuple(int(v) for v in g.split(":")) for g in case["groups"].split()]


def draw(rng):
    if rng.random() < 0.5:
        most = work(listed()[3])["flops"]
        while True:
            heads, kv_heads, dim = rng.choice([(32, 4, 64), (32, 8, 128), (32, 32, 128), (24, 4, 96), (6, 2, 64), (20, 1, 128), (10, 10, 80), (7, 1, 16), (16, 4, 112)])
            groups = " ".join("%d:%d" % (_spread(rng, 1, 256), 0 if rng.random() < 0.1 else _spread(rng, 1, 16384)) for _ in range(rng.choice([1, 1, 2, 3, 6])))
            c = _prefix(groups, _spread(rng, 1, 1024), heads, kv_heads, dim, rng.choice([8, 16, 16, 32, 64]))
            rows = sum(n for n, _ in _groups(c))
            if 2 <= rows <= 256 and work(c)["flops"] <= most and work(c)["bytes"] <= 2 << 30:
                return c
    return _logits(rng.choice(["rules", "choose"]), _spread(rng, 1, 256), rng.choice([_spread(rng, 200, 128256), 32000, 128256, 50001]), _spread(rng, 1, 6000),
                   _spread(rng, 1, 2000), rng.choice([0, 1, _spread(rng, 1, 300)]), rng.choice([0, 1, 2, 3]))


def _own_lengths(case):
    n = sum(r for r, _ in _groups(case))
    return [1 + (r * 7919 + 13) % case["own_keys"] for r in range(n)]


def work(case):
    if case["op"] == "prefix":
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        lens, at, keys, met = _own_lengths(case), 0, 0, 0
        for n, prefix in _groups(case):
            own_keys = sum(lens[at:at + n])
            keys += prefix + own_keys
            met += n * prefix + own_keys
            at += n
        return {"bytes": 2 * 2 * keys * G * D + 2 * 2 * at * H * D, "flops": 4 * D * H * met}
    R, V = case["rows"], case["vocab"]
    lens = _history_lengths(case)
    read = R * V * 4 + 4 * sum(p + a for p, a in lens) + 8 * R * case["bias"]
    if case["grammar"]:
        read += (R - R // case["grammar"]) * (-(-V // 32) * 4)
    return {"bytes": read + (R * V * 4 if case["op"] == "rules" else 8 * R), "flops": (4 if case["op"] == "rules" else 8) * R * V}


def _history_lengths(case):
    R = case["rows"]
    return [(1 + (r * 6151 + case["prompt"] - 1) % case["prompt"], (r * 3571 + case["answer"]) % (case["answer"] + 1)) for r in range(R)]


# --------------------------------------------------------------------------- what a program has in hand

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (_prepare_prefix if case["op"] == "prefix" else _prepare_logits)(case, g)


def _prepare_prefix(case, g):
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    groups, lens = _groups(case), _own_lengths(case)
    rows = len(lens)
    # pages: a group's whole shared pages once, every row's own behind them (a prefix that ends inside a page: the row's own copy of
    # that page holds its own keys only, the first row's holds the prefix's end as well)
    need, at = 1, 0
    plan = []                                             # per row: (shared pages' first, how many, own pages' first, how many)
    for n, prefix in groups:
        shared, first = prefix // page, need
        need += shared
        for r in range(at, at + n):
            mine = -(-(prefix + lens[r]) // page) - shared
            plan.append((first, shared, need, mine))
            need += mine
        at += n
    order = torch.randperm(need - 1, generator=g, device=DEV).cpu() + 1
    width = max(s + m for _, s, _, m in plan)
    tables = torch.zeros(rows, width, dtype=torch.int32)
    for r, (f, s, o, m) in enumerate(plan):
        tables[r, :s] = order[f - 1:f - 1 + s]
        tables[r, s:s + m] = order[o - 1:o - 1 + m]
    cache = torch.randn(2, need, G, page, D, generator=g, device=DEV, dtype=torch.float32).to(torch.bfloat16)
    qkv = torch.randn(rows, (H + 2 * G) * D, generator=g, device=DEV, dtype=torch.float32).mul_(1.5).to(torch.bfloat16)
    start = [0]
    for n, _ in groups:
        start.append(start[-1] + n)
    prefixes = [p for _, p in groups]
    ctx = [p + lens[r] for (n, p), s in zip(groups, start) for r in range(s, s + n)]
    i32 = dict(dtype=torch.int32, device=DEV)
    return dict(case=case, qkv=qkv, cache=cache, tables=tables.to(DEV), group_start=torch.tensor(start, **i32), group_prefix=torch.tensor(prefixes, **i32),
                q_start=torch.arange(rows, **i32), q_len=torch.ones(rows, **i32), ctx_len=torch.tensor(ctx, **i32),
                out=torch.empty(rows, H, D, dtype=torch.bfloat16, device=DEV), groups=groups, starts=start, ctx=ctx,
                max_prefix=max(prefixes), max_own=max(lens), scale=1.0 / math.sqrt(D))


def _prepare_logits(case, g):
    R, V = case["rows"], case["vocab"]
    lens = _history_lengths(case)
    slots, width = R + 3, case["prompt"] + case["answer"] + 2
    # texts repeat themselves: tokens are drawn with a heavy head
    u = torch.rand(slots, width, generator=g, device=DEV)
    history = (u.pow(6) * V).long().clamp_(max=V - 1).to(torch.int32)
    slot = torch.randperm(slots, generator=g, device=DEV)[:R].to(torch.int32)
    f32, i32 = dict(dtype=torch.float32, device=DEV), dict(dtype=torch.int32, device=DEV)

    def of_rows(lo, hi, off):                             # a third of the rows does without
        v = torch.rand(R, generator=g, device=DEV) * (hi - lo) + lo
        return torch.where(torch.arange(R, device=DEV) % 3 == 2, torch.full_like(v, off), v)

    s = dict(case=case, logits=torch.randn(R, V, generator=g, **f32).mul_(3.0), history=history, slot=slot,
             prompt_len=torch.tensor([p for p, _ in lens], **i32), total_len=torch.tensor([p + a for p, a in lens], **i32),
             repetition=of_rows(1.05, 1.5, 1.0), presence=of_rows(-0.5, 1.5, 0.0), frequency=of_rows(0.0, 0.7, 0.0),
             bias_tokens=None, bias_values=None, bias_len=None, mask=None, mask_row=None)
    if case["bias"]:
        n = min(case["bias"], V)
        s["bias_tokens"] = torch.rand(slots, V, generator=g, device=DEV).topk(n, dim=1).indices.to(torch.int32).contiguous()
        values = torch.randn(slots, n, generator=g, **f32).mul_(4.0)
        values[:, ::5] = float("-inf")                    # a ban
        s["bias_values"] = values
        s["bias_len"] = torch.tensor([n - r % (n + 1) if r % 4 == 3 else n for r in range(R)], **i32)
    if case["grammar"]:
        words = -(-V // 32)
        masks = max(1, R // 2)
        # what a grammar allows next: a few tokens, or most of them
        few = torch.zeros(masks, words * 32, dtype=torch.bool, device=DEV)
        few.scatter_(1, torch.randint(0, V, (masks, min(V, 40)), generator=g, device=DEV), True)
        most = torch.rand(masks, words * 32, generator=g, device=DEV) < 0.7
        bits = torch.where((torch.arange(masks, device=DEV) % 2 == 0)[:, None], few, most)
        bits[:, V:] = True                                # bits behind the vocabulary mean nothing
        weights = 1 << torch.arange(32, dtype=torch.int64, device=DEV)
        packed = (bits.view(masks, words, 32).long() * weights).sum(-1)
        s["mask"] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
        s["mask_row"] = torch.tensor([-1 if r % case["grammar"] == 0 and case["grammar"] > 1 else r % masks for r in range(R)], **i32)
    if case["op"] == "rules":
        s["out"] = torch.empty(R, V, **f32)
    else:
        s.update(temperature=torch.zeros(R, **f32), request=torch.arange(R, dtype=torch.int64, device=DEV), position=torch.zeros(R, **i32),
                 token=torch.empty(R, **i32), logprob=torch.empty(R, **f32))
    if own:
        from mini_inference_engine_b200.kernels import ops
        s["rules"] = ops.LogitRules(s["history"], s["slot"], s["prompt_len"], s["total_len"], repetition=s["repetition"], presence=s["presence"],
                                    frequency=s["frequency"], bias_tokens=s["bias_tokens"], bias_values=s["bias_values"], bias_len=s["bias_len"],
                                    mask=s["mask"], mask_row=s["mask_row"])
    return s


# --------------------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    if case["op"] == "prefix":
        return _own_prefix(s) if own else _plain_prefix(s)
    if own:
        from mini_inference_engine_b200.kernels import ops
        if case["op"] == "rules":
            return ops.apply_logit_rules(s["logits"], s["rules"], s["out"])
        ops.sample(s["logits"], s["temperature"], s["request"], s["position"], 0, s["token"], rules=s["rules"], logprob=s["logprob"])
        return s["token"], s["logprob"]
    x = _plain_rules(s)
    if case["op"] == "rules":
        return x
    token = _first_largest(x)
    top = x.amax(1, keepdim=True)
    total = torch.exp(x - top).sum(1)
    return token.to(torch.int32), x.gather(1, token[:, None]).squeeze(1) - (top.squeeze(1) + torch.log(total))


def _own_prefix(s):
    from mini_inference_engine_b200.kernels import ops
    c = s["case"]
    return ops.shared_prefix_attention(s["qkv"], s["qkv"].shape[1], s["cache"][0], s["cache"][1], s["tables"], s["q_start"], s["q_len"], s["ctx_len"],
                                       s["group_start"], s["group_prefix"], s["out"], c["heads"], c["kv_heads"], c["dim"], c["page"], s["scale"],
                                       max_prefix=s["max_prefix"], max_own=s["max_own"])


def _plain_prefix(s):
    c = s["case"]
    H, G, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    out = []
    for (n, prefix), first in zip(s["groups"], s["starts"]):
        q = s["qkv"][first:first + n, :H * D].float().view(n, G, H // G, D) * s["scale"]
        pages = s["tables"][first, :-(-prefix // page)].long()
        k, v = (t[pages].float().transpose(0, 1).reshape(G, -1, D)[:, :prefix] for t in s["cache"])
        before = torch.einsum("nghd,gkd->nghk", q, k)
        longest = max(s["ctx"][first:first + n]) - prefix
        places = prefix + torch.arange(longest, device=DEV)
        page_of = (places // page).clamp(max=s["tables"].shape[1] - 1)
        at = s["tables"][first:first + n].long()[:, page_of]                     # [n, longest]
        mine_k, mine_v = (t[at, :, places % page].float() for t in s["cache"])       # [n, longest, G, D]
        behind = torch.einsum("nghd,nkgd->nghk", q, mine_k)
        seen = places[None, :] < s["ctx_len"][first:first + n, None]
        behind = behind.masked_fill(~seen[:, None, None, :], float("-inf"))
        top = behind.amax(-1, keepdim=True)
        if prefix:
            top = torch.maximum(top, before.amax(-1, keepdim=True))
        before, behind = torch.exp(before - top), torch.exp(behind - top)
        total = before.sum(-1) + behind.sum(-1)
        o = torch.einsum("nghk,gkd->nghd", before, v) + torch.einsum("nghk,nkgd->nghd", behind, mine_v)
        out.append((o / total[..., None]).reshape(n, H, D))
    return torch.cat(out).to(torch.bfloat16)


def _plain_rules(s):
    x = s["logits"]
    R, V = x.shape
    text = s["history"][s["slot"].long()].long()
    place = torch.arange(text.shape[1], device=DEV)[None, :]
    alive = place < s["total_len"][:, None]
    answer = alive & (place >= s["prompt_len"][:, None])
    met = torch.zeros(R, V, device=DEV).scatter_add_(1, text, alive.float()) > 0
    count = torch.zeros(R, V, device=DEV).scatter_add_(1, text, answer.float())
    rep = s["repetition"][:, None]
    x = torch.where(met, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias_tokens"] is not None:
        own_tokens, values = s["bias_tokens"][s["slot"].long()].long(), s["bias_values"][s["slot"].long()]
        on = torch.arange(own_tokens.shape[1], device=DEV)[None, :] < s["bias_len"][:, None]
        x = x.scatter_add(1, own_tokens, torch.where(on, values, torch.zeros_like(values)))
    if s["mask"] is not None:
        words = s["mask"][s["mask_row"].long().clamp(min=0)]
        bits = (words[:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        allowed = bits.view(R, -1)[:, :V].bool() | (s["mask_row"] < 0)[:, None]
        x = x.masked_fill(~allowed, float("-inf"))
    return x


def _first_largest(x):
    """The lowest index of a row's largest value."""
    V = x.shape[1]
    places = torch.where(x == x.amax(1, keepdim=True), torch.arange(V, device=DEV)[None, :], V)
    return places.amin(1)


# --------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prefix":
        return _exact_prefix(s)
    rows = [_exact_row(s, r) for r in range(case["rows"])]
    if case["op"] == "rules":
        return torch.stack(rows)
    token = torch.stack([(x == x.max()).nonzero()[0, 0] for x in rows]).to(torch.int32)
    return token, torch.stack([torch.log_softmax(x, 0)[t] for x, t in zip(rows, token.tolist())])


def _exact_prefix(s):
    c = s["case"]
    H, G, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    keys, values = s["cache"]
    out = []
    for (n, prefix), first in zip(s["groups"], s["starts"]):
        for r in range(first, first + n):
            place = torch.arange(s["ctx"][r], device=DEV)
            table = torch.where(place < prefix, s["tables"][first].long()[place // page], s["tables"][r].long()[place // page])
            k, v = keys[table, :, place % page].double(), values[table, :, place % page].double()         # [ctx, G, D]
            q = s["qkv"][r, :H * D].double().view(G, H // G, D)
            weights = torch.softmax(torch.matmul(q, k.permute(1, 2, 0)) * s["scale"], -1)
            out.append(torch.matmul(weights, v.transpose(0, 1)).reshape(H, D))
    return torch.stack(out)


def _exact_row(s, r):
    x = s["logits"][r].double()
    V = x.numel()
    i = int(s["slot"][r])
    p, n = int(s["prompt_len"][r]), int(s["total_len"][r])
    text = s["history"][i].long()
    met = torch.bincount(text[:n], minlength=V) > 0
    count = torch.bincount(text[p:n], minlength=V).double()
    rep = float(s["repetition"][r])
    x = torch.where(met, torch.where(x < 0, x * rep, x / rep), x)
    x = x - float(s["frequency"][r]) * count
    x = x - float(s["presence"][r]) * (count >= 1).double()
    if s["bias_tokens"] is not None:
        m = int(s["bias_len"][r])
        x[s["bias_tokens"][i, :m].long()] += s["bias_values"][i, :m].double()
    if s["mask"] is not None and int(s["mask_row"][r]) >= 0:
        place = torch.arange(V, device=DEV)
        word = s["mask"][int(s["mask_row"][r])].long()[place // 32]
        x[(word >> (place % 32)) % 2 == 0] = float("-inf")
    return x
