"""Timed operators: what a decode step needs when requests share the beginning of their prompts and draw from filtered
distributions.

    attention   softmax attention of a step over paged keys and values whose requests fall into groups: the members of a group
                have their first `prefix` keys in the same pages, and behind these each has pages of its own.  A request of no
                group has only pages of its own.  Steps bring one token a request, or a portion of a prompt each.

                    out[t, h] = sum_j softmax_j(scale * q[t, h] . k[j, h // (heads / kv_heads)]) v[j, .]     j <= position of t

    sample      one token for every row of logits.  z = (logit - largest) / temperature, w = exp(z); in the order of falling logits
                (equal ones by index) a row keeps the first top_k tokens, of those the ones with a sum of w in front of them below
                top_p times their whole sum, of those the ones with w >= min_p, and always the first; the token is the kept one with
                the largest z - log(-log(u)), u a number in (0, 1) that a hash makes of the row's key and counter and the token's
                index.  Temperature 0: the largest logit.  NaN is as -infinity.

Attention's head layouts are those of the Qwen3 sizes that bench.py runs (32, 40 and 64 query heads on 8 of 128) and of the smaller
decoders; prefixes run from a page to the benchmark's context of 8192, batches to its 64 requests; 151936, 32000 and small odd
numbers are this repository's vocabularies.
"""
import math

import torch

own = False

DEV = "cuda:0"


def listed():
    return [
        # two answers to one short question, a few tokens in: the smallest step there is
        dict(name="attention 2 x (256 + 9)", op="attention", dtype="bfloat16", heads=16, kv_heads=4, dim=128, page=16, groups=1, members=2, alone=0, prefix=256, most=9, portion=1),
        # eight answers to one long prompt
        dict(name="attention 8 x (8192 + 100)", op="attention", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=16, groups=1, members=8, alone=0, prefix=8192, most=100, portion=1),
        # a full batch behind one long document, answers of up to 256 tokens: the largest
        dict(name="attention 64 x (8192 + 256)", op="attention", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=16, groups=1, members=64, alone=0, prefix=8192, most=256, portion=1),
        # three groups with prompts of their own beside requests that share nothing; five query heads a kv head
        dict(name="attention 3 groups and 5 alone", op="attention", dtype="bfloat16", heads=40, kv_heads=8, dim=128, page=16, groups=3, members=11, alone=5, prefix=2352, most=777, portion=1),
        # every member's own question is being read behind a common system prompt
        dict(name="attention portions 8 x 37", op="attention", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=16, groups=1, members=8, alone=0, prefix=2000, most=61, portion=37),
        # the 32-bit path, heads of 64
        dict(name="attention float32 6 x (1000 + 50)", op="attention", dtype="float32", heads=16, kv_heads=4, dim=64, page=8, groups=1, members=6, alone=0, prefix=1000, most=50, portion=1),
        # one request of a small vocabulary
        dict(name="sample 1 x 32000 top-p", op="sample", rows=1, vocab=32000, filters="top_p", values="smooth"),
        # one request, all filters
        dict(name="sample 1 x 151936 all", op="sample", rows=1, vocab=151936, filters="all", values="smooth"),
        # the benchmark's batch of eight, every request with filters of its own, some greedy
        dict(name="sample 8 x 151936 mixed", op="sample", rows=8, vocab=151936, filters="mixed", values="smooth"),
        # a full batch of nucleus sampling over logits of 16-bit steps: many equal values
        dict(name="sample 64 x 151936 top-p ties", op="sample", rows=64, vocab=151936, filters="top_p", values="stepped"),
        # an odd vocabulary of which most is masked, as a grammar does
        dict(name="sample 37 x 50003 masked", op="sample", rows=37, vocab=50003, filters="mixed", values="masked"),
        # the most requests an engine runs at a time
        dict(name="sample 256 x 151936 mixed", op="sample", rows=256, vocab=151936, filters="mixed", values="smooth"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    if rng.random() < 0.5:
        vocab = rng.choice([151936, 151936, 32000, log(256, 151936)])
        rows = min(log(1, 256), 256 * 151936 // vocab)
        return dict(op="sample", rows=rows, vocab=vocab, filters=rng.choice(["top_k", "top_p", "min_p", "all", "mixed", "mixed"]),
                    values=rng.choice(["smooth", "smooth", "stepped", "masked"]))
    f32 = rng.random() < 0.2
    heads, kv_heads = rng.choice([(32, 8), (40, 8), (64, 8), (16, 4), (16, 16), (8, 1)])
    page = rng.choice([8, 16, 16, 32])
    groups = rng.choice([1, 1, 1, 2, 3, 4])
    members = max(2, log(2, 64) // groups)
    alone = rng.choice([0, 0, log(1, 8)])
    prefix = page * max(1, log(page, 1024 if f32 else 8192) // page)
    most = log(1, 64 if f32 else 512)
    portion = 1 if f32 or rng.random() < 0.7 else log(2, 48)
    if portion > 1:                                  # a step brings as many tokens as its budget has
        members = max(2, min(members, 512 // (groups * portion)))
        alone = min(alone, 2)
    seqs = groups * members + alone
    while seqs * portion * heads * (prefix + most + portion) > (1 << 29) or seqs * (prefix + most) * kv_heads > 64 * 8448 * 8:
        prefix = page * max(1, prefix // page // 2)
        if prefix == page:
            most = max(1, most // 2)
    return dict(op="attention", dtype="float32" if f32 else "bfloat16", heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), page=page,
                groups=groups, members=members, alone=alone, prefix=prefix, most=most, portion=portion)


# ---- sizes -----------------------------------------------------------------------------------------------------

def batch(case, seed):
    """(group of each request or -1, prefix of each group, new tokens and length of each request), on the host: requests of all
    groups and of none in one mixed order, groups' prefixes from half the case's to all of it, own parts from one token to `most`.  The new tokens are the same for every seed."""
    g = torch.Generator().manual_seed(seed)
    page, most, portion = case["page"], case["most"], case["portion"]
    group = [i for i in range(case["groups"]) for _ in range(case["members"])] + [-1] * case["alone"]
    group = [group[i] for i in torch.randperm(len(group), generator=g).tolist()]
    pages = case["prefix"] // page
    prefix = [page * (pages - i * (pages // 2) // case["groups"]) for i in range(case["groups"])]
    share = torch.rand(len(group), generator=torch.Generator().manual_seed(len(group))).tolist()
    new = [max(1, int(portion * (0.5 + 0.5 * r) + 0.5)) for r in share]
    own_part = torch.randint(1, most + 1, (len(group),), generator=g).tolist()
    length = [(prefix[i] if i >= 0 else 0) + p + n - 1 for i, p, n in zip(group, own_part, new)]
    return group, prefix, new, length


def work(case):
    if case["op"] == "sample":
        return {"bytes": 4.0 * case["rows"] * (case["vocab"] + 8), "flops": 4.0 * case["rows"] * case["vocab"]}
    group, prefix, new, length = batch(case, 0)
    el = 2 if case["dtype"] == "bfloat16" else 4
    cached = sum(prefix) + sum(n - (prefix[i] if i >= 0 else 0) for i, n in zip(group, length))
    seen = sum(n * c - n * (n - 1) // 2 for n, c in zip(new, length))
    ints = 4 * (sum(-(-c // case["page"]) for c in length) + 4 * len(group))
    return {"bytes": float(el * case["dim"] * (2 * cached * case["kv_heads"] + 2 * sum(new) * case["heads"]) + ints),
            "flops": 4.0 * case["dim"] * case["heads"] * seen}


# ---- inputs ----------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, gen)
    group, prefix, new, length = batch(case, seed)
    page, dtype = case["page"], getattr(torch, case["dtype"])
    S, T = len(group), sum(new)
    behind = [-(-c // page) - (prefix[i] // page if i >= 0 else 0) for i, c in zip(group, length)]
    count = sum(p // page for p in prefix) + sum(behind)
    ids = torch.randperm(count, generator=torch.Generator().manual_seed(seed + 1)).tolist()
    shared = []
    for p in prefix:
        shared.append([ids.pop() for _ in range(p // page)])
    table = torch.full((S, max(-(-c // page) for c in length) + 3), -1, dtype=torch.int32)
    leader = {}
    prefix_of, prefix_lens = [-1] * S, [0] * S
    for s, i in enumerate(group):
        row = (shared[i] if i >= 0 else []) + [ids.pop() for _ in range(behind[s])]
        table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
        if i >= 0:
            prefix_of[s] = leader.setdefault(i, s)
            prefix_lens[prefix_of[s]] = prefix[i]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    kv = (count, case["kv_heads"], page, case["dim"])
    ints = dict(cu_tokens=cu, context_lens=length, prefix_of=prefix_of, prefix_lens=prefix_lens)
    state = {k: torch.tensor(v, dtype=torch.int32, device=DEV) for k, v in ints.items()}
    state.update(case=case, q=torch.randn(T, case["heads"], case["dim"], generator=gen, device=DEV).to(dtype),
                 k=torch.randn(kv, generator=gen, device=DEV).to(dtype), v=torch.randn(kv, generator=gen, device=DEV).to(dtype),
                 table=table.to(DEV), max_new=max(new), scale=1.0 / math.sqrt(case["dim"]))
    return state


def _prepare_sample(case, gen):
    R, V = case["rows"], case["vocab"]
    # rows of different sharpness, a few dozen tokens above the rest
    logits = torch.randn(R, V, generator=gen, device=DEV) * (1.0 + 2.0 * torch.rand(R, 1, generator=gen, device=DEV))
    at = torch.randint(0, V, (R, 48), generator=gen, device=DEV)
    logits += torch.zeros_like(logits).scatter_reduce_(1, at, 8.0 * torch.rand(R, 48, generator=gen, device=DEV), "amax")
    if case["values"] == "stepped":
        logits = logits.to(torch.bfloat16).float()
    if case["values"] == "masked":                    # up to 99 in 100 tokens are not allowed
        allowed = torch.rand(R, V, generator=gen, device=DEV) < 0.01 + 0.5 * torch.rand(R, 1, generator=gen, device=DEV)
        allowed[:, 0] = True
        logits = logits.masked_fill(~allowed, -math.inf)
    pick = torch.randint(0, 6, (R,), generator=gen, device=DEV)
    mixed, every = case["filters"] == "mixed", case["filters"] == "all"
    use_k = (pick == 0) | (pick == 2) if mixed else torch.full_like(pick, every or case["filters"] == "top_k", dtype=torch.bool)
    use_p = (pick == 1) | (pick == 2) | (pick == 4) if mixed else torch.full_like(pick, every or case["filters"] == "top_p", dtype=torch.bool)
    use_m = (pick == 3) | (pick == 4) if mixed else torch.full_like(pick, every or case["filters"] == "min_p", dtype=torch.bool)
    rand = lambda lo, hi: lo + (hi - lo) * torch.rand(R, generator=gen, device=DEV)      # noqa: E731
    temperature = torch.where(pick == 5, 0.0, rand(0.5, 1.5)) if mixed else rand(0.5, 1.5)
    return dict(case=case, logits=logits, temperature=temperature.float(),
                top_k=torch.where(use_k, torch.exp(rand(math.log(2), math.log(200))).int(), 0).int(),
                top_p=torch.where(use_p, 1.0 - torch.exp(rand(math.log(0.01), math.log(0.6))), 1.0).float(),
                min_p=torch.where(use_m, torch.exp(rand(math.log(0.005), math.log(0.3))), 0.0).float(),
                keys=torch.randint(-2 ** 63, 2 ** 63 - 1, (R,), generator=gen, device=DEV),
                counters=torch.randint(0, 4096, (R,), generator=gen, device=DEV).int())


# ---- one pass --------------------------------------------------------------------------------------------------

def run(state):
    if state["case"]["op"] == "sample":
        return _own_sample(state) if own else _plain_sample(state)
    return _own_attention(state) if own else _plain_attention(state)


def _own_attention(st):
    from lucciola_b200 import ops
    c = st["case"]
    out = torch.empty_like(st["q"])
    ops.attention_shared(st["q"], out, st["k"], st["v"], st["table"], st["cu_tokens"], st["context_lens"], st["prefix_of"], st["prefix_lens"],
                         st["max_new"], c["heads"], c["kv_heads"], c["dim"], c["page"], st["scale"], ops.current_stream())
    return out


def _own_sample(st):
    from lucciola_b200 import ops
    tokens = torch.empty(st["logits"].shape[0], dtype=torch.int32, device=st["logits"].device)
    ops.sample(tokens, st["logits"], ops.current_stream(), st["temperature"], st["keys"], st["counters"],
               top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])
    return tokens


def _plain_attention(st):
    """Every request gathers all its keys and values through its own table; requests side by side, padded to the longest."""
    c, q, table = st["case"], st["q"], st["table"].long()
    S, d, kv, g = table.shape[0], c["dim"], c["kv_heads"], c["heads"] // c["kv_heads"]
    cu, length = st["cu_tokens"].long(), st["context_lens"].long()
    new = cu[1:] - cu[:-1]
    at = torch.arange(st["max_new"], device=DEV)
    here = at < new[:, None]                                                              # [S, N]
    place = torch.where(here, cu[:-1, None] + at, 0)
    position = (length - new)[:, None] + at
    qp = q[place].float().view(S, -1, kv, g, d)
    k = st["k"][table.clamp(min=0)].transpose(2, 3).reshape(S, -1, kv, d).float()
    v = st["v"][table.clamp(min=0)].transpose(2, 3).reshape(S, -1, kv, d).float()
    score = torch.einsum("snkgd,slkd->skgnl", qp, k) * st["scale"]
    key = torch.arange(k.shape[1], device=DEV)
    score = score.masked_fill(~(key <= position[:, :, None])[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.einsum("skgnl,slkd->snkgd", p, v) / p.sum(-1).permute(0, 3, 1, 2)[..., None]
    return o.reshape(S, -1, c["heads"], d)[here].to(q.dtype)


def _shift(x, n):
    """x >> n of 64 bits without a sign."""
    return (x >> n) & ((1 << (64 - n)) - 1)


def _mix(x):
    x = (x ^ _shift(x, 30)) * (0xBF58476D1CE4E5B9 - (1 << 64))
    x = (x ^ _shift(x, 27)) * (0x94D049BB133111EB - (1 << 64))
    return x ^ _shift(x, 31)


def _plain_sample(st):
    """In 64 bits: a kept token's place next to the border, and two nearly equal scores, decide the result."""
    logits = st["logits"].double()
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    R, V = logits.shape
    top, order = torch.sort(logits, dim=1, descending=True, stable=True)
    hot = st["temperature"] > 0
    z = (top - top[:, :1]) / torch.where(hot, st["temperature"], 1.0).double()[:, None]
    w = torch.exp(z)
    rank = torch.arange(V, device=DEV)
    k = torch.where(st["top_k"] > 0, st["top_k"], V).long()
    keep = rank < k[:, None]
    w = w * keep
    total = torch.cumsum(w, 1)
    keep = keep & (((total - w) < st["top_p"].double()[:, None] * total[:, -1:]) | (st["top_p"] >= 1)[:, None])
    keep = keep & (w >= st["min_p"].double()[:, None])
    keep[:, 0] = True
    start = _mix(st["keys"] + (0x9E3779B97F4A7C15 - (1 << 64)) * (st["counters"].long() + 1))
    bits = _shift(_mix(start[:, None] ^ ((0xD6E8FEB86659FD93 - (1 << 64)) * (order + 1))), 41)
    u = (bits.double() + 0.5) / 2 ** 23
    score = torch.where(keep, z - torch.log(-torch.log(u)), -math.inf)
    best = score.amax(1, keepdim=True)
    token = torch.where(score == best, order, V).amin(1)
    return torch.where(hot, token, order[:, 0]).int()


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return _exact_sample(st) if case["op"] == "sample" else _exact_attention(st)


def _exact_attention(st):
    """Request by request, its keys in one piece."""
    c = st["case"]
    q, d, g = st["q"].double(), c["dim"], c["heads"] // c["kv_heads"]
    out = torch.empty_like(q)
    cu, length = st["cu_tokens"].tolist(), st["context_lens"].tolist()
    for s, n in enumerate(length):
        pages = st["table"][s, :-(-n // c["page"])].long()
        keys = [st[x].index_select(0, pages).double().permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, d)[:, :n] for x in ("k", "v")]
        a, b = cu[s], cu[s + 1]
        rows = q[a:b].reshape(b - a, c["kv_heads"], g * d).permute(1, 0, 2).reshape(c["kv_heads"], (b - a) * g, d)
        score = rows @ keys[0].transpose(1, 2) / math.sqrt(d)
        last = (n - (b - a) + torch.arange(b - a, device=DEV)).repeat_interleave(g)
        score = score + torch.where(torch.arange(n, device=DEV)[None] > last[:, None], -math.inf, 0.0)
        o = torch.softmax(score, -1) @ keys[1]
        out[a:b] = o.reshape(c["kv_heads"], b - a, g * d).permute(1, 0, 2).reshape(b - a, c["heads"], d)
    return out


def _exact_sample(st):
    """Row by row: the kept tokens are counted out by the value of the last of them, not through one sorted order of all."""
    V = st["logits"].shape[1]
    tokens = []
    index = torch.arange(V, device=DEV)
    M = (1 << 64) - 1
    for r in range(st["logits"].shape[0]):
        x = st["logits"][r].double()
        x[x != x] = -math.inf
        most = x.max()
        first = int(torch.nonzero(x == most)[0])
        t = float(st["temperature"][r])
        if not t > 0 or math.isinf(float(most)):
            tokens.append(first)
            continue
        z = (x - most) / t
        w = torch.exp(z)
        left = index
        k = int(st["top_k"][r])
        if 0 < k < V:
            border = torch.kthvalue(x, V - k + 1).values
            above, equal = torch.nonzero(x > border)[:, 0], torch.nonzero(x == border)[:, 0]
            left = torch.cat([above, equal[:k - len(above)]])
        p = float(st["top_p"][r])
        left = left[torch.argsort(left)]
        left = left[torch.argsort(x[left], descending=True, stable=True)]
        if p < 1:
            s = torch.cumsum(w[left], 0)
            in_front = torch.cat([torch.zeros(1, dtype=torch.float64, device=DEV), s[:-1]])
            left = left[:max(1, int((in_front < p * s[-1]).sum()))]
        left = left[:max(1, int((w[left] >= float(st["min_p"][r])).sum()))]
        key = (int(st["keys"][r]) + 0x9E3779B97F4A7C15 * (int(st["counters"][r]) + 1)) & M
        for n, f in ((30, 0xBF58476D1CE4E5B9), (27, 0x94D049BB133111EB)):
            key = (key ^ (key >> n)) * f & M
        key ^= key >> 31
        h = (left + 1) * (0xD6E8FEB86659FD93 - (1 << 64)) ^ (key - (1 << 64) if key >> 63 else key)
        for n, f in ((30, 0xBF58476D1CE4E5B9), (27, 0x94D049BB133111EB)):
            h = (h ^ ((h >> n) & (M >> n))) * (f - (1 << 64))
        h = h ^ ((h >> 31) & (M >> 31))
        u = (2 * ((h >> 41) & 0x7FFFFF) + 1).double() / 2 ** 24
        score = z[left] - torch.log(-torch.log(u))
        tokens.append(int(left[score == score.max()].min()))
    return torch.tensor(tokens, dtype=torch.int32, device=DEV)
