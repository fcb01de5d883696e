"""Operators of a decode step with drafted tokens and shared blocks, as cases that can be timed and compared.

``listed()`` and ``draw()`` give cases (dicts of plain values), ``prepare()`` makes the inputs of
one, and ``run()`` is one pass: in plain torch operations where ``own`` is false, through
``localstrm_b200`` where it is true.  ``exact()`` is the same result from the definition in
64 bits, and ``work()`` the bytes and operations that a pass cannot do without.

Operators (``case["op"]``):

* ``rotate``   norms of queries and keys for each head, with the position rotation in the same pass
* ``drafts``   the trees of a step's drafted tokens, and which of them the sampled tokens accept
* ``attend``   softmax attention over the paged 8-bit cache, each drafted token seeing the context and its own branch
* ``compact``  the accepted tokens' keys and values to their places in the cache
* ``pages``    blocks that several rows hold; ``case["call"]`` is ``fork`` (rows that go on from the tokens of others: their full
  blocks shared, the one that is not full copied) or ``release`` (blocks of stopped rows, and of rejected tokens, back to
  the free list once nobody holds them)
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # One request's next token, 14 query heads on 2 key heads of 64: the smallest call, latency counts.
        dict(name="rotate, 1 token", op="rotate", tokens=1, heads=2, per=7, dim=64, rot=64, interleaved=False, norm=True, fused=True, far=2000, x="f16"),
        # Prompt chunks of a batch, slices of one fused projection.
        dict(name="rotate, prompts", op="rotate", tokens=8192, heads=8, per=4, dim=128, rot=128, interleaved=False, norm=True, fused=True, far=131071, x="bf16"),
        # One request with a small tree of drafted tokens: latency.
        dict(name="drafts, 1 request", op="drafts", rows=1, block=16, ctx_lo=700, ctx_hi=700, new_lo=6, new_hi=6, stops=False),
        # A batch of requests with trees of uneven sizes, stop tokens among the sampled ones.
        dict(name="drafts, batch", op="drafts", rows=256, block=16, ctx_lo=0, ctx_hi=8000, new_lo=17, new_hi=64, stops=True),
        # The attention of the small tree over a short context: latency.
        dict(name="attend, 1 short request", op="attend", rows=1, block=16, heads=2, per=7, dim=64, ctx_lo=700, ctx_hi=700, new_lo=6, new_hi=6, x="f16"),
        # A decode batch with trees over contexts of uneven lengths.
        dict(name="attend, batch", op="attend", rows=48, block=16, heads=8, per=4, dim=128, ctx_lo=50, ctx_hi=8000, new_lo=8, new_hi=32, x="bf16"),
        # A few requests with large trees over long contexts: the work has to be split along the context.
        dict(name="attend, long contexts", op="attend", rows=3, block=32, heads=8, per=8, dim=128, ctx_lo=60001, ctx_hi=99991, new_lo=64, new_hi=64, x="bf16"),
        # One request's accepted tokens move up in one layer's cache: latency.
        dict(name="compact, 1 request", op="compact", rows=1, block=16, heads=2, dim=64, ctx_lo=700, ctx_hi=700, new_lo=6, new_hi=6, kept_lo=3, kept_hi=3),
        # The same for a batch with large trees.
        dict(name="compact, batch", op="compact", rows=256, block=16, heads=8, dim=128, ctx_lo=0, ctx_hi=4000, new_lo=24, new_hi=64, kept_lo=1, kept_hi=12),
        # One prompt, three more samples of it.
        dict(name="fork, 1 prompt", op="pages", call="fork", rows=1, times=3, block=16, heads=2, dim=64, ctx_lo=1001, ctx_hi=1001, spare=20),
        # Eight samples of each of 64 prompts.
        dict(name="fork, batch", op="pages", call="fork", rows=64, times=7, block=16, heads=8, dim=128, ctx_lo=50, ctx_hi=8000, spare=600),
        # A batch of samples that share their prompts: every third one stopped, the others give back rejected tokens' blocks.
        dict(name="release, shared prompts", op="pages", call="release", rows=64, times=7, block=16, ctx_lo=50, ctx_hi=8000, new_lo=1, new_hi=600, every=3, back=40),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "drafts", "attend", "attend", "attend", "compact", "pages", "pages"])
    x = rng.choice(["bf16", "f16"])
    if op == "rotate":
        heads, per, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8]), rng.choice([64, 80, 96, 128, 128, 256])
        most = 8192 * 40 * 128 // ((heads * per + heads) * dim * 2)  # f32 has twice the bytes
        return dict(op=op, tokens=min(_log(rng, 1, 16000), most), heads=heads, per=per, dim=dim, rot=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.7, fused=rng.random() < 0.5, far=rng.choice([4000, 131071, 1000003]), x=rng.choice([x, x, "f32"]))
    block = rng.choice([16, 32, 64, 128])
    if op == "drafts":
        return dict(op=op, rows=_log(rng, 1, 256), block=block, ctx_lo=0, ctx_hi=_log(rng, 1, 8000), new_lo=rng.choice([0, 1, 5]), new_hi=rng.choice([5, 8, 16, 31, 64]), stops=rng.random() < 0.5)
    heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256])
    if op == "attend":
        rows, per, most = _log(rng, 1, 64), rng.choice([1, 2, 3, 4, 7, 8, 16]), _log(rng, 2, 128)
        # the keys, and the products of the queries with them, stay below the largest listed cases'
        hi = min(_log(rng, 1, 100000), 3_000_000 * 16 // (rows * heads * dim // 8), 80_000_000_000 // (rows * heads * per * dim * most))
        return dict(op=op, rows=rows, block=block, heads=heads, per=per, dim=dim, ctx_lo=rng.choice([0, 1 + hi // 3]), ctx_hi=max(1, hi), new_lo=rng.choice([1, max(1, most // 2)]), new_hi=most, x=x)
    if op == "compact":
        rows, most = _log(rng, 1, 256), rng.choice([4, 8, 16, 31, 64])
        heads = min(heads, 1024 // dim)
        return dict(op=op, rows=rows, block=block, heads=heads, dim=dim, ctx_lo=0, ctx_hi=min(_log(rng, 1, 4000), 600_000 // rows), new_lo=rng.choice([1, 4]), new_hi=most, kept_lo=1, kept_hi=_log(rng, 1, most))
    rows, times = _log(rng, 1, 64), rng.choice([1, 2, 3, 7])
    hi = _log(rng, 1, 8000)
    if rng.random() < 0.5:
        rows = max(1, min(rows, 64 * 7 * 16 * 8 * 128 // (times * block * heads * dim)))
        return dict(op=op, call="fork", rows=rows, times=times, block=block, heads=heads, dim=dim, ctx_lo=1, ctx_hi=min(hi, 8000 * 64 * 16 // (rows * block)),
                    spare=1 + int(rows * times * rng.uniform(0.5, 1.3)))
    return dict(op=op, call="release", rows=rows, times=times, block=block, ctx_lo=1, ctx_hi=hi, new_lo=1, new_hi=_log(rng, 1, 600), every=rng.choice([1, 2, 3, 5]), back=rng.choice([1, 8, 40]))


# ------------------------------------------------------------------- sizes of a case (host)
def _spread(lo, hi, rows, salt):
    """`rows` whole numbers spread over [lo, hi], the same for every seed."""
    return [lo + ((b + 1) * 2654435761 * (2 * salt + 1) % (1 << 32)) * (hi - lo + 1) // (1 << 32) for b in range(rows)]


def _lengths(case):
    """(tokens in the cache before the step, new tokens) of each row."""
    return _spread(case["ctx_lo"], case["ctx_hi"], case["rows"], 1), _spread(case.get("new_lo", 0), case.get("new_hi", 0), case["rows"], 2)


def _kept(case):
    """Accepted tokens of each row: the first one, and others that all have to move."""
    return [max(1, min(kept, n - 1)) for kept, n in zip(_spread(case["kept_lo"], case["kept_hi"], case["rows"], 3), _lengths(case)[1])]


def _samples(case):
    """(prompt, tokens after it, prompt's tokens) of the samples of a release, whose rows share their prompts' full blocks."""
    n = case["rows"] * (case["times"] + 1)
    prompts = _spread(case["ctx_lo"], case["ctx_hi"], case["rows"], 1)
    return [b % case["rows"] for b in range(n)], _spread(case["new_lo"], case["new_hi"], n, 2), prompts


def _call(case):
    return case.get("call", case["op"])


def work(case):
    op = _call(case)
    if op == "rotate":
        values = case["tokens"] * (case["heads"] * case["per"] + case["heads"]) * case["dim"]
        return {"bytes": 2 * values * SIZE[case["x"]] + 4 * case["tokens"] + 2 * case["rot"] + (2 * case["dim"] * SIZE[case["x"]] if case["norm"] else 0),
                "flops": values * (6 if case["norm"] else 3)}
    ctx, new = _lengths(case)
    bs = case["block"]
    up = lambda v: -(-v // bs)  # noqa: E731
    if op == "drafts":
        # parents, tokens, sampled tokens and codes in; spans, positions, paths and tokens out; per row four numbers in and four out
        return {"bytes": sum(new) * (12 + 4 * case["stops"] + 8 + 4 + 8) + 28 * case["rows"], "flops": 0}
    if op == "attend":
        heads, dim, queries = case["heads"], case["dim"], case["per"] * case["heads"]
        # the branch that a token sees is not known here: one token for each, itself
        seen = sum(m * c + m for c, m in zip(ctx, new))
        kv = sum(c + m for c, m in zip(ctx, new))
        pages = sum(up(c + m) for c, m in zip(ctx, new))
        return {"bytes": 2 * heads * dim * kv + 8 * heads * pages + 4 * pages + 2 * queries * dim * sum(new) * SIZE[case["x"]], "flops": 4 * queries * dim * seen}
    if op == "compact":
        heads, dim, kept = case["heads"], case["dim"], _kept(case)
        pages = sum(up(c + k) - c // bs for c, k in zip(ctx, kept))
        return {"bytes": 4 * heads * dim * (sum(kept) - case["rows"]) + 16 * heads * pages + 4 * pages + 4 * sum(kept) + 16 * case["rows"], "flops": 0}
    if op == "fork":
        n = case["times"]
        full = sum(c // bs for c in ctx)
        part = min(sum(c % bs > 0 for c in ctx) * n, case["spare"])
        # table entries from row to row, a counter up for each; blocks that are not full, with their scales, and their ids
        return {"bytes": n * full * 16 + part * (4 * case["heads"] * (case["dim"] * bs + 4) + 20) + 20 * n * case["rows"], "flops": 0}
    who, tail, prompts = _samples(case)
    back = sum(up(prompts[p] // bs * bs + t) for b, (p, t) in enumerate(zip(who, tail)) if b % case["every"] == 0)
    own_back = sum(up(t) for b, t in enumerate(tail) if b % case["every"] == 0)
    return {"bytes": 20 * len(who) + 4 * back + 8 * (back - own_back) + 4 * own_back, "flops": 0}


# ---------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(lens, width, total, g, bs):
    """A block table of `total` shuffled blocks: each row holds the blocks of its length, -1 behind them; and the ids left over."""
    held = (lens.long() + bs - 1) // bs
    ids = torch.randperm(total, generator=g, device=DEV)
    first = held.cumsum(0) - held
    j = torch.arange(width, device=DEV)
    table = torch.where(j < held[:, None], ids[(first[:, None] + j).clamp(max=total - 1)], -1).int()
    return table, ids[int(held.sum()):].int()


def _cache(total, heads, bs, dim, g):
    """Keys and values in 8 bits with a power of two per block and head."""
    cache = {}
    for name in ("k", "v"):
        values = torch.empty(total, heads, bs, dim, dtype=torch.float8_e4m3fn, device=DEV)
        for at in range(0, total, 4096):  # in pieces: a large cache does not fit many times over
            part = values[at: at + 4096]
            part.copy_((torch.randn(part.shape, generator=g, device=DEV) * 100).clamp(-448, 448))
        cache[name] = values
        cache[name + "_scale"] = torch.exp2(torch.randint(-9, -5, (total, heads), generator=g, device=DEV).float())
    return cache


def _step(case, g):
    """A step's numbers: rows of `ctx` tokens that got `new` more, laid out row after row; the tree of each row's new tokens."""
    ctx, new = _lengths(case)
    rows, granted = case["rows"], _ints(new)
    starts = torch.zeros(rows + 1, dtype=torch.int32, device=DEV)
    starts[1:] = granted.cumsum(0)
    s = dict(case=case, lens=_ints([c + m for c, m in zip(ctx, new)]), granted=granted, starts=starts, tokens=sum(new), most=max(1, max(new)))
    # Trees as drafters make them: half of the tokens go on from the one before, the others branch off anywhere.
    i = torch.arange(s["tokens"], device=DEV)
    row = torch.searchsorted(starts[1:].long(), i, right=True)
    local = i - starts.long()[row]
    u = torch.rand(s["tokens"], generator=g, device=DEV)
    other = (torch.rand(s["tokens"], generator=g, device=DEV, dtype=torch.float64) * local).long().clamp(min=0)
    parent = torch.where(u < 0.5, local - 1, torch.minimum(other, local - 1))
    s["parents"] = torch.where(local == 0, -1, parent).int()
    s["row"], s["local"] = row, local
    return s


def prepare(case, seed):
    g = _gen(seed)
    op = _call(case)
    if op == "rotate":
        t, heads, queries, dim, dt = case["tokens"], case["heads"], case["heads"] * case["per"], case["dim"], DTYPES[case["x"]]
        x = torch.randn(t, (queries + 2 * heads) * dim, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(t, 1, generator=g, device=DEV))
        x = x.to(dt)
        q, k = x[:, : queries * dim].unflatten(1, (queries, dim)), x[:, queries * dim: (queries + heads) * dim].unflatten(1, (heads, dim))
        if not case["fused"]:
            q, k = q.contiguous(), k.contiguous()
        weight = lambda: (1 + 0.2 * torch.randn(dim, generator=g, device=DEV)).to(dt) if case["norm"] else None  # noqa: E731
        freqs = (10000.0 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])).float()
        return dict(case=case, q=q, k=k, freqs=freqs, q_weight=weight(), k_weight=weight(), positions=torch.randint(0, case["far"] + 1, (t,), generator=g, device=DEV).int())
    bs = case["block"]
    if op in ("drafts", "attend", "compact"):
        s = _step(case, g)
        if op == "drafts":
            # Where a token has children, the sampled token is mostly that of one of them.
            n, rows = s["tokens"], case["rows"]
            tokens = torch.randint(0, 151936, (n,), generator=g, device=DEV)
            targets = torch.randint(0, 151936, (n,), generator=g, device=DEV)
            start = s["starts"].long()[s["row"]]
            up = torch.where(s["parents"] >= 0, start + s["parents"], n)
            child = torch.full((n + 1,), -1, device=DEV).scatter_reduce(0, up, torch.arange(n, device=DEV), "amax")[:n]
            agrees = (child >= 0) & (torch.rand(n, generator=g, device=DEV) < 0.8)
            targets = torch.where(agrees, tokens[child.clamp(min=0)] if n else targets, targets)
            codes = torch.where(torch.rand(n, generator=g, device=DEV) < 0.02, 1, 0).int() if case["stops"] else None
            # The first tokens of a few rows are given: the end of a prompt in front of the drafts.
            given = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.1, 2, 1).int()
            s.update(draft=tokens.int(), targets=targets.int(), codes=codes, given=given)
            return s
        heads, dim = case["heads"], case["dim"]
        total = sum(-(-(c + m) // bs) for c, m in zip(*_lengths(case))) + 5
        s["table"], _ = _pages(s["lens"], -(-int(s["lens"].max()) // bs), total, g, bs)
        s.update(_cache(total, heads, bs, dim, g))
        if op == "attend":
            span, positions = _plain_tree(s)  # what plan_tree gives, once per step: every layer's attention reads it
            q = torch.randn(s["tokens"], heads * case["per"], dim, generator=g, device=DEV).to(DTYPES[case["x"]])
            s.update(span=span, positions=positions, q=q, scale=1.0 / math.sqrt(dim))
            return s
        # The accepted tokens of each row: the first one and some of those behind the second, in order.
        kept = _ints(_kept(case)).long()
        order = torch.rand(case["rows"], s["most"], generator=g, device=DEV)
        j = torch.arange(s["most"], device=DEV)
        order = torch.where((j < 2) | (j >= s["granted"][:, None]), 2.0, order)
        rank = order.argsort(1).argsort(1)
        take = (j == 0) | ((rank < (kept - 1)[:, None]) & (order < 2.0))
        at = take.cumsum(1) - 1
        path = torch.full((case["rows"], s["most"] + 1), -1, device=DEV).scatter(1, torch.where(take, at, s["most"]), j.expand_as(take))[:, :-1]
        s["path"] = path[s["row"], s["local"]].int()
        s["counts"] = take.sum(1).int()
        s["kept_lens"] = (s["lens"] - s["granted"] + s["counts"]).int()
        return s
    if op == "fork":
        # rows [0, rows) hold prompts, the others are idle; each prompt is forked `times` times
        rows, n = case["rows"], case["rows"] * case["times"]
        ctx = _lengths(case)[0]
        lens = _ints(ctx + [0] * n)
        total = sum(-(-c // bs) for c in ctx) + case["spare"]
        width = -(-max(ctx) // bs) + 2
        table, free = _pages(lens, width, total, g, bs)
        pool = torch.zeros(total, dtype=torch.int32, device=DEV)
        pool[: free.numel()] = free
        i = torch.arange(n, device=DEV)
        return dict(case=case, table=table, lens=lens, free=pool, n_free=_ints([free.numel()]), shares=torch.zeros(total, dtype=torch.int32, device=DEV),
                    src=(i % rows).int(), dst=(rows + i).int(), **_cache(total, case["heads"], bs, case["dim"], g))
    # release: samples of shared prompts, each with blocks of its own behind the shared ones
    who, tail, prompts = _samples(case)
    n = len(who)
    shared = [p // bs for p in prompts]
    lens = [shared[p] * bs + t for p, t in zip(who, tail)]
    own_blocks = [-(-ln // bs) - shared[p] for p, ln in zip(who, lens)]
    total = sum(shared) + sum(own_blocks) + 50
    width = -(-max(lens) // bs) + 1
    ids = torch.randperm(total, generator=g, device=DEV).int()
    first_shared = _ints([0] + shared).long().cumsum(0)
    first_own = _ints([sum(shared)] + own_blocks).long().cumsum(0)
    p, j = _ints(who).long(), torch.arange(width, device=DEV)
    sh, b = _ints(shared).long()[p][:, None], torch.arange(n, device=DEV)
    at = torch.where(j < sh, first_shared[p][:, None] + j, first_own[b][:, None] + j - sh)
    held = ((_ints(lens) + bs - 1) // bs)[:, None]
    table = torch.where(j < held, ids[at.clamp(max=total - 1)], -1).int()
    used = sum(shared) + sum(own_blocks)
    shares = torch.zeros(total, dtype=torch.int32, device=DEV)
    shares[ids[: sum(shared)].long()] = case["times"]
    free = torch.zeros(total, dtype=torch.int32, device=DEV)
    free[: total - used] = ids[used:]
    codes = (b % case["every"] == 0).int() * torch.randint(1, 3, (n,), generator=g, device=DEV).int()
    keep = (_ints(lens) - torch.randint(0, case["back"] + 1, (n,), generator=g, device=DEV).int()).clamp(min=0)
    keep = torch.maximum(keep, (sh[:, 0] * bs).int())
    return dict(case=case, table=table, lens=_ints(lens), codes=codes, keep=keep, shares=shares, free=free, n_free=_ints([total - used]))


# -------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    return {"rotate": _plain_rotate, "drafts": _plain_drafts, "attend": _plain_attend, "compact": _plain_compact, "fork": _plain_fork, "release": _plain_release}[_call(s["case"])](s)


def _run_own(s):
    import localstrm_b200 as lb
    case = s["case"]
    op = _call(case)
    if op == "rotate":
        return lb.norm_rotate(s["q"], s["k"], s["positions"], s["freqs"], q_weight=s["q_weight"], k_weight=s["k_weight"], interleaved=case["interleaved"])
    if op == "fork":
        f = lb.fork_blocks(s["table"], s["lens"], s["src"], s["dst"], s["shares"], s["free"], s["n_free"], case["block"])
        lb.copy_blocks(lb.KVCache8(s["k"], s["v"], s["k_scale"], s["v_scale"]), f.copies)
        return f.lens, f.n_free, f.granted, f.copies, s["table"], s["shares"], s["k"], s["v"], s["k_scale"], s["v_scale"]
    if op == "release":
        lens, n_free = lb.release_blocks(s["table"], s["lens"], s["codes"], s["free"], s["n_free"], case["block"], keep=s["keep"], shares=s["shares"])
        return lens, n_free, s["free"], s["shares"]
    plan = lb.StepPlan(starts=s["starts"], granted=s["granted"], lens=s["lens"])
    if op == "drafts":
        tree = lb.plan_tree(plan, s["parents"])
        a = lb.accept_drafts(plan, tree, s["draft"], s["targets"], codes=s["codes"], given=s["given"])
        return tree.span, tree.positions, a.path, a.tokens, a.counts, a.lens, a.last, a.codes
    cache = lb.KVCache8(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if op == "attend":
        return lb.attend(s["q"], cache, s["table"], plan, scale=s["scale"], tree=lb.TreePlan(s["span"], s["positions"], s["parents"]))
    lb.compact_kv(cache, s["table"], plan, s["path"], s["counts"])
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _plain_rotate(s):
    case = s["case"]
    half = case["rot"] // 2
    angle = s["positions"].double()[:, None, None] * s["freqs"].double()
    cos, sin = angle.cos().float(), angle.sin().float()

    def one(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
        a, b = (x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]) if case["interleaved"] else (x[..., :half], x[..., half: 2 * half])
        c, d = a * cos - b * sin, b * cos + a * sin
        turned = torch.stack([c, d], -1).flatten(-2) if case["interleaved"] else torch.cat([c, d], -1)
        return torch.cat([turned, x[..., 2 * half:]], -1).to(s["q"].dtype)
    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


def _family(s):
    """(parent, real, up) of the rows' new tokens, padded to the most that a row has: up[b, i, j] is 1 where j is i or an ancestor of it."""
    i = torch.arange(s["most"], device=DEV)
    real = i < s["granted"][:, None]
    at = (s["starts"].long()[:-1, None] + i).clamp(max=max(0, s["tokens"] - 1))
    parent = torch.where(real, s["parents"].long()[at], -1)
    parent = torch.where((parent >= 0) & (parent < i), parent, -1)
    up = ((parent[..., None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, (s["most"] - 1).bit_length())):
        up = (up @ up > 0).float()
    return parent, real, up


def _flat(s, x, none):
    """One value per token of the step from the padded ones."""
    return x[s["row"], s["local"]].int() if s["tokens"] else torch.full((0,), none, dtype=torch.int32, device=DEV)


def _plain_tree(s):
    """(span, positions): a token's place in its tree's pre-order and the number of tokens of its branch; its position."""
    parent, real, up = _family(s)
    size = (up * real[..., None]).sum(1)
    i = torch.arange(s["most"], device=DEV)
    earlier = ((parent[..., None] == parent[:, None]) & (i < i[:, None]) & real[..., None] & real[:, None]).float()
    depth = up.sum(-1) - 1
    order = depth + (up @ (earlier @ size[..., None]))[..., 0]
    positions = (s["lens"] - s["granted"])[:, None] + depth
    return torch.stack([_flat(s, order, 0), _flat(s, size, 0)], -1), _flat(s, positions, 0)


def _plain_drafts(s):
    span, positions = _plain_tree(s)
    parent, real, up = _family(s)
    rows, most = parent.shape
    i = torch.arange(most, device=DEV)
    at = (s["starts"].long()[:-1, None] + i).clamp(max=max(0, s["tokens"] - 1))
    draft, target = s["draft"].long()[at], s["targets"].long()[at]
    code = s["codes"][at] if s["codes"] is not None else torch.zeros_like(parent)
    given = torch.minimum(s["given"], s["granted"])[:, None].long().clamp(min=1)
    p = parent.clamp(min=0)
    good = (parent >= given - 1) & (draft == target.gather(1, p)) & (code.gather(1, p) == 0)
    first = (good[:, None] & (parent[..., None] == parent[:, None]) & (i < i[:, None])).any(-1)
    good = real & ((i < given) | (good & ~first))
    taken = good & ((up * (~good)[:, None]).sum(-1) == 0)
    counts = taken.sum(1)
    path = torch.full((rows, most + 1), -1, device=DEV).scatter(1, torch.where(taken, taken.cumsum(1) - 1, most), i.expand_as(taken))[:, :-1]
    said = torch.where(path >= 0, target.gather(1, path.clamp(min=0)), -1)
    shift = i + given - 1
    said = torch.where(shift < most, said.gather(1, shift.clamp(max=most - 1)), -1)
    end = path.gather(1, (counts - 1).clamp(min=0)[:, None])
    last = torch.where(counts > 0, target.gather(1, end.clamp(min=0))[:, 0], -1)
    stop = torch.where(counts > 0, code.gather(1, end.clamp(min=0))[:, 0], 0)
    lens = s["lens"] - s["granted"] + counts
    return span, positions, _flat(s, path, -1), _flat(s, said, -1), counts.int(), lens.int(), last.int(), stop.int()


def _plain_attend(s):
    case = s["case"]
    heads, per, dim, bs = case["heads"], case["per"], case["dim"], case["block"]
    lens, granted, starts, table = s["lens"].long(), s["granted"].long(), s["starts"].long(), s["table"].long().clamp(min=0)
    rows, width = table.shape
    keys, most = width * bs, s["most"]

    def gather(name):
        x = s[name].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * s[name + "_scale"][table][..., None, None]
        return x.transpose(1, 2).reshape(rows, heads, keys, dim)

    i = torch.arange(most, device=DEV)
    at = (starts[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[at]  # [rows, queries, heads * per, dim]
    q = q.view(rows, most, heads, per, dim).permute(0, 2, 3, 1, 4).reshape(rows, heads, per * most, dim)
    scores = (q @ gather("k").transpose(2, 3)).view(rows, heads, per, most, keys) * s["scale"]
    # the context, and of the new tokens those whose branch the query lies in
    order, size = s["span"].long()[..., 0], s["span"].long()[..., 1]
    t = torch.arange(keys, device=DEV)
    j = t - (lens - granted)[:, None]
    tok = (starts[:-1, None] + j).clamp(0, s["tokens"] - 1)
    below = order[at][..., None] - order[tok][:, None]
    seen = (t < lens[:, None])[:, None] & ((j < 0)[:, None] | ((below >= 0) & (below < size[tok][:, None])))
    seen = seen | (i >= granted[:, None])[..., None]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(scores.sub_(scores.amax(-1, keepdim=True)))
    total = p.sum(-1, keepdim=True)
    v = torch.where((t < lens[:, None])[:, None, :, None], gather("v"), 0.0)
    o = (p.view(rows, heads, per * most, keys) @ v).view(rows, heads, per, most, dim) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(rows, most, heads * per, dim)
    return o[s["row"], s["local"]].to(s["q"].dtype)


def _plain_compact(s):
    bs = s["case"]["block"]
    starts, table = s["starts"].long()[:-1], s["table"].long()
    old, now = (s["lens"] - s["granted"]).long(), (s["lens"] - s["granted"] + s["counts"]).long()
    steps = torch.arange((s["most"] + bs - 2) // bs + 1, device=DEV)
    at = torch.minimum((old // bs)[:, None] + steps, ((now - 1) // bs)[:, None])  # the blocks that a row's accepted tokens go to; the last one again behind them
    page = table.gather(1, at)
    pos = at[..., None] * bs + torch.arange(bs, device=DEV)
    real = pos < now[:, None, None]
    i = pos - old[:, None, None]
    tok = (starts[:, None, None] + i).clamp(0, s["tokens"] - 1)
    source = torch.where((i >= 0) & real, old[:, None, None] + s["path"].long()[tok], pos)
    source_page = table.gather(1, (source // bs).flatten(1)).view_as(source)
    heads = torch.arange(s["case"]["heads"], device=DEV)[:, None]
    for name in ("k", "v"):
        codes, scale = s[name].view(torch.uint8), s[name + "_scale"]
        was = codes[source_page[:, :, None], heads, (source % bs)[:, :, None]]  # [rows, blocks, heads, tokens, dim]
        its = scale[source_page].transpose(2, 3)
        most = torch.where(real[:, :, None], its, 0.0).amax(-1)
        ratio = its / most[..., None]
        moved = (was.view(torch.float8_e4m3fn).float() * ratio[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        codes[page] = torch.where(real[:, :, None, :, None], moved, was)
        scale[page] = most
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _plain_fork(s):
    bs, table, free, lens = s["case"]["block"], s["table"].long(), s["free"].long(), s["lens"].long()
    src, dst, n_free = s["src"].long(), s["dst"].long(), s["n_free"].long()
    t = lens[src]
    full, need = t // bs, (t % bs > 0).long()
    taken = need.cumsum(0)
    ok = (need == 0) | (taken <= n_free)
    granted = torch.where(ok, t, 0)
    after = n_free - (need * ok).sum()
    fresh = free[(n_free - taken).clamp(0, free.numel() - 1)]
    j = torch.arange(table.shape[1], device=DEV)
    shared = ok[:, None] & (j < full[:, None])
    mine = ok[:, None] & (need > 0)[:, None] & (j == full[:, None])
    rows = torch.where(shared, table[src], torch.where(mine, fresh[:, None], table[dst]))
    s["shares"].index_add_(0, table[src].clamp(min=0).flatten(), shared.flatten().int())
    part = table[src].gather(1, full[:, None].clamp(max=table.shape[1] - 1))[:, 0]
    copy = ok & (need > 0)
    copies = torch.where(copy[:, None], torch.stack([part, fresh], -1), -1)
    s["table"][dst] = rows.int()
    # a row without a copy writes a block of its source over itself
    a = table[src].gather(1, ((t - 1) // bs)[:, None])[:, 0]
    b = torch.where(copy, fresh, a)
    for name in ("k", "v"):
        codes = s[name].view(torch.uint8)
        codes[b] = codes[a]
        s[name + "_scale"][b] = s[name + "_scale"][a]
    out = lens.index_copy(0, dst, torch.where(ok, t, lens[dst]))
    return out.int(), after.int(), granted.int(), copies.int(), s["table"], s["shares"], s["k"], s["v"], s["k_scale"], s["v_scale"]


def _plain_release(s):
    bs, table, free, n_free, shares = s["case"]["block"], s["table"].long(), s["free"].long(), s["n_free"].long(), s["shares"].long()
    rows, width = table.shape
    lens = s["lens"].long()
    now = torch.where(s["codes"] != 0, 0, torch.minimum(s["keep"].long().clamp(min=0), lens))
    j = torch.arange(width, device=DEV)
    given = ((j >= ((now + bs - 1) // bs)[:, None]) & (j < ((lens + bs - 1) // bs)[:, None])).flatten()
    ids = torch.where(given, table.flatten(), free.numel())  # one more counter for those that stay
    times = torch.zeros(free.numel() + 1, dtype=torch.int64, device=DEV).scatter_add(0, ids, torch.ones_like(ids))[:-1]
    at = torch.arange(rows * width, device=DEV)
    last = torch.full((free.numel() + 1,), -1, device=DEV).scatter_reduce(0, ids, at, "amax")[:-1]
    goes = times > shares
    left = (shares - times).clamp(min=0)
    safe = ids.clamp(max=free.numel() - 1)
    out = given & goes[safe] & (last[safe] == at)
    place = n_free + out.cumsum(0) - 1
    pool = torch.cat([free, free[:1]]).scatter(0, torch.where(out, place, free.numel()).clamp(max=free.numel()), ids)[:-1]
    s["free"].copy_(pool)
    s["shares"].copy_(left)
    return now.int(), (n_free + out.sum()).clamp(max=free.numel()).int(), s["free"], s["shares"]


# --------------------------------------------------------------------- definitions, 64 bits
def exact(case, seed):
    if _call(case) in ("drafts", "release"):
        return None  # whole numbers: they are compared as they are
    s = prepare(case, seed)
    if _call(case) == "fork":  # one after the other, each block that is not full copied to the free list's next
        table, lens, free, n_free = (s[n].tolist() for n in ("table", "lens", "free", "n_free"))
        out = [s[n].double() for n in ("k", "v", "k_scale", "v_scale")]
        left = n_free[0]
        for a in s["src"].tolist():
            if lens[a] % case["block"]:
                left -= 1
                if left >= 0:
                    for x in out:
                        x[free[left]] = x[table[a][lens[a] // case["block"]]]
        return (None,) * 6 + tuple(out)
    if case["op"] == "rotate":
        out = []
        half = case["rot"] // 2
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            y = x.double()
            if w is not None:
                y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6) * w.double()
            z = y.clone()
            for i in range(half):
                m, n = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
                a = (s["positions"].double() * s["freqs"][i].double())[:, None]
                z[..., m] = y[..., m] * torch.cos(a) - y[..., n] * torch.sin(a)
                z[..., n] = y[..., m] * torch.sin(a) + y[..., n] * torch.cos(a)
            out.append(z)
        return tuple(out)
    lens, granted, starts, table = (s[n].tolist() for n in ("lens", "granted", "starts", "table"))
    bs = case["block"]
    if case["op"] == "compact":
        path, counts = s["path"].tolist(), s["counts"].tolist()
        out = []
        for name in ("k", "v"):
            codes, scale = s[name].double(), s[name + "_scale"].double()
            for b in range(case["rows"]):
                old, now = lens[b] - granted[b], lens[b] - granted[b] + counts[b]
                for block in range(old // bs, (now - 1) // bs + 1):
                    page, lo, hi = table[b][block], max(old, block * bs), min(now, (block + 1) * bs)
                    come = [old + path[starts[b] + p - old] for p in range(lo, hi)]
                    rows = [(table[b][c // bs], c % bs) for c in come]
                    x = torch.stack([codes[p, :, o] * scale[p][:, None] for p, o in rows], 1)
                    top = torch.stack([scale[p] for p, _ in rows]).amax(0)
                    if lo > block * bs:
                        top = torch.maximum(top, scale[page])
                        codes[page, :, : lo - block * bs] = _to_e4m3(codes[page, :, : lo - block * bs] * (scale[page] / top)[:, None, None])
                    codes[page, :, lo - block * bs: hi - block * bs] = _to_e4m3(x / top[:, None, None])
                    scale[page] = top
            out.append((codes, scale))
        return out[0][0], out[1][0], out[0][1], out[1][1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    per, parents = case["per"], s["parents"].tolist()
    for b in range(case["rows"]):
        n, ctx = granted[b], lens[b] - granted[b]
        pages = torch.tensor(table[b][: -(-lens[b] // bs)], device=DEV)
        hidden = [[True] * n for _ in range(n)]
        for i in range(n):
            j = i
            while j >= 0:
                hidden[i][j] = False
                j = parents[starts[b] + j]
        mask = torch.zeros(n, lens[b], dtype=torch.bool, device=DEV)
        mask[:, ctx:] = torch.tensor(hidden, device=DEV)
        for h in range(case["heads"]):
            k, v = ((s[m][pages, h].double() * s[m + "_scale"][pages, h].double()[:, None, None]).reshape(-1, case["dim"])[: lens[b]] for m in ("k", "v"))
            for r in range(h * per, (h + 1) * per):
                z = (s["q"][starts[b]: starts[b + 1], r].double() @ k.t() * s["scale"]).masked_fill(mask, -math.inf)
                out[starts[b]: starts[b + 1], r] = torch.softmax(z, -1) @ v
    return out


def _to_e4m3(x):
    """x rounded to the nearest value of 4 exponent and 3 mantissa bits, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (x / step).round() * step
