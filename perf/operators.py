"""The decode-step operators around the sampler, as cases that can be timed and compared.

``listed()`` and ``draw()`` give cases (dicts of plain values), ``prepare()`` makes the inputs of
one, and ``run()`` is one pass: in plain torch operations where ``own`` is false, through
``localstrm_b200`` where it is true.  ``exact()`` is the same result from the definition in
64 bits, and ``work()`` the bytes and operations that a pass cannot do without.

Operators (``case["op"]``):

* ``int4``     ``y = x W^T`` for few rows ``x [rows, K]``; ``W[n, k] = (code[n, k] - 8) * scale[n, k / group]``
* ``plan``     block tables and slot maps of one step from the requests' lengths
* ``release``  the way back: the blocks of stopped requests return to the free list
* ``append``   new keys and values into a paged cache of 8-bit values, one scale per block and head
* ``attend``   softmax attention of the step's queries over that cache
"""
import math

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # One request's next token: the 4-bit vocabulary projection of one hidden state (the
        # sampler's vocabulary of 151,936), logits in f32 as the sampler takes them.
        dict(name="int4 head, 1 row", op="int4", rows=1, n=151936, k=4096, group=128, x="bf16", y="f32"),
        # A layer's projection of one token, ragged sizes: the smallest product, latency counts.
        dict(name="int4 projection, 3 rows", op="int4", rows=3, n=2057, k=896, group=64, x="f16", y="f16"),
        # The vocabulary projection of a decode batch (the 128,256-token vocabulary).
        dict(name="int4 head, 64 rows", op="int4", rows=64, n=128256, k=4096, group=128, x="bf16", y="f32"),
        # A decode step of 256 running requests: one token each, few need a new block.
        dict(name="plan, decode step", op="plan", rows=256, block=16, ctx_lo=1, ctx_hi=8192, new_lo=1, new_hi=1, width=516, spare=64),
        # A step that mixes prompts and decoding rows; the free list runs out before the last rows.
        dict(name="plan, prompts", op="plan", rows=1000, block=32, ctx_lo=0, ctx_hi=4000, new_lo=0, new_hi=131, width=130, spare=1500),
        # Requests that stopped in a full batch give their blocks back.
        dict(name="release, stopped rows", op="release", rows=512, block=16, ctx_lo=0, ctx_hi=16384, every=3, width=1024),
        # A decode step's keys and values, one token per request, most blocks half full.
        dict(name="append, decode step", op="append", rows=256, block=16, heads=8, dim=128, ctx_lo=0, ctx_hi=4000, new_lo=1, new_hi=1, x="bf16"),
        # Prompt chunks of uneven lengths on top of what the cache holds.
        dict(name="append, prompts", op="append", rows=24, block=32, heads=8, dim=128, ctx_lo=0, ctx_hi=999, new_lo=1, new_hi=2048, x="f16"),
        # One request alone, a short context, 14 query heads on 2 key heads: latency.
        dict(name="attend, 1 short request", op="attend", rows=1, block=16, heads=2, per=7, dim=64, ctx_lo=700, ctx_hi=700, new_lo=1, new_hi=1, x="f16"),
        # A decode batch over contexts of uneven lengths.
        dict(name="attend, decode batch", op="attend", rows=64, block=16, heads=8, per=4, dim=128, ctx_lo=50, ctx_hi=16000, new_lo=1, new_hi=1, x="bf16"),
        # A few requests over long contexts: the work has to be split along the context.
        dict(name="attend, long contexts", op="attend", rows=3, block=32, heads=8, per=8, dim=128, ctx_lo=90001, ctx_hi=131071, new_lo=1, new_hi=1, x="bf16"),
        # Prompt chunks against a cache that already holds a context (causal inside the chunk).
        dict(name="attend, prompt chunks", op="attend", rows=4, block=16, heads=8, per=4, dim=128, ctx_lo=1000, ctx_hi=6000, new_lo=256, new_hi=700, x="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["int4", "int4", "plan", "release", "append", "append", "attend", "attend", "attend"])
    if op == "int4":
        group = rng.choice([32, 64, 128])
        rows, k = _log(rng, 1, 64), group * max(1, _log(rng, 256, 8192) // group)
        n = min(_log(rng, 200, 150000), 128256 * 4096 // k)
        x = rng.choice(["bf16", "f16", "f32"])
        return dict(op=op, rows=rows, n=n, k=k, group=group, x=x, y=rng.choice([x, "f32"]))
    block = rng.choice([16, 32, 64, 128])
    if op == "plan":
        rows, hi = _log(rng, 1, 4000), _log(rng, 1, 8000)
        most = max(1, min(_log(rng, 1, 2000), 260000 // rows))
        width = -(-(hi + most) // block) + rng.choice([-1, 0, 3])
        return dict(op=op, rows=rows, block=block, ctx_lo=0, ctx_hi=hi, new_lo=rng.choice([0, 1]), new_hi=most, width=max(1, width),
                    spare=1 + int(rows * (1 + most / block) * rng.uniform(0.2, 1.2)))
    if op == "release":
        hi = _log(rng, 1, 16000)
        return dict(op=op, rows=_log(rng, 1, 2000), block=block, ctx_lo=0, ctx_hi=hi, every=rng.choice([1, 2, 3, 7]), width=-(-hi // block) + rng.choice([0, 5]))
    heads, dim, x = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256]), rng.choice(["bf16", "f16"])
    if op == "append":
        rows = _log(rng, 1, 400)
        return dict(op=op, rows=rows, block=block, heads=heads, dim=dim, ctx_lo=0, ctx_hi=_log(rng, 1, 2000), new_lo=1,
                    new_hi=rng.choice([1, max(1, min(_log(rng, 1, 2000), 24000 // rows))]), x=x)
    rows, per = _log(rng, 1, 64), rng.choice([1, 2, 3, 4, 7, 8, 16])
    most = rng.choice([1, 1, 1, _log(rng, 1, 128)])
    # the keys, and the products of the queries with them, stay below the largest listed cases'
    hi = min(_log(rng, 1, 100000), 4_000_000 * 16 // (rows * heads * dim // 8), 2_000_000_000 // (rows * heads * per * dim * most))
    return dict(op=op, rows=rows, block=block, heads=heads, per=per, dim=dim, ctx_lo=rng.choice([0, 1 + hi // 3]), ctx_hi=max(1, hi), new_lo=1, new_hi=most, x=x)


# ------------------------------------------------------------------- sizes of a case (host)
def _spread(lo, hi, rows, salt):
    """`rows` whole numbers spread over [lo, hi], the same for every seed."""
    return [lo + ((b + 1) * 2654435761 * (2 * salt + 1) % (1 << 32)) * (hi - lo + 1) // (1 << 32) for b in range(rows)]


def _lengths(case):
    """(tokens in the cache before the step, new tokens) of each row."""
    return _spread(case["ctx_lo"], case["ctx_hi"], case["rows"], 1), _spread(case.get("new_lo", 0), case.get("new_hi", 0), case["rows"], 2)


def work(case):
    if case["op"] == "int4":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * k // 2 + 2 * n * (k // case["group"]) + rows * (k * SIZE[case["x"]] + n * SIZE[case["y"]]), "flops": 2 * rows * n * k}
    ctx, new = _lengths(case)
    bs = case["block"]
    up = lambda v: -(-v // bs)  # noqa: E731
    if case["op"] == "plan":
        taken = sum(up(c + m) - up(c) for c, m in zip(ctx, new))
        # lengths in and out, starts, granted; slots and positions; new blocks out of the list into the table
        return {"bytes": 20 * case["rows"] + 12 * sum(new) + 8 * min(taken, case["spare"]) + 4 * case["rows"], "flops": 0}
    if case["op"] == "release":
        back = sum(up(c) for b, c in enumerate(ctx) if b % case["every"] == 0)
        return {"bytes": 12 * case["rows"] + 8 * back, "flops": 0}
    heads, dim = case["heads"], case["dim"]
    if case["op"] == "append":
        pages = sum((c + m - 1) // bs - c // bs + 1 for c, m in zip(ctx, new))
        old = sum(c % bs for c in ctx)  # kept values of half full blocks: read where their scale grows
        return {"bytes": 2 * heads * dim * (sum(new) * (SIZE[case["x"]] + 1) + old) + 16 * heads * pages + 4 * pages, "flops": 4 * heads * dim * sum(new)}
    queries = case["per"] * heads
    seen = sum(m * c + m * (m + 1) // 2 for c, m in zip(ctx, new))
    kv = sum(c + m for c, m in zip(ctx, new))
    pages = sum(up(c + m) for c, m in zip(ctx, new))
    return {"bytes": 2 * heads * dim * kv + 8 * heads * pages + 4 * pages + 2 * queries * dim * sum(new) * SIZE[case["x"]], "flops": 4 * queries * dim * seen}


# ---------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(lens, width, total, g, bs):
    """A block table of `total` shuffled blocks: each row holds the blocks of its length, -1 behind them; and the ids left over."""
    held = (lens.long().clamp(max=width * bs) + bs - 1) // bs
    ids = torch.randperm(total, generator=g, device=DEV)
    first = held.cumsum(0) - held
    j = torch.arange(width, device=DEV)
    table = torch.where(j < held[:, None], ids[(first[:, None] + j).clamp(max=total - 1)], -1).int()
    return table, ids, int(held.sum())


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "int4":
        rows, n, k, group = case["rows"], case["n"], case["k"], case["group"]
        packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=g, device=DEV)
        scales = (0.01 * torch.exp(0.5 * torch.randn(n, k // group, generator=g, device=DEV))).half()
        x = torch.randn(rows, k, generator=g, device=DEV)
        x *= torch.where(torch.rand(k, generator=g, device=DEV) < 0.004, 30.0, 1.0)  # a hidden state's few large channels
        return dict(case=case, packed=packed, scales=scales, x=x.to(DTYPES[case["x"]]))
    ctx, new = _lengths(case)
    bs, rows = case["block"], case["rows"]
    if case["op"] in ("plan", "release"):
        width = case["width"]
        lens = _ints(ctx)
        held = sum(min(-(-c // bs), width) for c in ctx)
        total = held + case.get("spare", 100)
        table, ids, held = _pages(lens, width, total, g, bs)
        free = torch.zeros(total, dtype=torch.int32, device=DEV)
        free[: total - held] = ids[held:].int()
        s = dict(case=case, table=table, lens=lens, free=free, n_free=_ints([total - held]))
        if case["op"] == "plan":
            s.update(new=_ints(new), capacity=sum(new) + 7)
        else:
            s.update(codes=(torch.arange(rows, device=DEV) % case["every"] == 0).int() * torch.randint(1, 3, (rows,), generator=g, device=DEV).int())
        return s
    heads, dim = case["heads"], case["dim"]
    lens = _ints([c + m for c, m in zip(ctx, new)])
    granted = _ints(new)
    width = -(-(max(c + m for c, m in zip(ctx, new))) // bs)
    total = sum(-(-(c + m) // bs) for c, m in zip(ctx, new)) + 5
    table, _, _ = _pages(lens, width, total, g, bs)
    starts = torch.zeros(rows + 1, dtype=torch.int32, device=DEV)
    starts[1:] = granted.cumsum(0)
    cache = {}
    for name in ("k", "v"):
        values = torch.empty(total, heads, bs, dim, dtype=torch.float8_e4m3fn, device=DEV)
        for at in range(0, total, 4096):  # in pieces: a large cache does not fit many times over
            part = values[at: at + 4096]
            part.copy_((torch.randn(part.shape, generator=g, device=DEV) * 100).clamp(-E4M3_MAX, E4M3_MAX))
        cache[name] = values
        cache[name + "_scale"] = torch.exp2(torch.randint(-9, -5, (total, heads), generator=g, device=DEV).float())
    s = dict(case=case, table=table, lens=lens, granted=granted, starts=starts, tokens=sum(new), most=max(new), **cache)
    t = DTYPES[case["x"]]
    if case["op"] == "append":
        spread = torch.exp(0.7 * torch.randn(sum(new), heads, 1, generator=g, device=DEV))  # some tokens make a block's scale grow
        s.update(new_k=(torch.randn(sum(new), heads, dim, generator=g, device=DEV) * spread).to(t), new_v=(torch.randn(sum(new), heads, dim, generator=g, device=DEV) * spread).to(t))
    else:
        s.update(q=torch.randn(sum(new), heads * case["per"], dim, generator=g, device=DEV).to(t), scale=1.0 / math.sqrt(dim))
    return s


# -------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    return {"int4": _plain_int4, "plan": _plain_plan, "release": _plain_release, "append": _plain_append, "attend": _plain_attend}[s["case"]["op"]](s)


def _run_own(s):
    import localstrm_b200 as lb
    op = s["case"]["op"]
    if op == "int4":
        return lb.int4_matvec(s["x"], lb.Int4Weight(s["packed"], s["scales"]), out_dtype=DTYPES[s["case"]["y"]])
    if op == "plan":
        p = lb.plan_blocks(s["table"], s["lens"], s["new"], s["free"], s["n_free"], s["case"]["block"], s["capacity"])
        return p.slots, p.positions, p.starts, p.granted, p.lens, p.n_free, s["table"]
    if op == "release":
        lens, n_free = lb.release_blocks(s["table"], s["lens"], s["codes"], s["free"], s["n_free"], s["case"]["block"])
        return lens, n_free, s["free"]
    cache = lb.KVCache8(s["k"], s["v"], s["k_scale"], s["v_scale"])
    plan = lb.StepPlan(starts=s["starts"], granted=s["granted"], lens=s["lens"])
    if op == "append":
        lb.append_kv(cache, s["new_k"], s["new_v"], s["table"], plan)
        return s["k"], s["v"], s["k_scale"], s["v_scale"]
    return lb.attend(s["q"], cache, s["table"], plan, scale=s["scale"])


def _plain_int4(s):
    p, scales = s["packed"], s["scales"].float()
    w = torch.stack([p & 15, p >> 4], -1).reshape(p.shape[0], -1).float() - 8.0
    w = (w.view(*scales.shape, -1) * scales[..., None]).view(p.shape[0], -1)
    return (s["x"].float() @ w.t()).to(DTYPES[s["case"]["y"]])


def _plain_plan(s):
    bs, cap, table, free = s["case"]["block"], s["capacity"], s["table"].long(), s["free"].long()
    rows, width = table.shape
    lens, n_free = s["lens"].long(), s["n_free"].long()
    new = s["new"].long().clamp(min=0)
    upto = new.cumsum(0)
    first = upto - new
    held = (lens + bs - 1) // bs
    fits = (new > 0) & (lens >= 0) & (upto <= cap) & (lens + new <= width * bs)
    need = torch.where(fits, (lens + new + bs - 1) // bs - held, 0)
    taken = need.cumsum(0)
    granted = torch.where(fits & ((need == 0) | (taken <= n_free)), new, 0)
    after = n_free - torch.where(granted > 0, need, 0).sum()
    j = torch.arange(width, device=DEV)
    k = (taken - need)[:, None] + j - held[:, None]  # which block of the step this entry of the table takes
    fresh = (granted > 0)[:, None] & (j >= held[:, None]) & (j < (held + need)[:, None])
    table = torch.where(fresh, free[(n_free - 1 - k).clamp(0, free.numel() - 1)], table)
    t = torch.arange(cap, device=DEV)
    row = torch.searchsorted(upto, t, right=True)
    real = row < rows
    row = row.clamp(max=rows - 1)
    pos = torch.where(real, lens[row] + t - first[row], 0)
    page = table[row, (pos // bs).clamp(0, width - 1)]
    slots = torch.where(real & (granted[row] > 0) & (page >= 0) & (page < free.numel()), page * bs + pos % bs, -1)
    starts = torch.cat([first, upto[-1:]]).clamp(max=cap)
    return slots, pos.int(), starts.int(), granted.int(), (lens + granted).int(), after.int(), table.int()


def _plain_release(s):
    bs, table, free, n_free = s["case"]["block"], s["table"].long(), s["free"].long(), s["n_free"].long()
    rows, width = table.shape
    lens, stop = s["lens"].long(), s["codes"] != 0
    back = torch.where(stop, (lens.clamp(0, width * bs) + bs - 1) // bs, 0)
    upto = back.cumsum(0)
    i = torch.arange(free.numel(), device=DEV) - n_free
    row = torch.searchsorted(upto, i, right=True).clamp(max=rows - 1)
    page = table[row, (i - (upto - back)[row]).clamp(0, width - 1)]
    free = torch.where((i >= 0) & (i < upto[-1]), page, free)
    return torch.where(stop, 0, lens).int(), (n_free + upto[-1:]).clamp(max=free.numel()).int(), free.int()


def _plain_append(s):
    bs, dim = s["case"]["block"], s["case"]["dim"]
    lens, granted, starts, table = s["lens"].long(), s["granted"].long(), s["starts"].long()[:-1], s["table"].long()
    old = lens - granted
    steps = torch.arange((s["most"] + bs - 2) // bs + 1, device=DEV)
    at = torch.minimum((old // bs)[:, None] + steps, ((lens - 1) // bs)[:, None])  # the blocks that a row writes; its last one again behind them
    page = torch.gather(table, 1, at)
    pos = at[..., None] * bs + torch.arange(bs, device=DEV)
    fresh = (pos >= old[:, None, None]) & (pos < lens[:, None, None])
    kept = pos < old[:, None, None]
    token = (starts[:, None, None] + pos - old[:, None, None]).clamp(0, s["tokens"] - 1)
    m = lambda t: t[:, :, None, :, None]  # noqa: E731  [rows, blocks, heads, tokens, dim]
    for name in ("k", "v"):
        x = s["new_" + name].float()[token].transpose(2, 3)
        codes, scale = s[name].view(torch.uint8), s[name + "_scale"]
        was_code = codes[page].view(torch.float8_e4m3fn).float()
        was = torch.where(kept.any(-1)[..., None], scale[page], 0.0)
        most = torch.where(m(fresh) & x.isfinite(), x.abs(), 0.0).amax((-1, -2))
        fraction, power = torch.frexp(most)  # most = fraction * 2^power, 448 = 0.875 * 2^9
        need = torch.exp2((power - 9 + (fraction > 0.875).int()).clamp(min=-126).float())
        need = torch.where(most > 0, need, 2.0 ** -126)
        now = torch.maximum(was, need)
        q = torch.where(m(fresh), (x / now[..., None, None]).clamp(-E4M3_MAX, E4M3_MAX), torch.where(m(kept), was_code * (was / now)[..., None, None], was_code))
        codes[page] = q.to(torch.float8_e4m3fn).view(torch.uint8)
        scale[page] = now
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _plain_attend(s):
    case = s["case"]
    heads, per, dim, bs = case["heads"], case["per"], case["dim"], case["block"]
    lens, granted, starts, table = s["lens"].long(), s["granted"].long(), s["starts"].long(), s["table"].long().clamp(min=0)
    rows, width = table.shape
    keys = width * bs

    def gather(name):
        x = s[name].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * s[name + "_scale"][table][..., None, None]
        return x.transpose(1, 2).reshape(rows, heads, keys, dim)

    i = torch.arange(s["most"], device=DEV)
    q = s["q"].float()[(starts[:-1, None] + i).clamp(max=s["tokens"] - 1)]  # [rows, queries, heads * per, dim]
    q = q.view(rows, s["most"], heads, per, dim).permute(0, 2, 3, 1, 4).reshape(rows, heads, per * s["most"], dim)
    scores = (q @ gather("k").transpose(2, 3)).view(rows, heads, per, s["most"], keys) * s["scale"]
    seen = torch.arange(keys, device=DEV) <= (lens - granted)[:, None, None] + i[:, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    live = torch.arange(keys, device=DEV) < lens[:, None]
    v = torch.where(live[:, None, :, None], gather("v"), 0.0)
    o = (p.view(rows, heads, per * s["most"], keys) @ v).view(rows, heads, per, s["most"], dim) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(rows, s["most"], heads * per, dim)
    t = torch.arange(s["tokens"], device=DEV)
    row = torch.searchsorted(starts[1:], t, right=True)
    return o[row, t - starts[row]].to(s["q"].dtype)


# --------------------------------------------------------------------- definitions, 64 bits
def exact(case, seed):
    if case["op"] in ("plan", "release"):
        return None  # whole numbers: they are compared as they are
    s = prepare(case, seed)
    if case["op"] == "int4":
        lo, hi = (s["packed"] & 15).double() - 8, (s["packed"] >> 4).double() - 8
        x, scale = s["x"].double(), s["scales"].double().repeat_interleave(case["group"] // 2, 1)
        return x[:, 0::2] @ (lo * scale).t() + x[:, 1::2] @ (hi * scale).t()
    lens, granted, starts, table = (s[n].tolist() for n in ("lens", "granted", "starts", "table"))
    bs = case["block"]
    if case["op"] == "append":
        out = []
        for name in ("k", "v"):
            codes, scale = s[name].double(), s[name + "_scale"].double()
            for b in range(case["rows"]):
                old = lens[b] - granted[b]
                for j in range(old // bs, (lens[b] - 1) // bs + 1):
                    page, lo, hi = table[b][j], max(old, j * bs), min(lens[b], (j + 1) * bs)
                    x = s["new_" + name][starts[b] + lo - old: starts[b] + hi - old].double().transpose(0, 1)  # [heads, tokens, dim]
                    most = x.abs().amax((1, 2))
                    need = torch.exp2(torch.ceil(torch.log2(most / E4M3_MAX)))
                    need = torch.where(most <= E4M3_MAX * need / 2, need / 2, need)  # a logarithm just above a whole number
                    if lo > j * bs:
                        now = torch.maximum(need, scale[page])
                        codes[page, :, : lo - j * bs] = _to_e4m3(codes[page, :, : lo - j * bs] * (scale[page] / now)[:, None, None])
                    else:
                        now = need
                    codes[page, :, lo - j * bs: hi - j * bs] = _to_e4m3(x / now[:, None, None])
                    scale[page] = now
            out.append((codes, scale))
        return out[0][0], out[1][0], out[0][1], out[1][1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    per = case["per"]
    for b in range(case["rows"]):
        pages = torch.tensor(table[b][: -(-lens[b] // bs)], device=DEV)
        at = torch.arange(lens[b], device=DEV)
        mask = at[None] > torch.arange(lens[b] - granted[b], lens[b], device=DEV)[:, None]
        for h in range(case["heads"]):
            k, v = ((s[n][pages, h].double() * s[n + "_scale"][pages, h].double()[:, None, None]).reshape(-1, case["dim"])[: lens[b]] for n in ("k", "v"))
            for r in range(h * per, (h + 1) * per):
                z = (s["q"][starts[b]: starts[b + 1], r].double() @ k.t() * s["scale"]).masked_fill(mask, -math.inf)
                out[starts[b]: starts[b + 1], r] = torch.softmax(z, -1) @ v
    return out


def _to_e4m3(x):
    """x rounded to the nearest value of 4 exponent and 3 mantissa bits, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (x / step).round() * step
