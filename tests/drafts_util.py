"""Plain forms of the operators around drafted tokens and shared blocks, for the tests: whole numbers row by
row on the host, computed values in 64 bits."""
import math
import random

import torch

from tests.decode_util import to_e4m3

TREE_MOST = 1024


def clean_parents(parents):
    """One row's parents as they count: an earlier token or -1; long rows are chains."""
    if len(parents) > TREE_MOST:
        return list(range(-1, len(parents) - 1))
    return [p if 0 <= p < i else -1 for i, p in enumerate(parents)]


def ancestors(parents):
    """[n][n] of whether j is i or an ancestor of it."""
    parents = clean_parents(parents)
    out = []
    for i, p in enumerate(parents):
        line = list(out[p]) if p >= 0 else [False] * len(parents)
        line[i] = True
        out.append(line)
    return out


def random_tree(n, rng, chain=0.5, root=0.05):
    return [-1 if i == 0 or rng.random() < root else i - 1 if rng.random() < chain else rng.randrange(i) for i in range(n)]


def row_ok(s, g, ln, T):
    return 0 < g <= ln and 0 <= s and s + g <= T


def tree_reference(parents, starts, granted, lens, T):
    """(span, positions) by walks through each row's forest."""
    span, positions = [[0, 0] for _ in range(T)], [0] * T
    for s, g, ln in zip(starts, granted, lens):
        if not row_ok(s, g, ln, T):
            continue
        par = clean_parents(parents[s: s + g])
        children = {}
        for i, p in enumerate(par):
            children.setdefault(p, []).append(i)
        order, stack = 0, [(c, 0) for c in reversed(children.get(-1, []))]
        while stack:
            i, depth = stack.pop()
            span[s + i][0], positions[s + i] = order, ln - g + depth
            order += 1
            stack += [(c, depth + 1) for c in reversed(children.get(i, []))]
        for i in reversed(range(g)):
            span[s + i][1] += 1
            if par[i] >= 0:
                span[s + par[i]][1] += span[s + i][1]
    return span, positions


def accept_reference(parents, tokens, targets, codes, given, starts, granted, lens, T):
    path, said, counts, out, last, stop = [-1] * T, [-1] * T, [], [], [], []
    for b, (s, g, ln) in enumerate(zip(starts, granted, lens)):
        if not row_ok(s, g, ln, T):
            counts.append(0)
            out.append(ln - max(g, 0))
            last.append(-1)
            stop.append(0)
            continue
        par = clean_parents(parents[s: s + g])
        n0 = min(max(given[b] if given else 1, 1), g)
        kept, new = list(range(n0)), []
        while True:
            cur = kept[-1]
            new.append(targets[s + cur])
            code = codes[s + cur] if codes else 0
            nxt = [i for i in range(cur + 1, g) if par[i] == cur and tokens[s + i] == targets[s + cur]]
            if code or not nxt:
                break
            kept.append(nxt[0])
        path[s: s + len(kept)] = kept
        said[s: s + len(new)] = new
        counts.append(len(kept))
        out.append(ln - g + len(kept))
        last.append(new[-1])
        stop.append(code)
    return path, said, counts, out, last, stop


def attend_tree_reference(q, k, v, ks, vs, table, starts, granted, lens, scale, parents):
    """(out, sum of |weight * value|, lse) in 64 bits; queries that see nothing give 0 and -inf, tokens of no row
    are NaN in all three."""
    T, hq, dim = q.shape
    blocks, heads, bs, _ = k.shape
    per = hq // heads
    out = torch.full((T, hq, dim), math.nan, dtype=torch.float64, device=q.device)
    mag, lse = out.clone(), torch.full((T, hq), math.nan, dtype=torch.float64, device=q.device)
    for s, g, ln, line in zip(starts, granted, lens, table):
        if not row_ok(s, g, ln, T) or ln > len(line) * bs:
            continue
        pages = torch.tensor(line[: -(-ln // bs)], device=q.device)
        good = (pages >= 0) & (pages < blocks)
        at = pages.clamp(0, blocks - 1)
        seen = torch.ones(g, ln, dtype=torch.bool, device=q.device)
        seen[:, ln - g:] = torch.tensor(ancestors(parents[s: s + g]), device=q.device)
        seen &= good.repeat_interleave(bs)[:ln]
        for h in range(heads):
            kk = (k[at, h].double() * ks[at, h].double()[:, None, None]).reshape(-1, dim)[:ln]
            vv = (v[at, h].double() * vs[at, h].double()[:, None, None]).reshape(-1, dim)[:ln]
            nan = vv.isnan()
            spoiled = seen.double() @ nan.double() > 0  # [g, dim]: a NaN among the values that it sees
            vv = torch.where(nan, 0.0, vv)
            for r in range(h * per, (h + 1) * per):
                z = torch.where(seen, torch.nan_to_num(q[s: s + g, r].double() @ kk.t(), 0.0) * scale, -math.inf)
                top = z.amax(-1, keepdim=True)
                top = torch.where(top == -math.inf, 0.0, top)
                p = torch.exp(z - top)
                tot = p.sum(-1, keepdim=True)
                part = p / torch.where(tot == 0, 1.0, tot)
                out[s: s + g, r] = torch.where(spoiled, math.nan, part @ vv)
                mag[s: s + g, r] = part @ vv.abs()
                lse[s: s + g, r] = (torch.log(tot) + top)[:, 0]
    return out, mag, lse


def compact_reference(values, scales, table, starts, granted, lens, path, counts):
    """compact_kv for one of k, v: values [blocks, heads, bs, dim] and scales [blocks, heads] in 64 bits, changed in place."""
    blocks, heads, bs, _ = values.shape
    T = len(path)
    for b, (s, g, ln) in enumerate(zip(starts, granted, lens)):
        kept = min(counts[b], g)
        if not row_ok(s, g, ln, T) or kept < 1 or ln > len(table[b]) * bs:
            continue
        old = ln - g
        before, scale_before = values.clone(), scales.clone()
        for j in range(old // bs, (old + kept - 1) // bs + 1):
            page = table[b][j]
            if not 0 <= page < blocks:
                continue
            come = {}
            for p in range(j * bs, min((j + 1) * bs, old + kept)):
                i = path[s + p - old] if p >= old else 0
                src = old + i if p >= old and p - old < i < g else p
                at = table[b][src // bs]
                come[p] = (at, src % bs) if 0 <= at < blocks else (page, p % bs)
            if all(c == (page, p % bs) for p, c in come.items()):
                continue
            top = torch.stack([scale_before[a] for a, _ in come.values()]).amax(0)
            for p, (a, o) in come.items():
                values[page, :, p % bs] = to_e4m3(before[a, :, o] * (scale_before[a] / top)[:, None])
            scales[page] = top


def fork_reference(table, lens, src, dst, upto, shares, free, n_free, bs):
    """fork_blocks one after the other; the table and shares afterwards too."""
    table, shares, out = [list(r) for r in table], list(shares), list(lens)
    B, width, blocks = len(table), len(table[0]), len(free)
    n_free = min(max(n_free, 0), blocks)
    left, wanted, named, granted, copies = n_free, 0, set(), [], []
    for i, (s, d) in enumerate(zip(src, dst)):
        t = 0
        if 0 <= s < B and 0 <= d < B and lens[d] == 0 and d not in named:
            t = min(lens[s], upto[i]) if upto else lens[s]
            t = t if 0 <= t <= width * bs else 0
        named.add(d)
        need = t % bs != 0
        wanted += need
        ok = t > 0 and (not need or wanted <= n_free)
        granted.append(t if ok else 0)
        copies.append([-1, -1])
        if not ok:
            continue
        for j in range(t // bs):
            table[d][j] = table[s][j]
            if 0 <= table[s][j] < blocks:
                shares[table[s][j]] += 1
        if need:
            left -= 1
            copies[-1] = [table[s][t // bs], free[left]]
            table[d][t // bs] = free[left]
            if 0 <= free[left] < blocks:
                shares[free[left]] = 0
        out[d] = t
    return dict(lens=out, n_free=[left], granted=granted, copies=copies), table, shares


def give_reference(table, lens, codes, keep, shares, free, n_free, bs):
    """release_blocks with keep and shares, one block after the other: (lens, n_free, free, shares)."""
    blocks, width = len(free), len(table[0])
    free, out, given = list(free), [], []
    for b, ln in enumerate(lens):
        now = 0 if codes[b] else min(max(keep[b], 0), ln) if keep else ln
        out.append(now)
        lo, hi = (-(-min(max(x, 0), width * bs) // bs) for x in (now, ln))
        given += [i for i in table[b][lo:hi] if 0 <= i < blocks]
    n_free = min(max(n_free, 0), blocks)
    back = given
    if shares is not None:
        shares, back, gone = list(shares), [], set()
        for i in given:
            shares[i] -= 1
        for i in reversed(given):  # the last holder's place counts
            if shares[i] < 0 and i not in gone:
                gone.add(i)
                back.insert(0, i)
        for i in gone:
            shares[i] = 0
    for i in back:
        if n_free < blocks:
            free[n_free] = i
            n_free += 1
    return out, [n_free], free, shares


def rotate_reference(x, positions, freqs, weight, eps, interleaved):
    """(result, sum of the magnitudes that enter it) in 64 bits."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    n = freqs.numel()
    a = positions.double()[:, None, None] * freqs.double()
    cos, sin = torch.cos(a), torch.sin(a)
    first = torch.arange(n, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else n)
    out, mag = y.clone(), y.abs()
    out[..., first] = y[..., first] * cos - y[..., second] * sin
    out[..., second] = y[..., second] * cos + y[..., first] * sin
    mag[..., first] = mag[..., second] = y[..., first].abs() + y[..., second].abs()
    return out, mag


def random_step(ctx, new, seed, gaps=False):
    """Host lists of a step: (starts, granted, lens, parents, T); rows with gaps refuse their tokens now and then."""
    rng = random.Random(seed)
    starts, parents = [0], []
    granted, lens = [], []
    for c, n in zip(ctx, new):
        refused = gaps and rng.random() < 0.2
        granted.append(0 if refused else n)
        lens.append(c + granted[-1])
        parents += random_tree(n, rng)
        starts.append(starts[-1] + n)
    return starts, granted, lens, parents, starts[-1]
