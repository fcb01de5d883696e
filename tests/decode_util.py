"""Plain 64-bit forms of the decode-step operators, for the tests."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def plan_reference(table, lens, new, free, n_free, bs, capacity):
    """plan_blocks row by row on host lists; returns a dict and the table afterwards."""
    table = [list(r) for r in table]
    width, blocks = len(table[0]), len(free)
    n_free = min(max(n_free, 0), blocks)
    left, wanted, tok = n_free, 0, 0
    slots, positions, starts, granted, out = [-1] * capacity, [0] * capacity, [], [], []
    for b, (ln, nw) in enumerate(zip(lens, new)):
        nw = max(nw, 0)
        starts.append(min(tok, capacity))
        have = -(-ln // bs)
        fits = nw > 0 and ln >= 0 and tok + nw <= capacity and ln + nw <= width * bs
        need = -(-(ln + nw) // bs) - have if fits else 0
        wanted += need
        ok = fits and (need == 0 or wanted <= n_free)
        if ok:
            for j in range(need):
                left -= 1
                table[b][have + j] = free[left]
        for i in range(nw):
            if tok + i < capacity:
                p = ln + i
                positions[tok + i] = p
                if ok and 0 <= table[b][p // bs] < blocks:
                    slots[tok + i] = table[b][p // bs] * bs + p % bs
        granted.append(nw if ok else 0)
        out.append(ln + granted[-1])
        tok += nw
    starts.append(min(tok, capacity))
    return dict(slots=slots, positions=positions, starts=starts, granted=granted, lens=out, n_free=[left]), table


def to_e4m3(x):
    """x (64 bits) to the nearest e4m3 value, ties to even, +-448 beyond the range, NaN kept."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6, max=448.0))) - 3)
    return ((x.clamp(-448, 448) / step).round() * step)


def scale_for(amax):
    """Smallest power of two s >= 2^-126 with amax <= 448 s, by trial."""
    s = 2.0 ** -126
    while amax > 448.0 * s:
        s *= 2.0
    return s


def append_reference(values, scales, x, table, starts, granted, lens):
    """append_kv for one of k, v: values [blocks, heads, bs, dim] and scales in 64 bits, changed in place."""
    bs = values.shape[2]
    for b, (s0, g, ln) in enumerate(zip(starts, granted, lens)):
        if not (0 < g <= ln <= len(table[b]) * bs and s0 + g <= x.shape[0]):
            continue
        old = ln - g
        for j in range(old // bs, (ln - 1) // bs + 1):
            page = table[b][j]
            if not 0 <= page < values.shape[0]:
                continue
            lo, hi = max(old, j * bs) - j * bs, min(ln - j * bs, bs)
            for h in range(values.shape[1]):
                new = x[s0 + j * bs + lo - old: s0 + j * bs + hi - old, h].double()
                fin = new[new.isfinite()].abs()
                s = scale_for(float(fin.max()) if fin.numel() else 0.0)
                was = float(scales[page, h])
                if lo > 0:
                    s = max(s, was)
                    if s != was:
                        values[page, h, :lo] = to_e4m3(values[page, h, :lo] * (was / s))
                values[page, h, lo:hi] = to_e4m3(new / s)
                scales[page, h] = s


def attend_reference(q, k, v, ks, vs, table, starts, granted, lens, scale):
    """(out, sum of |weight * value|, lse) in 64 bits; rows that see nothing give 0 and -inf, other rows
    of q are NaN in all three."""
    T, hq, dim = q.shape
    blocks, heads, bs, _ = k.shape
    per = hq // heads
    out = torch.full((T, hq, dim), math.nan, dtype=torch.float64, device=q.device)
    mag = out.clone()
    lse = torch.full((T, hq), math.nan, dtype=torch.float64, device=q.device)
    for b, (s0, g, ln) in enumerate(zip(starts, granted, lens)):
        if not (0 < g <= ln <= len(table[b]) * bs and s0 + g <= T):
            continue
        pages = torch.tensor(table[b][: -(-ln // bs)], device=q.device)
        good = (pages >= 0) & (pages < blocks)
        at = pages.clamp(0, blocks - 1)
        seen = good.repeat_interleave(bs)[:ln][None] & (torch.arange(ln, device=q.device)[None] <= torch.arange(ln - g, ln, device=q.device)[:, None])
        for h in range(heads):
            kk = (k[at, h].double() * ks[at, h].double()[:, None, None]).reshape(-1, dim)[:ln]
            vv = (v[at, h].double() * vs[at, h].double()[:, None, None]).reshape(-1, dim)[:ln]
            for r in range(h * per, (h + 1) * per):
                qq = q[s0: s0 + g, r].double()
                z = torch.where(seen, torch.where(seen, qq @ kk.t(), 0.0) * scale, -math.inf)
                top = z.amax(-1, keepdim=True)
                p = torch.where(seen, torch.exp(z - torch.where(top == -math.inf, 0.0, top)), 0.0)
                tot = p.sum(-1, keepdim=True)
                if bool(vv.isfinite().all()):
                    out[s0: s0 + g, r], mag[s0: s0 + g, r] = ((p @ x) / torch.where(tot == 0, 1.0, tot) for x in (vv, vv.abs()))
                for i in range(0 if bool(vv.isfinite().all()) else g):  # only what a query sees enters its sum
                    w = p[i][seen[i]] / tot[i]
                    out[s0 + i, r] = (w[:, None] * vv[seen[i]]).sum(0) if tot[i] != 0 else 0.0
                    mag[s0 + i, r] = (w[:, None] * vv[seen[i]].abs()).sum(0) if tot[i] != 0 else 0.0
                lse[s0: s0 + g, r] = torch.where(tot[:, 0] == 0, -math.inf, torch.log(tot[:, 0]) + torch.where(top[:, 0] == -math.inf, 0.0, top[:, 0]))
    return out, mag, lse


def make_rows(ctx, new, bs, extra=3, seed=0, device="cuda"):
    """Shuffled block table for rows of ctx + new tokens: (table list, tensor, starts, granted, lens, blocks)."""
    g = torch.Generator().manual_seed(seed)
    lens = [c + n for c, n in zip(ctx, new)]
    need = [-(-ln // bs) for ln in lens]
    blocks = sum(need) + extra
    ids = torch.randperm(blocks, generator=g).tolist()
    width = max(need + [1])
    table, at = [], 0
    for n in need:
        table.append(ids[at: at + n] + [-1] * (width - n))
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    return table, t(table), t(starts), t(new), t(lens), blocks


def random_cache(blocks, heads, bs, dim, seed=0, device="cuda"):
    """Cache tensors with codes of spread magnitudes and uneven power-of-two scales."""
    g = torch.Generator(device=device).manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn(blocks, heads, bs, dim, generator=g, device=device) * 100
        out.append(x.clamp(-448, 448).to(E4M3))
    for _ in range(2):
        out.append(torch.exp2(torch.randint(-9, -5, (blocks, heads), generator=g, device=device).float()))
    k, v, ks, vs = out
    return k, v, ks, vs
