"""The operators around drafted tokens and shared blocks on the GPU against plain forms: whole numbers
exactly, computed values in 64 bits."""
import random

import pytest
import torch

import localstrm_b200 as lb
from tests import decode_util as U
from tests import drafts_util as D

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
DEV = torch.device("cuda", 0)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------ norms and rotation
def check_rotate(q, k, positions, freqs, qw, kw, interleaved, eps=1e-6, **out):
    """All in f32: a sum of squares of at most 32 terms one after the other and joined in 5 steps (half of its
    error goes into the root), the root and its reciprocal to 2^-22, three products, sine and cosine to 2^-22 and their
    argument to 2^-23, two products and a sum: less than 32 times 2^-24 of the magnitudes that enter.  Then half a step of the type,
    and of its smallest numbers."""
    inputs = [x.clone() for x in (q, k)]
    got = lb.norm_rotate(q, k, positions, freqs, q_weight=qw, k_weight=kw, eps=eps, interleaved=interleaved, **out)
    for x, y, w in zip(inputs, got, (qw, kw)):
        want, mag = D.rotate_reference(x, positions, freqs, w, eps, interleaved)
        tol = 2.0 ** -19 * mag + torch.finfo(x.dtype).eps / 2 * want.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 0)
        off = (y.double() - want).abs()
        assert y.dtype == x.dtype and y.shape == x.shape
        assert bool((off <= tol).all()), (float((off - tol).max()), (off > tol).nonzero()[:4].tolist())
    return got


def rotate_case(T, hq, hk, dim, rot, dt, seed, far=131071, norm=True):
    g = gen(seed)
    q, k = (torch.randn(T, h, dim, generator=g, device=DEV).to(dt) for h in (hq, hk))
    freqs = (10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / max(rot, 1))).float()
    w = lambda: (1 + 0.3 * torch.randn(dim, generator=g, device=DEV)).to(dt) if norm else None
    return q, k, torch.randint(0, far + 1, (T,), generator=g, device=DEV).int(), freqs, w(), w()


@pytest.mark.parametrize("T,hq,hk,dim,rot", [
    (1, 1, 1, 64, 64), (1, 14, 2, 64, 64), (3, 32, 8, 128, 128), (257, 4, 1, 128, 64), (33, 6, 2, 256, 256), (20, 3, 3, 80, 80), (20, 5, 1, 80, 32),
    (9, 2, 1, 96, 96), (7, 3, 2, 512, 512), (5, 2, 2, 48, 16), (6, 2, 1, 72, 36), (4, 3, 1, 2, 2), (11, 2, 1, 66, 20), (2000, 32, 8, 128, 128),
    (3001, 1, 1, 64, 32), (4, 2, 1, 510, 254), (6, 4, 2, 128, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotate_sizes(T, hq, hk, dim, rot, dtype, interleaved):
    for norm in (True, False):
        q, k, pos, freqs, qw, kw = rotate_case(T, hq, hk, dim, rot, DTYPES[dtype], T + dim, norm=norm)
        first = check_rotate(q, k, pos, freqs, qw, kw, interleaved)
        again = lb.norm_rotate(q, k, pos, freqs, q_weight=qw, k_weight=kw, interleaved=interleaved)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_rotate_layouts_and_places():
    T, hq, hk, dim = 37, 6, 2, 128
    for dt in (torch.bfloat16, torch.float32):
        _, _, pos, freqs, qw, kw = rotate_case(T, hq, hk, dim, dim, dt, 5)
        for off in (0, 1):  # slices of a fused projection, 16-byte aligned and not; in place; one of the two only
            fused = torch.randn(T, 1400, generator=gen(6), device=DEV).to(dt)
            q, k = fused[:, off: off + hq * dim].view(T, hq, dim), fused[:, off + hq * dim: off + (hq + hk) * dim].view(T, hk, dim)
            want = check_rotate(q, k, pos, freqs, qw, kw, False)
            check_rotate(q, k, pos, freqs, None, kw, True)
            rest = fused[:, off + (hq + hk) * dim:].clone()
            got = check_rotate(q, k, pos, freqs, qw, kw, False, q_out=q, k_out=k)
            assert got[0] is q and got[1] is k and torch.equal(q, want[0]) and torch.equal(k, want[1])
            assert torch.equal(fused[:, off + (hq + hk) * dim:], rest) and bool((fused[:, :off] == fused[:, :off]).all())
        # head by head, results with strides of their own, inner strides other than 1, one key head for all tokens
        q = torch.randn(hq, T, dim, generator=gen(7), device=DEV).to(dt).transpose(0, 1)
        k = torch.randn(T, dim, hk, generator=gen(8), device=DEV).to(dt).transpose(1, 2)
        out = torch.zeros(T, hq, 200, dtype=dt, device=DEV)
        check_rotate(q, k, pos, freqs, qw, kw, False, q_out=out[:, :, :dim], k_out=torch.empty(hk, T, dim, dtype=dt, device=DEV).transpose(0, 1))
        assert bool((out[:, :, dim:] == 0).all())
        check_rotate(q, k[:1].expand(T, hk, dim), pos, freqs, qw, kw, False)
    # weights of another type, other eps, tiny values
    q, k, pos, freqs, _, _ = rotate_case(5, 2, 1, 64, 64, torch.float16, 9)
    w = 1 + 0.1 * torch.randn(64, generator=gen(1), device=DEV)
    check_rotate(q, k, pos, freqs, w, w.clone(), False, eps=1e-2)
    check_rotate(q * 0, k * 1e-3, pos, freqs, w.bfloat16(), w.bfloat16(), True)


def test_rotate_far_and_negative_positions():
    q, k, _, freqs, qw, kw = rotate_case(8, 2, 1, 128, 128, torch.float32, 3)
    check_rotate(q, k, ints([0, 1, 131071, 1 << 20, (1 << 24) + 1, 1 << 27, -5, -131072]), freqs, qw, kw, False)


def test_rotate_refusals():
    q, k, pos, freqs, qw, kw = rotate_case(4, 2, 1, 64, 64, torch.bfloat16, 1)
    bad = [(q[:3], k, pos, freqs), (q, k[..., :32], pos, freqs), (q, k, pos.long(), freqs), (q, k, pos[:3], freqs), (q, k, pos, freqs.double()),
           (q, k, pos, torch.ones(33, device=DEV)), (q, k, pos.cpu(), freqs), (q[0], k[0], pos, freqs)]
    for a in bad:
        with pytest.raises(ValueError):
            lb.norm_rotate(*a)
    for kw_ in (dict(q_weight=qw[:32]), dict(k_weight=kw.cpu()), dict(q_out=torch.empty_like(q, dtype=torch.float32)), dict(k_out=k[..., :32])):
        with pytest.raises(ValueError):
            lb.norm_rotate(q, k, pos, freqs, **kw_)
    for a, b in ((q.half(), k), (q.double(), k.double())):
        with pytest.raises(TypeError):
            lb.norm_rotate(a, b, pos, freqs)
    with pytest.raises(TypeError):
        lb.norm_rotate(q, k, pos, freqs, q_weight=qw, k_weight=kw.float())
    with pytest.raises(lb.SamplerError):
        lb.norm_rotate(q, k, pos, freqs, q_out=k.expand(4, 2, 64))  # rows over each other


# ------------------------------------------------------------------------------------------- trees
def step_tensors(starts, granted, lens):
    return lb.StepPlan(ints(starts), ints(granted), ints(lens))


@pytest.mark.parametrize("ctx,new", [([0], [1]), ([700], [6]), ([5, 0, 9, 33], [64, 3, 0, 17]), ([1] * 300, [i % 40 for i in range(300)]), ([10, 3, 8], [65, 129, 200]),
                                     ([4, 4], [1024, 1023]), ([2, 50], [1500, 7])])
@pytest.mark.parametrize("kind", ["mixed", "chains", "deep", "bushy"])
def test_trees_and_acceptance(ctx, new, kind):
    for seed in range(2):
        rng = random.Random(seed)
        starts, granted, lens, parents, T = D.random_step(ctx, new, seed, gaps=True)
        if kind != "mixed":
            parents = []
            for n in new:
                parents += D.random_tree(n, rng, chain={"chains": 1.0, "deep": 0.97, "bushy": 0.1}[kind], root={"chains": 0.0, "deep": 0.0, "bushy": 0.2}[kind])
        extra = 5 * seed  # tokens behind the last row
        parents += [7] * extra
        T += extra
        if seed and T > 3:  # what is no earlier token
            for bad in (T // 2, T - extra - 1, 1):
                parents[bad] = rng.choice([-7, 10 ** 6, T])
        plan = step_tensors(starts, granted, lens)
        tree = lb.plan_tree(plan, ints(parents))
        span, positions = D.tree_reference(parents, starts, granted, lens, T)
        assert tree.span.tolist() == span and tree.positions.tolist() == positions
        # few different tokens, so that several children agree, and branches are followed far
        tokens, targets = [rng.randrange(3) for _ in range(T)], [rng.randrange(3) for _ in range(T)]
        codes = [int(rng.random() < 0.03) * 2 for _ in range(T)]
        given = [rng.choice([1, 1, 1, 2, 5, 0, 10 ** 6]) for _ in ctx]
        for c, gv in ((None, None), (codes, None), (codes, given)):
            a = lb.accept_drafts(plan, tree, ints(tokens), ints(targets), codes=None if c is None else ints(c), given=None if gv is None else ints(gv))
            want = D.accept_reference(parents, tokens, targets, c, gv, starts, granted, lens, T)
            assert tuple(x.tolist() for x in (a.path, a.tokens, a.counts, a.lens, a.last, a.codes)) == want


def test_trees_odd_plans():
    # rows whose numbers do not fit: more new tokens than tokens, tokens outside the step; no rows; no tokens
    parents = [-1, 0, 1, 0, -1, 0]
    for starts, granted, lens in (([0, 3, 6], [3, 3], [2, 9]), ([0, 4, 6], [4, 3], [5, 9]), ([-2, 3, 6], [3, 3], [9, 9]), ([1, 3, 5], [2, 2], [9, 9]), ([0], [], [])):
        plan, B = step_tensors(starts, granted, lens), len(granted)
        tree = lb.plan_tree(plan, ints(parents))
        span, positions = D.tree_reference(parents, starts, granted, lens, 6)
        assert tree.span.tolist() == span and tree.positions.tolist() == positions
        a = lb.accept_drafts(plan, tree, ints(parents), ints(parents))
        assert tuple(x.tolist() for x in (a.path, a.tokens, a.counts, a.lens, a.last, a.codes)) == \
            D.accept_reference(parents, parents, parents, None, None, starts, granted, lens, 6)
    none = ints([])
    tree = lb.plan_tree(step_tensors([0, 0], [0], [5]), none)
    a = lb.accept_drafts(step_tensors([0, 0], [0], [5]), tree, none, none)
    assert tree.span.shape == (0, 2) and a.counts.tolist() == [0] and a.lens.tolist() == [5] and a.last.tolist() == [-1]
    # lengths in place
    plan = step_tensors([0, 6], [6], [16])
    a = lb.accept_drafts(plan, lb.plan_tree(plan, ints([-1, 0, 0, 2, 2, -1])), ints([50, 7, 8, 9, 9, 1]), ints([8, 0, 9, 33, 34, 2]), lens_out=plan.lens)
    assert a.lens is plan.lens and plan.lens.tolist() == [13]


# --------------------------------------------------------------------------------------- attention
def check_attend_tree(q, cache, rows, parents, scale=None, out=None):
    """As for the causal form: weights are rounded to f16 (2^-11 of the sum of |weight * value|), scores and
    exponentials in f32 held to a quarter of that, and the result is rounded once."""
    table, t, starts, granted, lens, blocks = rows
    sc = q.shape[2] ** -0.5 if scale is None else scale
    plan = lb.StepPlan(starts, granted, lens)
    tree = lb.plan_tree(plan, ints(parents))
    lse = torch.full(q.shape[:2], 77.0, device=DEV)
    y = torch.full(q.shape, 77.0, dtype=q.dtype, device=DEV) if out is None else out
    keep = q.clone()
    lb.attend(q, cache, t, plan, scale=scale, out=y, lse_out=lse, tree=tree)
    want, mag, wl = D.attend_tree_reference(keep, cache.k, cache.v, cache.k_scale, cache.v_scale, table, starts.tolist(), granted.tolist(), lens.tolist(), sc, parents)
    idle = wl.isnan()
    assert bool((lse[idle] == 77).all()) and (out is not None or bool((y[idle] == 77).all()))
    tol = 1.25 * 2.0 ** -11 * mag + torch.finfo(q.dtype).eps / 2 * want.abs() + (2.0 ** -24 if q.dtype == torch.float16 else 0)
    off = (y.double() - want).abs()
    # a result from half a step above f16's largest number on (65504 + 16) rounds to infinity
    over = y.isinf() & (want.abs() + tol >= 65520.0) & (want.sign() == y.sign()) if q.dtype == torch.float16 else torch.zeros_like(idle[..., None])
    ok = (off <= tol) | (want.isnan() & (y.isnan() | idle[..., None])) | over
    assert bool(ok.all()), (float((off - tol).nan_to_num(0).max()), ok.logical_not().nonzero()[:5].tolist())
    assert bool((((lse.double() - wl).abs() <= 2.0 ** -16 * (1 + wl.abs())) | (lse == wl) | idle).all())
    return y, lse


def tree_rows(ctx, new, bs, seed):
    rng = random.Random(seed)
    return U.make_rows(ctx, new, bs, seed=seed), [p for n in new for p in D.random_tree(n, rng)]


TREES = [  # few query rows, groups of 8, 16 and 32, and those of the tensor-memory kernel
    ([0], [1], 1, 1, 16, 64), ([700], [6], 2, 7, 16, 64), ([15, 16, 17, 0], [2, 5, 1, 3], 2, 4, 16, 128), ([300, 2, 1111], [3, 9, 16], 2, 4, 32, 128),
    ([0, 900], [8, 33], 1, 2, 64, 256), ([70, 0, 5, 33], [5, 40, 1, 16], 2, 3, 16, 128), ([5000, 40], [64, 31], 8, 8, 32, 128), ([1000, 3, 127, 128, 129], [64, 64, 1, 65, 127], 4, 4, 16, 128),
    ([900, 61, 64], [70, 128, 200], 8, 4, 16, 64), ([40], [600], 8, 2, 128, 128), ([0, 10], [64, 300], 8, 7, 64, 64), ([2000] * 8, [8] * 8, 8, 4, 16, 128)]


@pytest.mark.parametrize("ctx,new,heads,per,bs,dim", TREES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attend_tree_sizes(ctx, new, heads, per, bs, dim, dtype):
    rows, parents = tree_rows(ctx, new, bs, dim)
    cache = lb.KVCache8(*U.random_cache(rows[-1], heads, bs, dim, seed=per))
    q = torch.randn(sum(new) + 2, heads * per, dim, generator=gen(dim), device=DEV).to(DTYPES[dtype])
    y, lse = check_attend_tree(q, cache, rows, parents + [-1, -1])
    y2, lse2 = check_attend_tree(q, cache, rows, parents + [-1, -1])
    assert torch.equal(y[: sum(new)], y2[: sum(new)]) and torch.equal(lse, lse2)


@pytest.mark.parametrize("ctx,new,heads,per,bs,dim", [TREES[3], TREES[5], TREES[6], TREES[8], TREES[4]])
def test_attend_tree_of_chains_is_causal(ctx, new, heads, per, bs, dim):
    rows, _ = tree_rows(ctx, new, bs, 1)
    cache = lb.KVCache8(*U.random_cache(rows[-1], heads, bs, dim, seed=per))
    q = torch.randn(sum(new), heads * per, dim, generator=gen(dim), device=DEV).half()
    chains = [i - 1 for n in new for i in range(n)]
    y, lse = check_attend_tree(q, cache, rows, chains)
    lse2 = torch.empty_like(lse)
    causal = lb.attend(q, cache, rows[1], lb.StepPlan(*rows[2:5]), lse_out=lse2)
    # The two forms may take other kernels and cut the work elsewhere, so that sums round differently: both are within the
    # bound of the same exact result (the causal one by its own tests).
    want, mag, _ = U.attend_reference(q, cache.k, cache.v, cache.k_scale, cache.v_scale, rows[0], *(x.tolist() for x in rows[2:5]), dim ** -0.5)
    tol = 1.25 * 2.0 ** -11 * mag + torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -24
    assert bool(((y.double() - want).abs() <= tol).all()) and bool(((y.double() - causal.double()).abs() <= 2 * tol).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("per", [4, 3])
def test_attend_chunks_of_whole_and_half_groups(dim, per):
    """Groups of up to 128 query rows behind ones of 256, causal and as chains: in the first ones the two streams take
    every other step each, and must not take a stage of keys for one that comes later."""
    ctx, new = [1000, 2003, 61, 3340], [256, 353, 700, 431]
    rows = U.make_rows(ctx, new, 16, seed=dim + per)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 8, 16, dim, seed=per))
    q = torch.randn(sum(new), 8 * per, dim, generator=gen(dim), device=DEV).bfloat16()
    y, _ = check_attend_tree(q, cache, rows, [i - 1 for n in new for i in range(n)])
    want, mag, _ = U.attend_reference(q, cache.k, cache.v, cache.k_scale, cache.v_scale, rows[0], *(x.tolist() for x in rows[2:5]), dim ** -0.5)
    for _ in range(3):
        causal = lb.attend(q, cache, rows[1], lb.StepPlan(*rows[2:5]))
        assert bool(((causal.double() - want).abs() <= 1.25 * 2.0 ** -11 * mag + 2.0 ** -8 * want.abs()).all())


@pytest.mark.parametrize("ctx,new,heads,per,dim", [([20, 3], [9, 5], 2, 4, 128), ([20, 100], [64, 70], 8, 4, 128), ([20, 1], [33, 90], 8, 7, 64), ([5, 0], [7, 20], 2, 1, 256)])
def test_attend_tree_nan_and_bad_blocks(ctx, new, heads, per, dim):
    """NaN among keys and values of drafted tokens reaches their own branches alone; blocks that are none are not seen."""
    bs = 16
    rows, parents = tree_rows(ctx, new, bs, 4)
    table, t, starts, granted, lens, blocks = rows
    k, v, ks, vs = U.random_cache(blocks, heads, bs, dim, seed=3)
    rng = random.Random(5)
    vb, kb = v.view(torch.uint8), k.view(torch.uint8)
    for b in range(len(ctx)):  # values: a few columns of a few new tokens, and of one token of the context
        for pos in [ctx[b] + rng.randrange(new[b]) for _ in range(4)] + ([rng.randrange(ctx[b])] if b == 1 and ctx[b] else []):
            vb[table[b][pos // bs], rng.randrange(heads), pos % bs, rng.randrange(dim)] = rng.choice([0x7f, 0xff])
    q = torch.randn(sum(new), heads * per, dim, generator=gen(2), device=DEV).bfloat16()
    check_attend_tree(q, lb.KVCache8(k, v, ks, vs), rows, parents)
    # keys: the branch's queries are NaN, all others as without
    cache = lb.KVCache8(k, torch.where(v.float().isnan(), 0.0, v.float()).to(U.E4M3), ks, vs)
    y0, _ = check_attend_tree(q, cache, rows, parents)
    node = new[0] // 2
    pos = ctx[0] + node
    kb[table[0][pos // bs], 0, pos % bs, 3] = 0x7f
    plan = lb.StepPlan(starts, granted, lens)
    y = lb.attend(q, cache, t, plan, tree=lb.plan_tree(plan, ints(parents)))
    up = D.ancestors(parents[: new[0]])
    hit = torch.zeros(sum(new), heads * per, dtype=torch.bool, device=DEV)
    for i in range(new[0]):
        hit[i, :per] = up[i][node]
    assert torch.equal(y[~hit], y0[~hit]) and bool(y[hit].isnan().all())
    # a block of the new tokens that is none: what lies in it is not seen
    kb[table[0][pos // bs], 0, pos % bs, 3] = 0x21
    gone = ctx[0] // bs + 1
    if gone < len(table[0]) and table[0][gone] >= 0:
        for wrong in (-1, blocks, 10 ** 9):
            line = [list(r) for r in table]
            line[0][gone] = wrong
            check_attend_tree(q, cache, (line, ints(line), starts, granted, lens, blocks), parents)
    # none of its blocks: queries without a context see nothing at all
    line = [list(r) for r in table]
    line[1] = [-1] * len(line[1])
    check_attend_tree(q, cache, (line, ints(line), starts, granted, lens, blocks), parents)


def test_attend_tree_layouts_and_refusals():
    rows, parents = tree_rows([100, 33], [9, 20], 16, 2)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 2, 16, 128))
    for off in (0, 1):
        for dt in (torch.bfloat16, torch.float16):
            fused = torch.randn(29, 1400, generator=gen(2), device=DEV).to(dt)
            q = fused[:, off: off + 768].view(29, 6, 128)
            check_attend_tree(q, cache, rows, parents, scale=-0.05)
            out = torch.zeros(29, 6, 150, dtype=dt, device=DEV)
            check_attend_tree(q, cache, rows, parents, scale=0.3, out=out[:, :, off: off + 128])
            assert bool((out[:, :, off + 128:] == 0).all())
            check_attend_tree(q, cache, rows, parents, out=q)
    cache.v_scale.mul_(torch.exp2(torch.randint(-30, 30, cache.v_scale.shape, generator=gen(6), device=DEV).float()) * 1.3)
    check_attend_tree(torch.randn(29, 6, 128, generator=gen(3), device=DEV).half(), cache, rows, parents)
    # rows refused, a row whose numbers do not fit: left as they were
    table, t, starts, granted, lens, blocks = rows
    q = torch.randn(29, 6, 128, generator=gen(3), device=DEV).half()
    for g, ln in (([0, 20], [100, 53]), ([9, 60], [109, 53]), ([9, 20], [109, 10 ** 6])):
        check_attend_tree(q, cache, (table, t, starts, ints(g), ints(ln), blocks), parents)
    plan = lb.StepPlan(starts, granted, lens)
    tree = lb.plan_tree(plan, ints(parents))
    for bad in (tree.span[:28], tree.span.long(), tree.span.cpu(), tree.span.t().contiguous(), tree.span.flatten()):
        with pytest.raises((ValueError, RuntimeError)):
            lb.attend(q, cache, t, plan, tree=lb.TreePlan(bad, tree.positions, tree.parents))


# --------------------------------------------------------------------------- accepted tokens move up
@pytest.mark.parametrize("per,dim", [(4, 128), (4, 64), (16, 128)])
def test_attend_rows_between_the_kernels(per, dim):
    """Rows on both sides of every border between the kernels in one step: 16 to 64 query rows, lengths around 640, 1,024 and 2,560, and short ones."""
    new = [(4, 5, 8, 9, 12, 13, 15, 16)[i % 8] * 4 // per or 1 for i in range(72)]
    ctx = [(2559, 2560, 2561, 1023, 1024, 639, 640, 17, 0)[i // 8] - (n if i // 8 < 7 else 0) for i, n in enumerate(new)]
    rows, parents = tree_rows(ctx, new, 16, per)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 8, 16, dim, seed=per))
    q = torch.randn(sum(new) + 1, 8 * per, dim, generator=gen(dim), device=DEV).bfloat16()
    y, lse = check_attend_tree(q, cache, rows, parents + [-1])
    assert bool(y[: sum(new)].isfinite().all())
    chains = [i - 1 for n in new for i in range(n)]
    check_attend_tree(q, cache, rows, chains + [-1])
    got = lb.attend(q[: sum(new)], cache, rows[1], lb.StepPlan(*rows[2:5]))
    want, mag, _ = U.attend_reference(q[: sum(new)], cache.k, cache.v, cache.k_scale, cache.v_scale, rows[0], *(x.tolist() for x in rows[2:5]), dim ** -0.5)
    tol = 1.25 * 2.0 ** -11 * mag + torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -24
    assert bool(((got.double() - want).abs() <= tol).all())


def check_compact(rows, heads, bs, dim, path, counts, seed, scales=None, nan=False):
    table, t, starts, granted, lens, blocks = rows
    k, v, ks, vs = U.random_cache(blocks, heads, bs, dim, seed=seed)
    if scales is not None:
        for s in (ks, vs):
            s.copy_(scales(s))
    if nan:
        for x in (k, v):
            x.view(torch.uint8)[torch.rand(x.shape, generator=gen(seed), device=DEV) < 0.05] = 0x7f
            x.view(torch.uint8)[torch.rand(x.shape, generator=gen(seed + 1), device=DEV) < 0.02] = 0x80
    cache = lb.KVCache8(k.clone(), v.clone(), ks.clone(), vs.clone())
    lb.compact_kv(cache, t, lb.StepPlan(starts, granted, lens), ints(path), ints(counts))
    for was, scale, now, scale_now in ((k, ks, cache.k, cache.k_scale), (v, vs, cache.v, cache.v_scale)):
        values, s = was.cpu().double(), scale.cpu().double()
        D.compact_reference(values, s, table, starts.tolist(), granted.tolist(), lens.tolist(), path, counts)
        same = (now.cpu().double() == values) | (now.cpu().double().isnan() & values.isnan())
        assert bool(same.all()), same.logical_not().nonzero()[:5].tolist()
        assert torch.equal(scale_now.cpu().double(), s)


def random_paths(new, rng):
    path, counts = [], []
    for n in new:
        keep = sorted({0, *(i for i in range(n) if rng.random() < rng.choice([0.1, 0.5, 0.9]))}) if n else []
        path += keep + [-1] * (n - len(keep))
        counts.append(len(keep))
    return path, counts


@pytest.mark.parametrize("ctx,new,heads,bs,dim", [
    ([0], [1], 1, 16, 64), ([700], [6], 2, 16, 64), ([15, 16, 17, 0, 31], [9, 40, 64, 33, 3], 3, 16, 128), ([5, 100], [64, 500], 2, 32, 128),
    ([30, 1], [20, 70], 1, 64, 256), ([9, 250], [30, 30], 2, 256, 8), ([3, 40], [17, 50], 2, 16, 80), ([8] * 90, [i % 7 for i in range(90)], 1, 16, 64)])
def test_compact_matches_block_by_block(ctx, new, heads, bs, dim):
    rng = random.Random(dim)
    for seed in range(3):
        rows = U.make_rows(ctx, new, bs, seed=seed)
        check_compact(rows, heads, bs, dim, *random_paths(new, rng), seed=seed, nan=seed == 2)


def test_compact_scales_and_odd_paths():
    rng = random.Random(1)
    rows = U.make_rows([20, 7], [40, 30], 16, seed=3)
    # scales far apart (codes become small ones of few bits, or 0), and no powers of two
    check_compact(rows, 2, 16, 64, *random_paths([40, 30], rng), seed=1, scales=lambda s: torch.exp2(torch.randint(-20, 3, s.shape, generator=gen(4), device=DEV).float()))
    check_compact(rows, 2, 16, 64, *random_paths([40, 30], rng), seed=2, scales=lambda s: s * (torch.rand(s.shape, generator=gen(5), device=DEV) + 0.5))
    # entries that are no later token stay; the same token twice; all, none and too many accepted
    path = [0, 39, 39, 1, -4, 5, 70, 10 ** 9, 12, 12] + [-1] * 30 + list(range(30))
    for counts in ([10, 30], [0, 1], [40, 10 ** 6], [-3, 2]):
        check_compact(rows, 2, 16, 64, path, counts, seed=6)
    # refused rows, numbers that do not fit, blocks that are none
    table, t, starts, granted, lens, blocks = rows
    path, counts = random_paths([40, 30], rng)
    for g, ln in (([0, 30], [20, 37]), ([61, 30], [60, 37]), ([40, 30], [60, 10 ** 6]), ([40, 31], [60, 38])):
        check_compact((table, t, starts, ints(g), ints(ln), blocks), 2, 16, 64, path, counts, seed=7)
    for b, j, wrong in ((0, 1, -1), (0, 2, 10 ** 9), (1, 0, blocks), (1, 1, -1)):
        line = [list(r) for r in table]
        line[b][j] = wrong
        check_compact((line, ints(line), starts, granted, lens, blocks), 2, 16, 64, path, counts, seed=8)


# ---------------------------------------------------------------------------------- shared blocks
def make_table(lens, bs, blocks, rng, spare_width=0):
    ids = rng.sample(range(blocks), blocks)
    width = max([1] + [-(-ln // bs) for ln in lens]) + spare_width
    table = []
    for ln in lens:
        n = -(-ln // bs)
        table.append([ids.pop() for _ in range(n)] + [-1] * (width - n))
    return table, ids


@pytest.mark.parametrize("rows,n,bs,hi,spare", [(1, 3, 16, 1001, 20), (5, 9, 16, 100, 3), (40, 600, 16, 300, 350), (3, 2500, 4, 20, 1000), (60, 61, 256, 9000, 0), (2000, 5000, 16, 40, 3000)])
def test_fork_matches_one_after_the_other(rows, n, bs, hi, spare):
    for seed in range(2):
        rng = random.Random(seed)
        B = rows + n
        lens = [rng.randrange(hi + 1) for _ in range(rows)] + [0] * n
        blocks = sum(-(-ln // bs) for ln in lens) + spare + 1
        table, left = make_table(lens, bs, blocks, rng, 1)
        free = left + [0] * (blocks - len(left))
        src, dst = [rng.randrange(rows) for _ in range(n)], [rows + i for i in range(n)]
        rng.shuffle(dst)
        upto = [rng.choice([hi, rng.randrange(hi + 2), 10 ** 9]) for _ in range(n)] if seed else None
        if seed:  # rows outside, destinations twice, not idle, the source itself
            for i, (s, d) in zip(rng.sample(range(n), min(n, 6)), ((-1, dst[0]), (B, dst[0]), (0, -2), (0, B), (0, dst[-1]), (0, 0))):
                src[i], dst[i] = s, d
        shares = [rng.randrange(3) for _ in range(blocks)]
        t, sh = ints(table), ints(shares)
        f = lb.fork_blocks(t, ints(lens), ints(src), ints(dst), sh, ints(free), ints([len(left)]), bs, upto=None if upto is None else ints(upto))
        want, table2, shares2 = D.fork_reference(table, lens, src, dst, upto, shares, free, len(left), bs)
        assert {k: getattr(f, k).tolist() for k in want} == want
        assert t.tolist() == table2 and sh.tolist() == shares2
        # in place, and a table with rows further apart
        wide = torch.full((B, len(table[0]) + 3), -9, dtype=torch.int32, device=DEV)
        wide[:, : len(table[0])] = ints(table)
        sh, ln, nf = ints(shares), ints(lens), ints([len(left)])
        f = lb.fork_blocks(wide[:, : len(table[0])], ln, ints(src), ints(dst), sh, ints(free), nf, bs, upto=None if upto is None else ints(upto), lens_out=ln, n_free_out=nf)
        assert f.lens is ln and ln.tolist() == want["lens"] and nf.tolist() == want["n_free"] and sh.tolist() == shares2
        assert wide[:, : len(table[0])].tolist() == table2 and bool((wide[:, len(table[0]):] == -9).all())


@pytest.mark.parametrize("heads,bs,dim,n", [(1, 16, 8, 1), (2, 16, 64, 3), (8, 16, 128, 70), (3, 256, 256, 2), (1, 32, 72, 5)])
def test_copy_blocks(heads, bs, dim, n):
    blocks = 2 * n + 3
    cache = lb.KVCache8(*U.random_cache(blocks, heads, bs, dim))
    ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(n)).tolist()
    copies = [[ids[0 if i % 3 == 0 else i], ids[n + i]] for i in range(n)] + [[-1, -1], [blocks, ids[0]], [ids[0], -5], [ids[0], blocks + 7], [ids[0], ids[0]]]
    want = [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    for a, b in copies[:n]:
        for x in want:
            x.view(torch.uint8)[b] = x.view(torch.uint8)[a]
    lb.copy_blocks(cache, ints(copies))
    for x, y in zip(want, (cache.k, cache.v, cache.k_scale, cache.v_scale)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    lb.copy_blocks(cache, ints([]).view(0, 2))
    for bad in (ints(copies).flatten(), ints(copies).long(), ints(copies)[:, :1]):
        with pytest.raises(ValueError):
            lb.copy_blocks(cache, bad)


@pytest.mark.parametrize("rows,bs,hi", [(1, 16, 0), (1, 16, 700), (7, 16, 100), (300, 16, 900), (3000, 4, 60), (40, 32, 20000)])
def test_release_shared_and_kept(rows, bs, hi):
    for seed in range(3):
        rng = random.Random(seed)
        lens = [rng.randrange(hi + 1) for _ in range(rows)]
        blocks = sum(-(-ln // bs) for ln in lens) + 40
        table, left = make_table(lens, bs, blocks, rng)
        shares = [0] * blocks
        for b in range(1, rows):  # rows that hold the beginning of others
            if rng.random() < 0.6:
                a = rng.randrange(b)
                for j in range(min(lens[a], lens[b]) // bs):
                    if table[b][j] != table[a][j]:
                        left.append(table[b][j])
                        table[b][j] = table[a][j]
        holders = {}
        for b in range(rows):
            for j in range(-(-lens[b] // bs)):
                holders[table[b][j]] = holders.get(table[b][j], 0) + 1
        left = [i for i in range(blocks) if i not in holders]
        rng.shuffle(left)
        for i, h in holders.items():
            shares[i] = h - 1 - (seed == 2 and h > 1 and rng.random() < 0.2)  # now and then one holder too many gives it back: once is what counts
        free = left + [0] * (blocks - len(left))
        codes = [int(rng.random() < 0.4) * 2 for _ in range(rows)]
        keep = [rng.choice([ln, max(0, ln - rng.randrange(60)), -3, ln + 5]) for ln in lens]
        if seed == 1 and hi:  # entries that are no blocks
            table[0][0] = 10 ** 9
            table[-1][-1] = -1
        for kp, sh in ((keep, shares), (None, shares), (keep, None)):
            if sh is None:
                line, _ = make_table(lens, bs, blocks, rng)
            else:
                line = table
            fr, s = ints(free), None if sh is None else ints(sh)
            got = lb.release_blocks(ints(line), ints(lens), ints(codes), fr, ints([len(left)]), bs, keep=None if kp is None else ints(kp), shares=s)
            want = D.give_reference(line, lens, codes, kp, sh, free, len(left), bs)
            assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
            assert fr.tolist()[: want[1][0]] == want[2][: want[1][0]] and fr.tolist() == want[2]
            assert s is None or s.tolist() == want[3]
            ln, nf, fr2, s2 = ints(lens), ints([len(left)]), ints(free), None if sh is None else ints(sh)
            lb.release_blocks(ints(line), ln, ints(codes), fr2, nf, bs, lens_out=ln, n_free_out=nf, keep=None if kp is None else ints(kp), shares=s2)
            assert ln.tolist() == want[0] and nf.tolist() == want[1] and torch.equal(fr, fr2)
        # nobody shares, everything kept: the release that was there before
        line, _ = make_table(lens, bs, blocks, rng)
        a, b = ints(free), ints(free)
        want = lb.release_blocks(ints(line), ints(lens), ints(codes), a, ints([len(left)]), bs)
        got = lb.release_blocks(ints(line), ints(lens), ints(codes), b, ints([len(left)]), bs, shares=torch.zeros(blocks, dtype=torch.int32, device=DEV))
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1]) and torch.equal(a, b)


def test_state_refusals():
    table, one, two = ints([[0, 1], [2, 3]]), ints([1]), ints([1, 1])
    for bad in (dict(keep=one), dict(keep=two.long()), dict(shares=one), dict(shares=ints([0] * 8).cpu())):
        with pytest.raises(ValueError):
            lb.release_blocks(table, two, two, ints([0] * 8), one, 16, **bad)
    good = dict(block_table=table, lens=two, src_rows=one, dst_rows=one, shares=ints([0] * 8), free_blocks=ints([0] * 8), n_free=one, block_size=16)
    for bad in (dict(lens=one), dict(dst_rows=two), dict(src_rows=one.long()), dict(shares=one), dict(n_free=two), dict(upto=two), dict(lens_out=one), dict(n_free_out=two),
                dict(free_blocks=ints([]))):
        with pytest.raises(ValueError):
            lb.fork_blocks(**{**good, **bad})
    plan, cache = lb.StepPlan(ints([0, 1, 2]), two, two), lb.KVCache8.empty(8, 1, 16, 64, device=DEV)
    for bad in (dict(path=two.long()), dict(counts=one)):
        with pytest.raises(ValueError):
            lb.compact_kv(cache, table, plan, **{**dict(path=two, counts=two), **bad})
    with pytest.raises(ValueError):
        lb.plan_tree(plan, two.long())
    tree = lb.plan_tree(plan, two)
    for bad in (dict(tokens=one), dict(targets=two.long()), dict(codes=one), dict(given=one), dict(lens_out=one)):
        with pytest.raises(ValueError):
            lb.accept_drafts(plan, tree, **{**dict(tokens=two, targets=two), **bad})


# ------------------------------------------------------------------------- steps with drafted tokens
class Toy:
    """One layer of attention with tied random embeddings: the next token is the largest of W o.  Its state lies in a
    paged cache; a step takes drafted tokens with their trees."""
    HEADS, PER, DIM, BS, VOCAB = 2, 2, 64, 16, 40

    def __init__(self, rows, blocks, width, seed):
        g = gen(seed)
        q, k = self.HEADS * self.PER * self.DIM, self.HEADS * self.DIM
        self.embed = torch.randn(self.VOCAB, q + 2 * k, generator=g, device=DEV).half()
        self.head = torch.randn(q, self.VOCAB, generator=g, device=DEV)
        self.weights = [(1 + 0.2 * torch.randn(self.DIM, generator=g, device=DEV)).half() for _ in range(2)]
        self.freqs = (100.0 ** (-torch.arange(0, self.DIM, 2, device=DEV, dtype=torch.float64) / self.DIM)).float()
        self.cache = lb.KVCache8.empty(blocks, self.HEADS, self.BS, self.DIM, device=DEV)
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=DEV)
        self.free, self.n_free = torch.arange(blocks, dtype=torch.int32, device=DEV), ints([blocks])

    def step(self, new, tokens, parents, given, eos=-1):
        T, q, k = tokens.numel(), self.HEADS * self.PER * self.DIM, self.HEADS * self.DIM
        plan = lb.plan_blocks(self.table, self.lens, new, self.free, self.n_free, self.BS, T, lens_out=self.lens, n_free_out=self.n_free)
        tree = lb.plan_tree(plan, parents)
        x = self.embed[tokens.long()]
        queries, keys, values = (y.unflatten(1, (-1, self.DIM)) for y in x.split((q, k, k), 1))
        queries, keys = lb.norm_rotate(queries, keys, tree.positions, self.freqs, q_weight=self.weights[0], k_weight=self.weights[1])
        lb.append_kv(self.cache, keys, values, self.table, plan)
        o = lb.attend(queries, self.cache, self.table, plan, tree=tree)
        logits = o.flatten(1).float() @ self.head
        targets = logits.argmax(-1).int()
        a = lb.accept_drafts(plan, tree, tokens, targets, codes=(targets == eos).int(), given=given)
        lb.compact_kv(self.cache, self.table, plan, a.path, a.counts)
        lb.release_blocks(self.table, self.lens, a.codes, self.free, self.n_free, self.BS, lens_out=self.lens, n_free_out=self.n_free, keep=a.lens)
        top = logits.topk(2).values
        return a, top[:, 0] - top[:, 1]


def prompt_step(toy, prompts):
    tokens = ints([t for p in prompts for t in p])
    return toy.step(ints([len(p) for p in prompts]), tokens, ints([i - 1 for p in prompts for i in range(len(p))]), ints([len(p) for p in prompts]))


def test_drafted_steps_give_the_tokens_of_single_ones():
    """Whatever is drafted, the tokens are those of sampling one by one.  The two ways round differently: f16 results of about
    0.35 with errors of up to 2^-11 of that, so some 2e-4 between the two, in 256 terms 0.0032 of a logit; where the two
    largest logits are less than six times that (0.02) apart, the token, and the row behind it, is not decided."""
    rng = random.Random(11)
    prompts = [[rng.randrange(40) for _ in range(n)] for n in (5, 16, 31)]
    want_n = 40
    one = Toy(3, 40, 8, seed=4)
    a, gap = prompt_step(one, prompts)
    truth, decided = [[t] for t in a.last.tolist()], [None] * 3
    for _ in range(want_n):
        a, gap = one.step(ints([1, 1, 1]), ints([t[-1] for t in truth]), ints([-1, -1, -1]), None)
        for b, t in enumerate(a.last.tolist()):
            if float(gap[b]) < 0.02 and decided[b] is None:
                decided[b] = len(truth[b])
            truth[b].append(t)
    toy = Toy(3, 40, 8, seed=4)
    a, _ = prompt_step(toy, prompts)
    got, steps = [[t] for t in a.last.tolist()], 0
    while min(len(t) for t in got) < want_n:
        new, tokens, parents = [], [], []
        for b, t in enumerate(got):
            n = rng.choice([1, 4, 9, 20])
            tree = D.random_tree(n, rng, chain=0.6, root=0.0)
            node = [t[-1]]
            depth = [0]
            for i in range(1, n):  # what would really come, or anything
                depth.append(depth[tree[i]] + 1)
                at = len(t) - 1 + depth[i]
                node.append(truth[b][at] if at < len(truth[b]) and rng.random() < 0.8 else rng.randrange(40))
            new.append(n)
            tokens += node
            parents += tree
        a, _ = toy.step(ints(new), ints(tokens), ints(parents), None)
        said, at = a.tokens.tolist(), 0
        for b, n in enumerate(new):
            out = [x for x in said[at: at + n] if x >= 0]
            assert len(out) == a.counts[b] and out[-1] == a.last[b]
            got[b] += out
            at += n
        steps += 1
        held = int(((toy.lens + 15) // 16).sum())
        assert int(toy.n_free) + held == 40
        assert toy.lens.tolist() == [len(p) + len(t) - 1 for p, t in zip(prompts, got)]
    decided = [want_n if n is None else min(n, want_n) for n in decided]
    assert sum(decided) >= 60
    for b, n in enumerate(decided):
        assert got[b][:n] == truth[b][:n]
    assert steps < 30  # several tokens a step


def test_drafted_step_captured_and_replayed():
    rng = random.Random(3)
    prompts = [[rng.randrange(40) for _ in range(n)] for n in (20, 7)]
    drafts = [[rng.randrange(40) for _ in range(12)] for _ in range(4)]
    parents, new = ints([-1, 0, 0, 1, 1, 2, -1, 0, 1, 1, 3, 0]), ints([6, 6])
    results = []
    for captured in (False, True):
        toy = Toy(2, 20, 8, seed=9)
        prompt_step(toy, prompts)
        tokens = torch.zeros(12, dtype=torch.int32, device=DEV)
        if captured:
            state = [x.clone() for x in (toy.table, toy.lens, toy.free, toy.n_free, toy.cache.k.view(torch.uint8), toy.cache.v.view(torch.uint8), toy.cache.k_scale, toy.cache.v_scale)]
            toy.step(new, tokens, parents, None)
            for x, y in zip((toy.table, toy.lens, toy.free, toy.n_free, toy.cache.k.view(torch.uint8), toy.cache.v.view(torch.uint8), toy.cache.k_scale, toy.cache.v_scale), state):
                x.copy_(y)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                a, _ = toy.step(new, tokens, parents, None)
        out = []
        for d in drafts:
            tokens.copy_(ints(d))
            if captured:
                graph.replay()
            else:
                a, _ = toy.step(new, tokens, parents, None)
            out += [x.clone() for x in (a.path, a.tokens, a.counts, a.lens, a.last, toy.lens, toy.n_free, toy.free, toy.table, toy.cache.k.view(torch.uint8), toy.cache.v_scale)]
        results.append(out)
    for x, y in zip(*results):
        assert torch.equal(x, y)


def test_samples_of_a_prompt_share_its_blocks():
    """Samples that fork a prompt go on as rows that have it for themselves; their blocks all come back."""
    rng = random.Random(5)
    prompt = [rng.randrange(40) for _ in range(37)]
    toys = [Toy(4, 30, 8, seed=2) for _ in range(2)]
    first = [[rng.randrange(40) for _ in range(4)] for _ in range(6)]
    shares = torch.zeros(30, dtype=torch.int32, device=DEV)
    shared, alone = toys
    prompt_step(shared, [prompt, [], [], []])
    f = lb.fork_blocks(shared.table, shared.lens, ints([0, 0, 0]), ints([1, 2, 3]), shares, shared.free, shared.n_free, 16, upto=ints([37, 37, 32]),
                       lens_out=shared.lens, n_free_out=shared.n_free)
    lb.copy_blocks(shared.cache, f.copies)
    assert f.granted.tolist() == [37, 37, 32] and shared.n_free.tolist() == [30 - 3 - 2] and int(shares.sum()) == 6
    prompt_step(alone, [prompt, prompt, prompt, prompt[:32]])
    for tokens in first:
        outs = []
        for toy in toys:
            plan = lb.plan_blocks(toy.table, toy.lens, ints([1] * 4), toy.free, toy.n_free, 16, 4, lens_out=toy.lens, n_free_out=toy.n_free)
            x = toy.embed[torch.tensor(tokens, device=DEV)]
            q, k, v = (y.unflatten(1, (-1, 64)) for y in x.split((256, 128, 128), 1))
            lb.append_kv(toy.cache, k, v, toy.table, plan)
            outs.append(lb.attend(q, toy.cache, toy.table, plan))
        assert torch.equal(*outs)
    lb.release_blocks(shared.table, shared.lens, ints([1, 0, 1, 0]), shared.free, shared.n_free, 16, lens_out=shared.lens, n_free_out=shared.n_free, shares=shares)
    assert int(shares.sum()) == 2
    lb.release_blocks(shared.table, shared.lens, ints([0, 1, 0, 1]), shared.free, shared.n_free, 16, lens_out=shared.lens, n_free_out=shared.n_free, shares=shares)
    assert int(shares.sum()) == 0 and shared.n_free.tolist() == [30] and sorted(shared.free.tolist()) == list(range(30)) and shared.lens.tolist() == [0] * 4


def test_two_streams_and_another_order():
    """Calls on two streams at once, each with what it works on."""
    rows, parents = tree_rows([3000, 900, 10], [40, 64, 9], 16, 3)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 8, 16, 128))
    plan = lb.StepPlan(*rows[2:5])
    q = [torch.randn(113, 32, 128, generator=gen(i), device=DEV).bfloat16() for i in range(2)]
    tree = lb.plan_tree(plan, ints(parents))
    pos = ints(list(range(113)))
    freqs = torch.rand(64, generator=gen(1), device=DEV)
    want = [(lb.attend(x, cache, rows[1], plan, tree=tree), *lb.norm_rotate(x, x[:, :8], pos, freqs)) for x in q]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((lb.attend(q[i], cache, rows[1], plan, tree=tree), *lb.norm_rotate(q[i], q[i][:, :8], pos, freqs)))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))
