"""Operators around drafted tokens and shared blocks on the GPU: orders of work, layouts and states beside those of
test_gpu_drafts.py."""
import random

import pytest
import torch

import localstrm_b200 as lb
from tests import decode_util as U
from tests import drafts_util as D
from tests.test_gpu_drafts import DEV, check_attend_tree, check_rotate, gen, ints, make_table, rotate_case

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


# ------------------------------------------------------------------------------ norms and rotation
@pytest.mark.parametrize("T,heads,dim,off", [(1, 3, 64, 0), (37, 6, 128, 0), (37, 6, 128, 1), (200, 1, 80, 0), (5, 64, 66, 0)])
def test_rotate_heads_in_turn(T, heads, dim, off):
    """Queries, keys and values of each head beside each other, token by token and head by head: in place, and from two of
    the places into two others; what lies between stays."""
    _, _, pos, freqs, qw, kw = rotate_case(T, 1, 1, dim, dim - dim % 4, torch.bfloat16, T)
    n = T * heads * 4 * dim
    for order in (lambda x: x.view(T, heads, 4, dim), lambda x: x.view(heads, 4, T, dim).permute(2, 0, 1, 3)):
        flat = torch.randn(off + n + 3, generator=gen(dim), device=DEV).bfloat16()
        four = order(flat[off: off + n])
        want = check_rotate(four[:, :, 0], four[:, :, 1], pos, freqs, qw, kw, False)
        before = flat.clone()
        lb.norm_rotate(four[:, :, 0], four[:, :, 1], pos, freqs, qw, kw, q_out=four[:, :, 2], k_out=four[:, :, 3])
        expect = before.clone()
        order(expect[off: off + n])[:, :, 2], order(expect[off: off + n])[:, :, 3] = want
        assert torch.equal(flat, expect)
        lb.norm_rotate(four[:, :, 0], four[:, :, 1], pos, freqs, qw, kw, q_out=four[:, :, 0], k_out=four[:, :, 1])
        order(expect[off: off + n])[:, :, 0], order(expect[off: off + n])[:, :, 1] = want
        assert torch.equal(flat, expect)
        for bad in (dict(q_out=four[:, :, 1]), dict(k_out=four[:, :, 0]), dict(q_out=four[:, :, 2], k_out=four[:, :, 2])):
            with pytest.raises(lb.SamplerError):
                lb.norm_rotate(four[:, :, 0], four[:, :, 1], pos, freqs, **bad)
        assert torch.equal(flat, expect)


def test_rotate_in_place_leaves_what_lies_around():
    """Slices of a fused projection that do not begin on 16 bytes: what lies in front of the queries and behind the keys."""
    T, hq, hk, dim = 37, 6, 2, 128
    _, _, pos, freqs, qw, kw = rotate_case(T, hq, hk, dim, dim, torch.bfloat16, 5)
    for off in (0, 1, 5):
        fused = torch.randn(T, 1400, generator=gen(6), device=DEV).bfloat16()
        before, end = fused.clone(), off + (hq + hk) * dim
        q, k = fused[:, off: off + hq * dim].view(T, hq, dim), fused[:, off + hq * dim: end].view(T, hk, dim)
        check_rotate(q, k, pos, freqs, qw, kw, False, q_out=q, k_out=k)
        assert torch.equal(fused[:, :off], before[:, :off]) and torch.equal(fused[:, end:], before[:, end:])


# --------------------------------------------------------------------------------------- attention
def lagging(rows, new, heads, per, dim, seed):
    """A cache and queries with which the two halves of a group of 256 query rows take different times: the scores of the
    first half grow by some 12 (powers of two) every 64 tokens, so that its sums are rescaled at every step, those of the
    second half hardly differ.  The largest scores are about 60: f32 holds them, and the sums of 16 products at a time that
    lead to them, to 2^-18, a 2^-18 of the weight, well below the quarter of 2^-11 left for it."""
    table, _, _, _, lens, blocks = rows
    bs = 16
    k, v, ks, vs = U.random_cache(blocks, heads, bs, dim, seed=seed)
    ks.fill_(2.0 ** -7)
    for line, ln in zip(table, lens.tolist()):
        pages = torch.tensor(line[: -(-ln // bs)], device=DEV)
        grow = (torch.arange(len(pages) * bs, device=DEV).view(-1, bs) * (448 / 320)).clamp(max=448).to(U.E4M3)
        k.view(torch.uint8)[pages, :, :, 0] = grow.view(torch.uint8)[:, None]
    q = torch.randn(sum(new), heads * per, dim, generator=gen(seed), device=DEV)
    at = torch.cat([torch.arange(n * per, device=DEV) for n in new]).view(-1, per)  # row of the queries of one key head
    big = 12 / 64 * 320 / 448 * 2 ** 7 / 1.4427 * dim ** 0.5
    q.view(-1, heads, per, dim)[..., 0] = torch.where(at % 256 < 128, big, 0.0)[:, None]
    return lb.KVCache8(k, v, ks, vs), q.bfloat16()


MIXED = {
    "prompts of 200 tokens": ([0] * 40, [200] * 40),
    "prompts of 90 and 150": ([0] * 60, [90, 150] * 30),
    "chunks of one step beside small trees": ([0, 3] * 60, [33 + i % 32 if i % 2 == 0 else 8 + i % 25 for i in range(120)]),
    "all lengths": ([0] * 70, [33 + (i * 97) % 268 if i % 3 else 8 + i % 25 for i in range(70)]),
}


@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("name", MIXED)
def test_attend_small_groups_between_whole_ones(name, dim):
    """Groups of up to 128 query rows, for which the two streams of the tensor-memory kernel work together, between
    groups of 256 of one and two steps, which they take on their own: neither may run into the other's queries."""
    ctx, new = MIXED[name]
    heads, per = 8, 4
    rows = U.make_rows(ctx, new, 16, seed=dim)
    cache, q = lagging(rows, new, heads, per, dim, seed=len(new))
    parents = [p for i, n in enumerate(new) for p in D.random_tree(n, random.Random(i), root=0.0)]
    plan = lb.StepPlan(*rows[2:5])
    y, lse = check_attend_tree(q, cache, rows, parents)
    tree = lb.plan_tree(plan, ints(parents))
    want, mag, _ = U.attend_reference(q, cache.k, cache.v, cache.k_scale, cache.v_scale, rows[0], *(x.tolist() for x in rows[2:5]), dim ** -0.5)
    causal = lb.attend(q, cache, rows[1], plan)
    assert bool(((causal.double() - want).abs() <= 1.25 * 2.0 ** -11 * mag + 2.0 ** -8 * want.abs()).all())
    busy, side = torch.zeros(1 << 24, device=DEV), torch.cuda.Stream()
    for i in range(12):  # the same in every bit, with other work beside it too
        if i % 2:
            with torch.cuda.stream(side):
                busy.add_(1)
        assert torch.equal(lb.attend(q, cache, rows[1], plan, tree=tree), y) and torch.equal(lb.attend(q, cache, rows[1], plan), causal)
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------------- shared blocks
@pytest.mark.parametrize("rows,hi", [(33, 200), (64, 4000), (511, 900), (512, 9000), (5000, 60), (16384, 20)])
def test_release_kept_without_shares(rows, hi):
    """Blocks of rejected tokens where no block is shared: clusters of 2 to 16 CTAs that write to each other's shared memory
    from their first pass on, with other work on the SMs, so that they do not all begin at once; captured too."""
    rng = random.Random(rows)
    bs = 16
    lens = [rng.randrange(hi + 1) for _ in range(rows)]
    blocks = sum(-(-ln // bs) for ln in lens) + 7
    table, left = make_table(lens, bs, blocks, rng)
    free = left + [0] * (blocks - len(left))
    codes = [int(rng.random() < 0.3) for _ in lens]
    keep = [max(0, ln - rng.randrange(40)) for ln in lens]
    want = D.give_reference(table, lens, codes, keep, None, free, len(left), bs)
    line, ln, cd, kp, fr0, nf = ints(table), ints(lens), ints(codes), ints(keep), ints(free), ints([len(left)])
    x, side = torch.randn(2048, 2048, device=DEV), torch.cuda.Stream()

    def give():
        fr = fr0.clone()
        return (*lb.release_blocks(line, ln, cd, fr, nf, bs, keep=kp), fr)

    got = [give()]
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(side):
            x @ x
        got.append(give())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = give()
    for _ in range(3):
        graph.replay()
    for lens_out, n_free, fr in got + [again]:
        assert lens_out.tolist() == want[0] and n_free.tolist() == want[1] and fr.tolist() == want[2]


def test_rows_cut_inside_shared_blocks():
    """A row that is to go on from the middle of a block that another one holds is forked and released: what it writes then
    is its own, and the other's block stays as it is in every bit."""
    heads, bs, dim = 2, 16, 64
    cache = lb.KVCache8(*U.random_cache(12, heads, bs, dim))
    table, lens = ints([[3, 5, 7], [-1] * 3, [-1] * 3]), ints([40, 0, 0])
    free, n_free, shares = ints([8, 9, 10, 11, 0, 1, 2, 4, 6, 0, 0, 0]), ints([9]), ints([0] * 12)
    fork = lambda src, dst, upto: lb.fork_blocks(table, lens, ints([src]), ints([dst]), shares, free, n_free, bs, upto=ints([upto]), lens_out=lens, n_free_out=n_free)
    lb.copy_blocks(cache, fork(0, 1, 40).copies)
    lb.copy_blocks(cache, fork(1, 2, 20).copies)  # row 1 cut to 20 tokens: inside block 5, which row 0 holds
    lb.release_blocks(table, lens, ints([0, 1, 0]), free, n_free, bs, lens_out=lens, n_free_out=n_free, shares=shares)
    assert lens.tolist() == [40, 0, 20] and shares.tolist() == [0, 0, 0, 1] + [0] * 8 and n_free.tolist() == [8]
    before = [x[[3, 5, 7]].clone() for x in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    assert torch.equal(cache.k.view(torch.uint8)[table[2, 1].item()], cache.k.view(torch.uint8)[5])
    plan = lb.plan_blocks(table, lens, ints([0, 0, 5]), free, n_free, bs, 5, lens_out=lens, n_free_out=n_free)
    x = 1e4 * torch.randn(5, heads, dim, generator=gen(1), device=DEV)
    lb.append_kv(cache, x, x, table, plan)
    for was, now in zip(before, (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)):
        assert torch.equal(was, now[[3, 5, 7]])
    lb.release_blocks(table, lens, ints([1, 0, 1]), free, n_free, bs, lens_out=lens, n_free_out=n_free, shares=shares)
    assert n_free.tolist() == [12] and sorted(free.tolist()) == list(range(12)) and shares.tolist() == [0] * 12


# --------------------------------------------------------------------------- accepted tokens move up
@pytest.mark.parametrize("zeros", ["all", "some"])
def test_compact_scales_of_zero(zeros):
    """A caller's own cache may hold blocks whose scales are 0: codes move as they are where all of a block's tokens come
    from such ones, and become 0 beside others."""
    rows = U.make_rows([20, 7, 3], [40, 30, 9], 16, seed=5)
    table, t, starts, granted, lens, blocks = rows
    k, v, ks, vs = U.random_cache(blocks, 2, 16, 64, seed=1)
    for s in (ks, vs):
        s[torch.rand(s.shape, generator=gen(2), device=DEV) < (2.0 if zeros == "all" else 0.4)] = 0.0
    cache = lb.KVCache8(k.clone(), v.clone(), ks.clone(), vs.clone())
    path, counts = [], []
    for n in (40, 30, 9):
        kept = sorted({0, *random.Random(n).sample(range(n), n // 2)})
        path += kept + [-1] * (n - len(kept))
        counts.append(len(kept))
    lb.compact_kv(cache, t, lb.StepPlan(starts, granted, lens), ints(path), ints(counts))
    for was, scale, now, scale_now in ((k, ks, cache.k, cache.k_scale), (v, vs, cache.v, cache.v_scale)):
        one = torch.where(scale == 0, 2.0 ** -200, scale.double()).cpu()  # so far below the others that codes beside them become 0
        values, s = was.cpu().double(), one.clone()
        D.compact_reference(values, s, table, starts.tolist(), granted.tolist(), lens.tolist(), path, counts)
        assert torch.equal(now.cpu().double(), values)
        assert torch.equal(scale_now.cpu().double(), torch.where(s == 2.0 ** -200, 0.0, s))


# ------------------------------------------------------------------------- drafted tokens and the sampler
def node_histories(histories, new, tokens, parents):
    out, first = [], 0
    for history, n in zip(histories, new):
        line = []
        for i in range(n):
            p = parents[first + i]
            line.append((line[p] if p >= 0 else list(history)) + [tokens[first + i]])
        out += line
        first += n
    return out


def test_drafts_sampled_with_penalties():
    """Each drafted token's target with the history of its own branch, by the framework's sampler: the tokens are those of
    sampling one by one, with the same logits behind the same tokens and the same random number at the same place."""
    vocab, rows, steps = 300, 4, 30
    logits = 2 * torch.randn(vocab, vocab, generator=gen(1), device=DEV)  # behind each token
    uniforms = torch.rand(rows, 200, generator=gen(2), device=DEV)
    params = [lb.SamplingParams(temperature=t, top_k=k, top_p=0.95, repetition_penalty=r, frequency_penalty=f, presence_penalty=p)
              for t, k, r, f, p in ((0.8, 20, 1.3, 0.0, 0.0), (0.0, -1, 1.5, 0.2, 0.1), (1.1, 5, 1.0, 0.5, 0.3), (0.7, 40, 1.2, 0.1, 0.0))]
    rng = random.Random(3)
    prompts = [[rng.randrange(vocab) for _ in range(n)] for n in (3, 9, 1, 20)]
    truth = [list(p) for p in prompts]
    for i in range(steps + 40):
        tok = lb.sample_batch(logits[[t[-1] for t in truth]], params, truth, uniforms[:, i].contiguous()).tolist()
        for t, x in zip(truth, tok):
            t.append(x)
    said, lens, drafted = [list(p) for p in prompts], [len(p) - 1 for p in prompts], 0
    while min(len(s) - len(p) for s, p in zip(said, prompts)) < steps:
        new, tokens, parents, place = [], [], [], []
        for b, s in enumerate(said):
            n = rng.choice([1, 3, 8, 14])
            tree, depth = D.random_tree(n, rng, chain=0.6, root=0.0), [0]
            node = [s[-1]]
            for i in range(1, n):  # what will really come, or anything
                depth.append(depth[tree[i]] + 1)
                node.append(truth[b][len(s) - 1 + depth[i]] if rng.random() < 0.8 else rng.randrange(vocab))
            new.append(n)
            tokens += node
            parents += tree
            place += [(b, len(s) - len(prompts[b]) + d) for d in depth]
        B = [b for b, n in enumerate(new) for _ in range(n)]
        targets = lb.sample_batch(logits[tokens], [params[b] for b in B], node_histories([s[:-1] for s in said], new, tokens, parents),
                                  torch.stack([uniforms[at] for at in place]))
        starts = [sum(new[:i]) for i in range(rows + 1)]
        plan = lb.StepPlan(ints(starts), ints(new), ints([ln + n for ln, n in zip(lens, new)]))
        a = lb.accept_drafts(plan, lb.plan_tree(plan, ints(parents)), ints(tokens), targets)
        got, lens = a.tokens.tolist(), a.lens.tolist()
        for b, s in enumerate(said):
            s += [x for x in got[starts[b]: starts[b + 1]] if x >= 0]
            assert s == truth[b][: len(s)] and lens[b] == len(s) - 1
        drafted += 1
    assert drafted < steps  # several tokens a step


def test_drafts_sampled_in_a_captured_step():
    """Sampler with penalties from device arrays, and the acceptance, in one graph: other logits, random numbers, drafts and
    histories with each replay."""
    from localstrm_b200.sampling import build_history_csr
    vocab, new, rng = 500, [5, 1, 9], random.Random(2)
    T = sum(new)
    parents = [p for n in new for p in D.random_tree(n, rng, root=0.0)]
    rp = lb.RowParams.from_params([lb.SamplingParams(temperature=0.9, top_k=30, repetition_penalty=1.4)] * T, DEV)
    plan = lb.StepPlan(ints([0, 5, 6, 15]), ints(new), ints([25, 8, 10]))
    sampler = lb.BatchSampler(DEV)

    def inputs(seed):
        tokens = [random.Random(seed + i).randrange(4) for i in range(T)]  # few, so that branches are followed
        offs, ids = build_history_csr(node_histories([[seed % vocab] * 6, [1, 2], [7]], new, tokens, parents), T, vocab)
        logits = torch.randn(T, vocab, generator=gen(seed), device=DEV)
        logits[:, :4] += 6
        return logits, torch.rand(T, generator=gen(seed), device=DEV), ints(tokens), ints(offs.tolist()), ints(ids.tolist())

    def step(logits, u, tokens, offs, ids):
        tok = sampler.sample(logits, rp, offs, ids, u)
        return tok, lb.accept_drafts(plan, lb.plan_tree(plan, ints_of), tokens, tok)

    ints_of = ints(parents)
    buffers = [x.clone() for x in inputs(0)]
    step(*buffers)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, a = step(*buffers)
    for seed in range(1, 5):
        fresh = inputs(seed)
        for x, y in zip(buffers, fresh):
            x.copy_(y)
        graph.replay()
        got = [x.clone() for x in (tok, a.path, a.tokens, a.counts, a.lens, a.last)]
        want_tok, b = step(*fresh)
        for x, y in zip(got, (want_tok, b.path, b.tokens, b.counts, b.lens, b.last)):
            assert torch.equal(x, y)
        assert D.accept_reference(parents, fresh[2].tolist(), want_tok.tolist(), None, None, [0, 5, 6, 15], new, [25, 8, 10], T)[2] == b.counts.tolist()


# --------------------------------------------------------------------------- shared blocks in one graph
def test_fork_copy_and_release_captured():
    """Forks, the copies of their last blocks and the release of all of them in one graph, replayed from other states, on
    another stream than the one it was captured on."""
    heads, bs, dim, B, blocks = 2, 16, 64, 6, 40
    cache = lb.KVCache8(*U.random_cache(blocks, heads, bs, dim))
    table, lens, n_free, shares = (torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((B, 5), (B,), (1,), (blocks,)))
    free, src, dst, upto, codes = (torch.zeros(s, dtype=torch.int32, device=DEV) for s in (blocks, 3, 3, 3, B))

    def run():
        f = lb.fork_blocks(table, lens, src, dst, shares, free, n_free, bs, upto=upto, lens_out=lens, n_free_out=n_free)
        lb.copy_blocks(cache, f.copies)
        after = [x.clone() for x in (lens, n_free, shares, table, f.granted, f.copies, cache.k.view(torch.uint8), cache.v_scale)]
        lb.release_blocks(table, lens, codes, free, n_free, bs, lens_out=lens, n_free_out=n_free, shares=shares)
        return after + [x.clone() for x in (lens, n_free, free, shares)]

    def start(seed):
        rng = random.Random(seed)
        ids = rng.sample(range(blocks), blocks)
        ln = [rng.randrange(1, 81), rng.randrange(1, 81), rng.randrange(1, 81), 0, 0, 0]
        rows = [[ids.pop() for _ in range(-(-n // bs))] for n in ln]
        left = rng.choice([1, 2, len(ids)])
        for t, v in ((table, [r + [-1] * (5 - len(r)) for r in rows]), (lens, ln), (n_free, [left]), (shares, [0] * blocks), (free, ids[:left] + [0] * (blocks - left)),
                     (src, [rng.randrange(3) for _ in range(3)]), (dst, rng.sample([3, 4, 5], 3)), (upto, [rng.randrange(1, 90) for _ in range(3)]),
                     (codes, [rng.randrange(2) for _ in range(B)])):
            t.copy_(ints(v))
        for x, y in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale), U.random_cache(blocks, heads, bs, dim, seed=seed)):
            x.copy_(y.view(torch.uint8) if y.dtype == U.E4M3 else y)

    start(0)
    run()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        kept = run()
    for seed in range(1, 9):
        start(seed)
        line, ln, left, fr = table.tolist(), lens.tolist(), int(n_free), free.tolist()
        want = [x.clone() for x in run()]
        f, line2, sh2 = D.fork_reference(line, ln, src.tolist(), dst.tolist(), upto.tolist(), [0] * blocks, fr, left, bs)
        assert want[0].tolist() == f["lens"] and want[1].tolist() == f["n_free"] and want[2].tolist() == sh2 and want[3].tolist() == line2
        start(seed)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(x, y) for x, y in zip(kept, want))


# ------------------------------------------------------------------------------ prompts, and long caches
@pytest.mark.parametrize("heads,per,dim", [(8, 4, 128), (2, 7, 64), (2, 3, 256)])
def test_attend_prompt_chunks_beside_trees(heads, per, dim):
    """A chunk of more than 1,024 new tokens is a chain whatever its parents say; trees, a single token, an idle row and a
    refused one in the same step."""
    ctx, new = [3, 700, 2600, 0, 40, 90, 1500], [1100, 20, 9, 1, 0, 33, 300]
    rng = random.Random(dim)
    rows = list(U.make_rows(ctx, new, 16, seed=dim))
    parents = [p for n in new for p in D.random_tree(n, rng)]
    granted, lens = rows[3].clone(), rows[4].clone()
    granted[5], lens[5] = 0, 90  # refused: its tokens stay as they are
    rows[3], rows[4] = granted, lens
    cache = lb.KVCache8(*U.random_cache(rows[-1], heads, 16, dim, seed=per))
    q = torch.randn(sum(new) + 3, heads * per, dim, generator=gen(dim), device=DEV).bfloat16()
    y, _ = check_attend_tree(q, cache, tuple(rows), parents + [-1] * 3)
    at = int(rows[2][5])
    assert bool((y[at: at + 33] == 77).all()) and bool((y[sum(new):] == 77).all()) and bool(y[:at].isfinite().all())
    plan = lb.StepPlan(*rows[2:5])
    tree = lb.plan_tree(plan, ints(parents + [-1] * 3))
    assert tree.positions[:1100].tolist() == list(range(3, 1103)) and tree.positions[at: at + 33].tolist() == [0] * 33


def test_blocks_behind_four_gigabytes():
    """Blocks whose places pass 32 bits: attention, accepted tokens, copies and appended tokens as in a small cache."""
    heads, bs, dim, far = 8, 16, 128, 280_000  # 16 KB a block: 4.6 GB of keys, and of values
    new, ctx = [20, 9, 40, 1], [100, 3000, 35, 17]
    table, t, starts, granted, lens, blocks = U.make_rows(ctx, new, bs, seed=1)
    small = lb.KVCache8(*U.random_cache(blocks, heads, bs, dim, seed=2))
    big = lb.KVCache8(*(torch.empty(far, heads, bs, dim, dtype=torch.uint8, device=DEV).view(U.E4M3) for _ in range(2)),
                      *(torch.ones(far, heads, device=DEV) for _ in range(2)))
    ends = (0, far - blocks)  # low blocks are other ones, so that a place that lost its upper bits shows
    parts = lambda c: (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale)
    for b, s in zip(parts(big), parts(small)):
        b[: blocks] = s.flip(0)
        b[far - blocks:] = s
    assert (far - blocks) * heads * bs * dim > 2 ** 32
    up = torch.where(t >= 0, t + ends[1], t)
    plan, rng = lb.StepPlan(starts, granted, lens), random.Random(4)
    tree = lb.plan_tree(plan, ints([p for n in new for p in D.random_tree(n, rng)]))
    q = torch.randn(sum(new), 32, dim, generator=gen(3), device=DEV).bfloat16()
    kv = torch.randn(2, sum(new), heads, dim, generator=gen(4), device=DEV)
    path, counts = [], []
    for n in new:
        kept = sorted({0, *rng.sample(range(n), n // 2)})
        path += kept + [-1] * (n - len(kept))
        counts.append(len(kept))
    out = []
    for cache, tab, off in ((small, t, 0), (big, up.contiguous(), ends[1])):
        lb.append_kv(cache, kv[0], kv[1], tab, plan)
        o = [lb.attend(q, cache, tab, plan, tree=tree), lb.attend(q, cache, tab, plan)]
        lb.compact_kv(cache, tab, plan, ints(path), ints(counts))
        lb.copy_blocks(cache, ints([[table[1][0] + off, table[2][1] + off], [table[1][5] + off, blocks - 1 + off]]))
        out.append(o + [x[off: off + blocks].clone() for x in parts(cache)])
    assert all(torch.equal(x, y) for x, y in zip(*out))
    assert torch.equal(big.k.view(torch.uint8)[:blocks], U.random_cache(blocks, heads, bs, dim, seed=2)[0].view(torch.uint8).flip(0))
