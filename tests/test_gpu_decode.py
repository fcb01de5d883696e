"""The decode-step operators on the GPU against plain 64-bit forms."""
import math

import pytest
import torch

import localstrm_b200 as lb
from localstrm_b200 import sampling as S
from tests import decode_util as U

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
DEV = torch.device("cuda", 0)
E4M3 = torch.float8_e4m3fn
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------- 4-bit products
def int4_case(rows, n, k, group, seed, scale_dtype=torch.float16):
    g = gen(seed)
    packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=g, device=DEV)
    scales = (0.02 * torch.exp(torch.randn(n, k // group, generator=g, device=DEV))).to(scale_dtype)
    x = torch.randn(rows, k, generator=g, device=DEV)
    return lb.Int4Weight(packed, scales), x


def int4_check(y, x, w):
    """Products of the 16-bit operands are exact in f32; what rounds is the running f32 sums of K / 16
    tensor steps (twice 2^-24 each, they may truncate), the sum over the groups, and the result."""
    wd = torch.stack([w.packed & 15, w.packed >> 4], -1).reshape(w.packed.shape[0], -1).double() - 8
    wd = wd * w.scales.double().repeat_interleave(w.group, 1)
    want, size = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    k = x.shape[-1]
    tol = (3 * k / 16 + 2 * k / w.group + 8) * 2.0 ** -23 * size + torch.finfo(y.dtype).eps / 2 * want.abs() + 2.0 ** -24 * (y.dtype == torch.float16)
    off = (y.double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


@pytest.mark.parametrize("rows,n,k,group", [
    (1, 1, 32, 32), (1, 17, 64, 64), (2, 16, 128, 128), (3, 2057, 896, 64), (8, 33, 160, 32), (9, 515, 256, 256),
    (5, 4099, 1120, 32), (17, 130, 8192, 128), (33, 1000, 512, 128), (64, 771, 4096, 128), (65, 96, 384, 384),
    (1, 151936, 896, 128), (8, 20000, 640, 128)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_int4_sizes(rows, n, k, group, dtype):
    w, x = int4_case(rows, n, k, group, seed=rows * 1000 + n, scale_dtype=torch.bfloat16 if n % 2 else torch.float16)
    x = x.to(DTYPES[dtype])
    int4_check(lb.int4_matvec(x, w), x, w)
    y = lb.int4_matvec(x, w, out_dtype=torch.float32)
    int4_check(y, x, w)
    assert torch.equal(y, lb.int4_matvec(x, w, out_dtype=torch.float32))  # the same sums in the same order


def test_int4_layouts_and_values():
    w, x = int4_case(6, 301, 256, 64, seed=3)
    wide = torch.zeros(6, 700, device=DEV)
    for off in (0, 3):  # a slice of a wider tensor, 16-byte aligned rows and not
        for dt in DTYPES.values():
            xs = wide.to(dt)
            xs[:, off: off + 256] = x.to(dt)
            int4_check(lb.int4_matvec(xs[:, off: off + 256], w), xs[:, off: off + 256], w)
    xt = x.t().contiguous().t()
    int4_check(lb.int4_matvec(xt, w), xt, w)
    out = torch.full((6, 400), 7.0, device=DEV)
    lb.int4_matvec(x, w, out=out[:, 50:351])
    int4_check(out[:, 50:351], x, w)
    assert bool((out[:, :50] == 7).all()) and bool((out[:, 351:] == 7).all())
    int4_check(lb.int4_matvec(x[2], w)[None], x[2:3], w)
    assert lb.int4_matvec(x[:0], w).shape == (0, 301)
    # f32 values of all magnitudes (their three bf16 parts are exact down to 2^-126), bf16 up to its end
    big = x * torch.exp2(torch.randint(-60, 60, (1, 256), generator=gen(5), device=DEV).float())
    int4_check(lb.int4_matvec(big, w), big, w)
    # what is not finite stays in its row
    x[1, 7], x[3, 9] = math.nan, math.inf
    y = lb.int4_matvec(x, w)
    int4_check(y[[0, 2, 4, 5]], x[[0, 2, 4, 5]], w)
    assert bool(y[1].isnan().all()) and not bool(y[3].isfinite().any())


@pytest.mark.parametrize("rows,n,k,dtype", [(1, 200, 20480, "f32"), (3, 5000, 20480, "f32"), (2, 130, 150016, "bf16"), (8, 5000, 51200, "f16")])
def test_int4_long_rows(rows, n, k, dtype):
    """Rows that do not fit the shared memory of an SM, or only when several SMs share them."""
    w, x = int4_case(rows, n, k, 128, seed=rows + k)
    x = x.to(DTYPES[dtype])
    int4_check(lb.int4_matvec(x, w), x, w)


def launches(f):
    """Kernel launches of a call, counted in a graph that captures it."""
    rt = pytest.importorskip("cuda.bindings.runtime")
    g = torch.cuda.CUDAGraph(keep_graph=True)
    f()
    with torch.cuda.graph(g):
        f()
    err, _, n = rt.cudaGraphGetNodes(g.raw_cuda_graph(), 0)
    err, nodes, n = rt.cudaGraphGetNodes(g.raw_cuda_graph(), n)
    return sum(rt.cudaGraphNodeGetType(x)[1] == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for x in nodes[:n])


@pytest.mark.parametrize("rows,n,k,dtype,most", [
    (8, 1000, 14336, "f32", 1), (8, 4096, 14336, "bf16", 1), (3, 4096, 14336, "f32", 1), (4, 1000, 28672, "f16", 1), (2, 2057, 11008, "f32", 1),
    (8, 40000, 8192, "bf16", 3), (8, 40000, 4096, "f32", 3), (5, 40003, 4096, "f32", 3), (2, 40000, 16384, "f32", 3), (7, 40000, 8224, "f16", 3)])
def test_int4_few_rows_read_the_matrix_once(rows, n, k, dtype, most):
    """Two to eight long rows: one launch for all of them, or the operand, the product and the sum of the other kernel."""
    w, x = int4_case(rows, n, k, 32, seed=rows + k)
    x = x.to(DTYPES[dtype])
    int4_check(lb.int4_matvec(x, w), x, w)
    assert launches(lambda: lb.int4_matvec(x, w)) <= most
    # without a workspace of that size, as a C caller may: the same result in more passes
    lib, y = lb._lib.load(), torch.empty(rows, n, device=DEV)
    code = {"f32": 0, "bf16": 1, "f16": 2}
    assert lib.lss_int4_matvec(x.data_ptr(), code[dtype], rows, k, k, w.packed.data_ptr(), w.scales.data_ptr(), 2, n, 32, y.data_ptr(), 0, n, None, 0,
                               torch.cuda.current_stream().cuda_stream) == 0
    int4_check(y, x, w)


@pytest.mark.parametrize("rows,n,k,dtype", [(1, 14336, 4096, "bf16"), (8, 4096, 14336, "bf16"), (8, 4096, 14336, "f32"), (1, 9000, 2048, "f16")])
def test_int4_clusters_run_at_one_time(rows, n, k, dtype):
    """No second wave for a split of the columns: its clusters are all on the device at once."""
    drv = pytest.importorskip("cuda.bindings.driver")
    w, x = int4_case(rows, n, k, 128, seed=n)
    x = x.to(DTYPES[dtype])
    int4_check(lb.int4_matvec(x, w), x, w)
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        lb.int4_matvec(x, w)
    graph = drv.CUgraph(g.raw_cuda_graph())
    _, _, count = drv.cuGraphGetNodes(graph, 0)
    _, (node,), count = drv.cuGraphGetNodes(graph, count)
    assert count == 1
    _, p = drv.cuGraphKernelNodeGetParams(node)
    kind = drv.CUlaunchAttributeID.CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION
    size = max(1, drv.cuGraphKernelNodeGetAttribute(node, kind)[1].clusterDim.x)
    cfg, at = drv.CUlaunchConfig(), drv.CUlaunchAttribute()
    cfg.gridDimX, cfg.blockDimX, cfg.sharedMemBytes = p.gridDimX, p.blockDimX, p.sharedMemBytes
    cfg.gridDimY = cfg.gridDimZ = cfg.blockDimY = cfg.blockDimZ = 1
    at.id, at.value.clusterDim.x, at.value.clusterDim.y, at.value.clusterDim.z = kind, size, 1, 1
    cfg.attrs, cfg.numAttrs = [at], 1
    err, active = drv.cuOccupancyMaxActiveClusters(p.func, cfg)
    assert int(err) == 0 and p.gridDimX // size <= active


@pytest.mark.parametrize("rows,n,k,dtype", [(9, 76000, 512, "bf16"), (64, 76100, 384, "f16"), (20, 76001, 256, "f32"), (16, 100000, 128, "bf16"),
                                            (70, 82000, 640, "bf16"), (33, 151936, 160, "f16")])
def test_int4_waves(rows, n, k, dtype):
    """More row blocks than fit the SMs at a time, with few and many of them left for the last turn."""
    w, x = int4_case(rows, n, k, 32, seed=n)
    x = x.to(DTYPES[dtype])
    y = lb.int4_matvec(x, w, out_dtype=torch.float32)
    int4_check(y, x, w)
    assert torch.equal(y, lb.int4_matvec(x, w, out_dtype=torch.float32))


def test_int4_output_beside_and_over_the_input():
    w, x = int4_case(3, 64, 128, 32, seed=31)
    both = torch.zeros(3, 200, device=DEV)
    both[:, :128] = x
    lb.int4_matvec(both[:, :128], w, out=both[:, 128:192])
    int4_check(both[:, 128:192].contiguous(), x, w)
    for out in (both[:, :64], both[:, 100:164]):
        with pytest.raises((RuntimeError, ValueError)):
            lb.int4_matvec(both[:, :128], w, out=out)
    assert torch.equal(both[:, :128], x)


def test_plan_writes_lengths_over_the_new_ones():
    """65,536 tokens of 4,096 rows: many CTAs, if the state were not written in place."""
    B, bs = 4096, 16
    table = torch.arange(B, dtype=torch.int32, device=DEV).view(B, 1).contiguous()
    lens, free, nf = ints([0] * B), ints(list(range(B))), ints([B])
    for _ in range(20):
        new = ints([16] * B)
        p = lb.plan_blocks(table, lens, new, free, nf, bs, 16 * B, lens_out=new)
        assert p.starts.tolist() == list(range(0, 16 * B + 1, 16)) and bool((new == 16).all()) and bool((p.granted == 16).all())


def test_int4_quantize_and_sample_hidden():
    w = torch.randn(777, 256, generator=gen(9), device=DEV)
    q = lb.Int4Weight.quantize(w, group=64)
    step = q.scales.float().repeat_interleave(64, 1)
    # half a step; the f16 rounding of the scale shifts the largest value (code 7) by 7 * 2^-11 of one
    assert bool(((q.dequantize() - w).abs() <= step * (0.5 + 7 * 2.0 ** -10)).all())
    h = torch.randn(5, 256, generator=gen(10), device=DEV)
    logits = lb.int4_matvec(h, q)
    u = torch.rand(5, generator=gen(11), device=DEV)
    params = [S.SamplingParams(temperature=t, top_k=20, top_p=0.9, repetition_penalty=1.1) for t in (0.0, 0.5, 0.8, 1.0, 1.3)]
    past = [[1, 2, 3], None, [5, 5], [], [700]]
    got = lb.sample_hidden(h, q, params, past, uniforms=u)
    assert torch.equal(got, S.sample_batch(logits, params, past, uniforms=u))
    assert got[0] == logits[0].argmax()


def test_int4_row_slices_and_vocabulary_shards(monkeypatch):
    """Rows of a matrix by themselves (their scales may start on any 16-bit boundary), and the projection in
    front of the vocabulary-sharded sampler."""
    from localstrm_b200 import distributed as D
    w, x = int4_case(3, 700, 96, 32, seed=21)
    whole = lb.int4_matvec(x, w)
    for a, b in ((1, 350), (351, 700)):
        assert torch.equal(lb.int4_matvec(x, lb.Int4Weight(w.packed[a:b], w.scales[a:b])), whole[:, a:b])
    # one rank that holds the whole vocabulary: its all-gather is a copy
    held = []
    monkeypatch.setattr(D, "_world", lambda group: (1, 0))
    monkeypatch.setattr(D.dist, "all_gather_into_tensor", lambda out, rec, group=None: (held.append(rec.clone()), out.copy_(rec)))
    head = lb.Int4Weight.quantize(torch.randn(2000, 128, generator=gen(22), device=DEV), 128)
    h = torch.randn(4, 128, generator=gen(23), device=DEV)
    temp, top_p, u = (torch.full((4,), v, device=DEV) for v in (0.8, 0.9, 0.37))
    s = D.VocabShardSampler(DEV, K=64)
    got = s.sample_hidden(h, head, 0, 2000, temp, top_p, u, top_k=[64] * 4)
    logits = lb.int4_matvec(h, head)
    assert torch.equal(got, s.sample(logits, 0, 2000, temp, top_p, u)) and torch.equal(held[0], held[1])
    prm = [S.SamplingParams(temperature=0.8, top_k=64, top_p=0.9)] * 4
    assert torch.equal(got, S.sample_batch(logits, prm, uniforms=u))
    with pytest.raises(ValueError):
        s.sample_hidden(h, head, 0, 2000, temp, top_p, u, top_k=[3] * 4)


def test_attend_in_place_and_at_once():
    """The output over the queries; two captured steps that share everything but the workspace."""
    for ctx, new in (([700, 30, 0], [1, 1, 1]), ([9000], [1]), ([100, 0, 700], [900, 513, 300])):
        rows = U.make_rows(ctx, new, 16)
        cache = lb.KVCache8(*U.random_cache(rows[-1], 8, 16, 128))
        q = torch.randn(sum(new), 32, 128, generator=gen(1), device=DEV).bfloat16()
        plan = lb.StepPlan(*rows[2:5])
        want = lb.attend(q, cache, rows[1], plan)
        own = q.clone()
        lb.attend(own, cache, rows[1], plan, out=own)
        assert torch.equal(own, want)
        graphs, outs = [], []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(lb.attend(q, cache, rows[1], plan))
            graphs.append(g)
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("rows", [5, 16, 30, 64])
def test_int4_f32_rows_are_exact(rows, group):
    """One value of 24 bits per row, weights that are powers of two: the product is that value at another place, so
    all three parts of it have to arrive, in the right order and column."""
    g, n, k = gen(group + rows), 150, 768
    codes = torch.tensor([0, 4, 6, 7, 9, 10, 12], dtype=torch.uint8, device=DEV)[torch.randint(0, 7, (n, k), generator=g, device=DEV)]
    scales = torch.exp2(torch.randint(-6, 7, (n, k // group), generator=g, device=DEV).float()).half()
    w = lb.Int4Weight(codes[:, ::2] | (codes[:, 1::2] << 4), scales)
    dense = (codes.double() - 8) * scales.double().repeat_interleave(group, 1)
    at = torch.arange(rows, device=DEV)
    for shift in range(0, k, rows):
        v = (torch.randint(0, 1 << 23, (rows,), generator=g, device=DEV) | (1 << 23) | 1).float() * torch.exp2(torch.randint(-40, 20, (rows,), generator=g, device=DEV).float())
        v = torch.where(at % 2 == 0, v, -v)
        cols = (shift + at) % k
        x = torch.zeros(rows, k, device=DEV)
        x[at, cols] = v
        assert torch.equal(lb.int4_matvec(x, w).double(), v.double()[:, None] * dense[:, cols].t()), shift


# --------------------------------------------------------------------------------- block tables
def plan_case(rows, bs, hi_ctx, hi_new, spare, seed, width_cut=0):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, hi_ctx + 1, (rows,), generator=g).tolist()
    new = torch.randint(-1, hi_new + 1, (rows,), generator=g).tolist()
    width = max(1, -(-(hi_ctx + hi_new) // bs) - width_cut)
    held = [min(-(-n // bs), width) for n in lens]
    blocks = sum(held) + spare
    ids = torch.randperm(blocks, generator=g).tolist()
    table, at = [], 0
    for n in held:
        table.append(ids[at: at + n] + [-1] * (width - n))
        at += n
    return table, lens, new, ids[at:] + [0] * at, len(ids) - at


@pytest.mark.parametrize("rows,bs,hi_ctx,hi_new,spare,cut,pad", [
    (1, 16, 0, 1, 1, 0, 0), (1, 1, 5, 3, 9, 0, 2), (7, 16, 40, 5, 3, 0, 5), (64, 32, 300, 1, 64, 0, 0),
    (1000, 16, 200, 33, 900, 1, 3), (1024, 7, 100, 9, 400, 0, -500), (1025, 128, 4000, 60, 300, 2, 1), (4099, 16, 50, 40, 9000, 0, 11)])
def test_plan_matches_row_by_row(rows, bs, hi_ctx, hi_new, spare, cut, pad):
    table, lens, new, free, n_free = plan_case(rows, bs, hi_ctx, hi_new, spare, seed=rows + bs, width_cut=cut)
    capacity = max(0, sum(max(n, 0) for n in new) + pad)
    want, table_after = U.plan_reference(table, lens, new, free, n_free, bs, capacity)
    t, ln, nf = ints(table), ints(lens), ints([n_free])
    p = lb.plan_blocks(t, ln, ints(new), ints(free), nf, bs, capacity)
    for name, v in want.items():
        assert getattr(p, name).tolist() == v, name
    assert t.tolist() == table_after and ln.tolist() == lens and nf.tolist() == [n_free]
    # in place, in a wider table
    wide = torch.full((rows, len(table[0]) + 5), -7, dtype=torch.int32, device=DEV)
    wide[:, : len(table[0])] = ints(table)
    p = lb.plan_blocks(wide[:, : len(table[0])], ln, ints(new), ints(free), nf, bs, capacity, lens_out=ln, n_free_out=nf)
    for name, v in want.items():
        assert getattr(p, name).tolist() == v, name
    assert wide[:, : len(table[0])].tolist() == table_after and bool((wide[:, len(table[0]):] == -7).all())
    assert ln.tolist() == want["lens"]


def test_plan_odd_inputs():
    # no rows; no room; lengths and counts that make no sense; ids outside the cache
    p = lb.plan_blocks(torch.empty(0, 4, dtype=torch.int32, device=DEV), ints([]), ints([]), ints([3, 4]), ints([2]), 16, 5)
    assert p.slots.tolist() == [-1] * 5 and p.starts.tolist() == [0] and p.n_free.tolist() == [2]
    table = [[9, -1], [1, -1], [5, 0], [2, -1]]
    for n_free, cap in ((3, 30), (99, 30), (-5, 30), (3, 0)):
        args = ([-4, 3, 2147483647, 16], [2, 2, 5, 2], [0, 77, 2, 1, 0, 0], n_free, 16, cap)
        want, after = U.plan_reference(table, *args)
        t = ints(table)
        p = lb.plan_blocks(t, ints(args[0]), ints(args[1]), ints(args[2]), ints([n_free]), 16, cap)
        assert p.granted.tolist() == want["granted"] and p.slots.tolist() == want["slots"] and t.tolist() == after
        assert p.n_free.tolist() == want["n_free"] and p.starts.tolist() == want["starts"]


def test_plan_order_of_service():
    """Who goes on behind a refused row: rows that need no block always, the others only if blocks were not the reason."""
    table = [[0, 1, -1, -1], [2, -1, -1, -1], [3, -1, -1, -1], [4, -1, -1, -1]]
    plan = lambda new, capacity: lb.plan_blocks(ints(table), ints([20, 3, 16, 4]), ints(new), ints([5, 6, 0, 0, 0, 0, 0]), ints([1]), 16, capacity)
    # row 0 lacks a block: row 1 needs none and goes on, row 2 needs the one that is left and does not get it
    p = plan([40, 2, 1, 3], 60)
    assert p.granted.tolist() == [0, 2, 0, 3] and p.n_free.tolist() == [1]
    # row 0 is too long for the table: the block is row 2's
    p = plan([45, 2, 1, 3], 60)
    assert p.granted.tolist() == [0, 2, 1, 3] and p.n_free.tolist() == [0] and p.slots.tolist()[47] == 5 * 16
    # row 0 ends behind the capacity, and so do all rows behind it in the step's order
    assert plan([16, 2, 1, 3], 15).granted.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("rows,bs,hi", [(1, 16, 0), (5, 16, 100), (1000, 32, 700), (3000, 4, 60)])
def test_release_then_plan_again(rows, bs, hi):
    table, lens, _, free, n_free = plan_case(rows, bs, hi, 1, 10, seed=rows)
    g = torch.Generator().manual_seed(rows + 1)
    codes = torch.randint(0, 3, (rows,), generator=g).tolist()
    want, left = list(free), n_free
    for b in range(rows):
        if codes[b]:
            for j in range(min(-(-lens[b] // bs), len(table[b]))):
                want[left] = table[b][j]
                left += 1
    t, ln, f, nf = ints(table), ints(lens), ints(free), ints([n_free])
    after, n_after = lb.release_blocks(t, ln, ints(codes), f, nf, bs)
    assert f.tolist() == want and n_after.tolist() == [left]
    assert after.tolist() == [0 if c else n for c, n in zip(codes, lens)] and ln.tolist() == lens and nf.tolist() == [n_free]
    # in place, and once more: the rows hold nothing now
    lb.release_blocks(t, ln, ints(codes), f, nf, bs, lens_out=ln, n_free_out=nf)
    lb.release_blocks(t, ln, ints(codes), f, nf, bs, lens_out=ln, n_free_out=nf)
    assert f.tolist() == want and nf.tolist() == [left] and ln.tolist() == after.tolist()
    # a block list that is full already stays as it is
    full = ints([len(free)])
    _, n_full = lb.release_blocks(t, ints(lens), ints([1] * rows), f, full, bs)
    assert f.tolist() == want and n_full.tolist() == [len(free)]


# ---------------------------------------------------------------------------- 8-bit cache: write
def check_append(k, v, rows, heads, bs, dim, seed, out_of=None):
    table, t, starts, granted, lens, blocks = rows
    cache = lb.KVCache8(*U.random_cache(blocks, heads, bs, dim, seed))
    want = [(c.double(), s.double()) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    for x, (c, s) in zip((k, v), want):
        U.append_reference(c, s, x, table, starts.tolist(), granted.tolist(), lens.tolist())
    lb.append_kv(cache, k, v, t, lb.StepPlan(starts, granted, lens))
    for name, (c, s) in zip("kv", want):
        assert torch.equal(getattr(cache, name + "_scale").double(), s), name
        assert torch.equal(getattr(cache, name).double().nan_to_num(999.0), c.nan_to_num(999.0)), name
    return cache


@pytest.mark.parametrize("ctx,new,heads,bs,dim", [
    ([0], [1], 1, 16, 64), ([15, 16, 17, 0], [1, 1, 1, 1], 2, 16, 128), ([3, 0, 31], [60, 16, 1], 3, 32, 64),
    ([100, 7], [0, 130], 2, 64, 256), ([0, 5, 250], [256, 300, 7], 1, 128, 128), ([1], [700], 1, 256, 64), ([2, 9], [5, 40], 5, 16, 8)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_append_matches_block_by_block(ctx, new, heads, bs, dim, dtype):
    g = gen(sum(ctx) + dim)
    spread = torch.exp(1.5 * torch.randn(sum(new), heads, 1, generator=g, device=DEV))
    k, v = ((torch.randn(sum(new), heads, dim, generator=g, device=DEV) * spread).to(DTYPES[dtype]) for _ in range(2))
    check_append(k, v, U.make_rows(ctx, new, bs, seed=dim), heads, bs, dim, seed=bs)


def test_append_values_and_layouts():
    rows = U.make_rows([5, 0, 40], [7, 33, 1], 16)
    g = gen(1)
    # one fused projection: keys and values are slices of it, 16-byte aligned rows and not
    for off in (0, 1):
        for dt in DTYPES.values():
            fused = torch.randn(41, 900, generator=g, device=DEV).to(dt)
            k, v = (fused[:, off + a: off + a + 256].view(41, 2, 128) for a in (128, 384))
            check_append(k, v, rows, 2, 16, 128, seed=2)
    # heads that share one value (stride 0), tokens inside heads, an inner stride that is not 1
    x = torch.randn(41, 1, 64, generator=g, device=DEV)
    check_append(x.expand(41, 4, 64), x.expand(41, 4, 64) * 3, rows, 4, 16, 64, seed=3)
    y = torch.randn(4, 41, 64, generator=g, device=DEV).transpose(0, 1)
    check_append(y, y.flip(0), rows, 4, 16, 64, seed=4)
    z = torch.randn(41, 64, 4, generator=g, device=DEV).transpose(1, 2)
    check_append(z, z, rows, 4, 16, 64, seed=5)
    # zeros, the smallest and largest numbers, exact powers and borders of the scale, not finite ones
    s = torch.randn(41, 2, 64, generator=g, device=DEV)
    s[0] = 0
    s[7:] = s[7:] * 2.0 ** -130
    check_append(s, -s, rows, 2, 16, 64, seed=6)
    s = torch.zeros(41, 2, 64, device=DEV)
    s[:, 0, 0], s[:, 1, 1] = 448.0 * 4, 449.0
    s[:, 0, 1] = 3.0e38
    check_append(s, torch.full_like(s, 1.75), rows, 2, 16, 64, seed=7)
    s = torch.randn(41, 2, 64, generator=g, device=DEV)
    s[3, 0, 5], s[9, 1, 6], s[20, 0, 7] = math.nan, math.inf, -math.inf
    check_append(s, s, rows, 2, 16, 64, seed=8)
    check_append(torch.full_like(s, math.nan), torch.full_like(s, math.inf), rows, 2, 16, 64, seed=9)


def test_append_passes_over_what_does_not_fit():
    table, t, starts, granted, lens, blocks = U.make_rows([5, 0, 40, 3], [7, 33, 1, 2], 16)
    k = torch.randn(43, 2, 64, generator=gen(2), device=DEV)
    # a refused row, a row of fewer tokens than granted, one behind the table, blocks outside the cache
    for g2, l2, edit in (([0, 33, 1, 2], None, None), ([7, 34, 1, 2], [12, 33, 41, 5], None), (None, [12, 33, 4100, 5], None),
                         (None, None, (1, 1, -1)), (None, None, (1, 0, blocks)), (None, None, (2, 2, 2 ** 31 - 1))):
        tb = [list(r) for r in table]
        if edit:
            tb[edit[0]][edit[1]] = edit[2]
        rows = (tb, ints(tb), starts, ints(g2) if g2 else granted, ints(l2) if l2 else lens, blocks)
        check_append(k, -k, rows, 2, 16, 64, seed=10)
    check_append(k[:20], k[:20], (table, t, starts, granted, lens, blocks), 2, 16, 64, seed=11)  # tokens missing
    # a second step on the first one's blocks, the scale growing and not
    cache = lb.KVCache8.empty(8, 2, 16, 64)
    t2 = ints([[6, 3, 1]])
    ref = [torch.zeros(8, 2, 16, 64, dtype=torch.float64, device=DEV), torch.ones(8, 2, dtype=torch.float64, device=DEV)]
    for step, (old, n, size) in enumerate(((0, 5, 1.0), (5, 1, 30.0), (6, 1, 0.01), (7, 20, 500.0), (27, 1, 1.0))):
        x = torch.randn(n, 2, 64, generator=gen(30 + step), device=DEV) * size
        U.append_reference(ref[0], ref[1], x, [[6, 3, 1]], [0], [n], [old + n])
        lb.append_kv(cache, x, -x, t2, lb.StepPlan(ints([0, n]), ints([n]), ints([old + n])))
        assert torch.equal(cache.k.double(), ref[0]) and torch.equal(cache.k_scale.double(), ref[1])
        assert torch.equal(cache.v.double(), -ref[0])


# ------------------------------------------------------------------------------------ attention
def check_attend(q, cache, rows, scale=None, out=None):
    """The products with e4m3 codes are exact, the softmax sum is f32: what rounds is the weights to
    f16 (2^-11 each, so 2^-11 of the sum of |weight * value|), scores and exponentials in f32 (held to a
    quarter of that for the scores of these inputs, below 2^6), and the result."""
    table, t, starts, granted, lens, blocks = rows
    dim = q.shape[2]
    sc = dim ** -0.5 if scale is None else scale
    lse = torch.full(q.shape[:2], 77.0, device=DEV)
    y = torch.full(q.shape, 77.0, dtype=q.dtype, device=DEV) if out is None else out
    lb.attend(q, cache, t, lb.StepPlan(starts, granted, lens), scale=scale, out=y, lse_out=lse)
    want, mag, wl = U.attend_reference(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, starts.tolist(), granted.tolist(), lens.tolist(), sc)
    idle = wl.isnan() & (lse == 77)
    tol = 1.25 * 2.0 ** -11 * mag + torch.finfo(q.dtype).eps / 2 * want.abs() + (2.0 ** -24 if q.dtype == torch.float16 else 0)
    off = (y.double() - want).abs()
    # a result from half a step above f16's largest number on (65504 + 16) rounds to infinity
    over = y.isinf() & (want.abs() + tol >= 65520.0) & (want.sign() == y.sign()) if q.dtype == torch.float16 else torch.zeros_like(y, dtype=torch.bool)
    ok = (off <= tol) | (want.isnan() & (y.isnan() | idle[..., None])) | over
    assert bool(ok.all()), (float((off - tol).nan_to_num(0).max()), ok.logical_not().nonzero()[:5].tolist())
    assert bool((y[idle] == 77).all()) if out is None else True
    near = ((lse.double() - wl).abs() <= 2.0 ** -16 * (1 + wl.abs())) | (lse == wl) | wl.isnan()
    assert bool(near.all())
    return y, lse


@pytest.mark.parametrize("ctx,new,heads,per,bs,dim", [
    ([0], [1], 1, 1, 16, 64), ([15, 16, 17, 0], [1, 1, 1, 1], 2, 7, 16, 64), ([300, 2, 1111], [1, 1, 1], 2, 4, 32, 128),
    ([0, 900], [1, 1], 1, 16, 64, 256), ([70, 0, 5, 33], [5, 40, 1, 16], 2, 3, 16, 128), ([5000], [1], 1, 8, 128, 128),
    ([10, 300], [130, 77], 2, 4, 256, 64), ([3, 0, 100, 50], [0, 2, 0, 9], 1, 32, 16, 256), ([40], [200], 1, 1, 16, 128)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attend_sizes(ctx, new, heads, per, bs, dim, dtype):
    rows = U.make_rows(ctx, new, bs, seed=dim)
    cache = lb.KVCache8(*U.random_cache(rows[-1], heads, bs, dim, seed=per))
    q = torch.randn(sum(new) + 2, heads * per, dim, generator=gen(dim), device=DEV).to(DTYPES[dtype])
    y, lse = check_attend(q, cache, rows)
    y2, lse2 = check_attend(q, cache, rows)
    assert torch.equal(y, y2) or bool(y.isnan().any())
    assert torch.equal(lse, lse2)


@pytest.mark.parametrize("ctx,new,heads,per,bs,dim", [
    ([100, 0, 700], [900, 513, 300], 8, 4, 16, 128), ([0], [2100], 4, 2, 64, 64), ([37, 5, 4000, 0, 90], [200, 131, 257, 0, 640], 5, 3, 32, 128),
    ([1500, 64], [640, 1000], 2, 7, 256, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attend_prompt_chunks(ctx, new, heads, per, bs, dim, dtype):
    """Steps that fill groups of 256 query rows (the tensor-memory kernel), NaN among keys and values."""
    rows = U.make_rows(ctx, new, bs, seed=dim)
    table, t, starts, granted, lens, blocks = rows
    cache = lb.KVCache8(*U.random_cache(blocks, heads, bs, dim, seed=per))
    q = torch.randn(sum(new) + 2, heads * per, dim, generator=gen(dim), device=DEV).to(DTYPES[dtype])
    y, lse = check_attend(q, cache, rows)
    y2, lse2 = check_attend(q, cache, rows)
    idle = torch.zeros(q.shape[0], dtype=torch.bool, device=DEV)
    idle[sum(new):] = True
    assert torch.equal(y, y2) and torch.equal(lse, lse2) and bool(y[~idle].isfinite().all()) and bool((y[idle] == 77).all())
    check_attend(q, cache, rows, scale=-0.02)
    check_attend(q, cache, rows, scale=0.0)
    fused = torch.randn(sum(new) + 2, heads * per * dim + 5, generator=gen(3), device=DEV).to(DTYPES[dtype])
    out = torch.zeros(sum(new) + 2, heads * per, dim + 3, dtype=DTYPES[dtype], device=DEV)
    check_attend(fused[:, 5:].view(-1, heads * per, dim), cache, rows, out=out[:, :, :dim])
    # scales of the blocks that differ by far, one block outside the cache, what lies behind the rows' ends
    cache.k_scale.mul_(torch.rand(cache.k_scale.shape, generator=gen(5), device=DEV) + 0.5)
    cache.v_scale.mul_(torch.exp2(torch.randint(-20, 20, cache.v_scale.shape, generator=gen(6), device=DEV).float()) * 1.3)
    for b, ln in enumerate(lens.tolist()):
        if ln % bs and granted[b] > 0:
            cache.k.view(torch.uint8)[table[b][ln // bs], :, ln % bs:] = 0x7F
            cache.v.view(torch.uint8)[table[b][ln // bs], :, ln % bs:] = 0xFF
    tb = [list(r) for r in table]
    tb[0][0] = blocks
    check_attend(q, cache, (tb, ints(tb), starts, granted, lens, blocks))
    # NaN that some queries see and others do not
    b = len(ctx) - 1
    p = ctx[b] + new[b] // 2
    cache.v.view(torch.uint8)[table[b][p // bs], 0, p % bs, 7] = 0x7F
    y, _ = check_attend_nan(q, cache, rows)
    first = sum(new[:b])
    seen = torch.arange(ctx[b], ctx[b] + new[b], device=DEV) >= p
    assert torch.equal(y[first: first + new[b], 0, 7].isnan(), seen) and not bool(y[first: first + new[b], 0, 6].isnan().any())


@pytest.mark.parametrize("per,dim", [(4, 128), (7, 64), (16, 128), (4, 256)])
def test_attend_prompts_and_single_tokens_mixed(per, dim):
    """Steps in which some rows have one token, some a few and some a chunk; an idle row, padding behind them."""
    rows = U.make_rows([4000, 100, 0, 2500, 60, 9, 1300, 0], [1, 700, 300, 1, 20, 0, 15, 1], 16, seed=per)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 4, 16, dim, seed=per))
    q = torch.randn(1038 + 30, 4 * per, dim, generator=gen(dim), device=DEV).bfloat16()
    y, lse = check_attend(q, cache, rows)
    assert bool((y[1038:] == 77).all()) and bool((lse[1038:] == 77).all()) and bool(y[:1038].isfinite().all())


def kernels(f):
    """Names of the kernels that a call launches, from a graph that captures it."""
    drv = pytest.importorskip("cuda.bindings.driver")
    f()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        f()
    graph = drv.CUgraph(g.raw_cuda_graph())
    _, _, n = drv.cuGraphGetNodes(graph, 0)
    _, nodes, n = drv.cuGraphGetNodes(graph, n)
    return [drv.cuFuncGetName(drv.cuGraphKernelNodeGetParams(x)[1].func)[1].decode() for x in nodes[:n]]


@pytest.mark.parametrize("n,per,dim", [(5, 4, 128), (10, 4, 128), (11, 4, 128), (5, 4, 64), (15, 4, 64), (3, 16, 128), (0, 4, 128), (0, 7, 64)])
def test_attend_a_few_tokens_per_row(n, per, dim):
    """Batches on both sides of the borders between the kernels: n tokens in every row (0: 1 to 16 of them)."""
    new = [n or 1 + (i * 5) % 16 for i in range(64)]
    rows = U.make_rows([(53 * i) % 300 for i in range(64)], new, 16, seed=n)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 8, 16, dim, seed=per))
    q = torch.randn(sum(new), 8 * per, dim, generator=gen(dim + n), device=DEV).bfloat16()
    y, _ = check_attend(q, cache, rows)
    assert bool(y.isfinite().all())


@pytest.mark.parametrize("dim", [64, 128])
def test_attend_short_rows_share_their_tiles(dim):
    """Eight tokens of four query heads each, 32 query rows: not in groups of eight, which read the cache four times."""
    rows = U.make_rows([100] * 64, [8] * 64, 16)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 8, 16, dim))
    q = torch.zeros(512, 32, dim, dtype=torch.float16, device=DEV)
    names = kernels(lambda: lb.attend(q, cache, rows[1], lb.StepPlan(*rows[2:5])))
    assert names and not [x for x in names if f"lss_attend_kernelILi{dim}ELi2ELi1E" in x], names


def check_attend_nan(q, cache, rows):
    """As check_attend where some values are NaN: the places of NaN, the others against a cache without it."""
    clean = lb.KVCache8(cache.k, torch.where(cache.v.float().isnan(), 0.0, cache.v.float()).to(E4M3), cache.k_scale, cache.v_scale)
    y0, l0 = check_attend(q, clean, rows)
    table, t, starts, granted, lens, blocks = rows
    lse, y = torch.full(q.shape[:2], 77.0, device=DEV), torch.full(q.shape, 77.0, dtype=q.dtype, device=DEV)
    lb.attend(q, cache, t, lb.StepPlan(starts, granted, lens), out=y, lse_out=lse)
    assert torch.equal(lse, l0) and bool(((y == y0) | y.isnan()).all())
    return y, lse


def test_attend_many_rows():
    ctx = [(i * 37) % 90 for i in range(1300)]
    new = [1 if i % 5 else 0 for i in range(1300)]
    rows = U.make_rows(ctx, new, 16)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 1, 16, 64))
    q = torch.randn(sum(new), 2, 64, generator=gen(1), device=DEV).half()
    check_attend(q, cache, rows)


def test_attend_layouts_and_scales():
    rows = U.make_rows([100, 33], [1, 20], 16)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 2, 16, 128))
    for off in (0, 1):  # queries as a slice of a fused projection, 16-byte aligned and not; an output of its own strides
        for dt in (torch.bfloat16, torch.float16):
            fused = torch.randn(21, 1400, generator=gen(2), device=DEV).to(dt)
            q = fused[:, off: off + 768].view(21, 6, 128)
            check_attend(q, cache, rows)
            out = torch.zeros(21, 6, 150, dtype=dt, device=DEV)
            check_attend(q, cache, rows, scale=0.3, out=out[:, :, off: off + 128])
            assert bool((out[:, :, off + 128:] == 0).all())
    q = torch.randn(6, 21, 128, generator=gen(3), device=DEV).half().transpose(0, 1)
    check_attend(q, cache, rows, scale=0.0)
    check_attend(q, cache, rows, scale=-0.05)
    # large queries (bf16 reaches far beyond f16), tiny ones, rows of zeros
    q = torch.randn(21, 6, 128, generator=gen(4), device=DEV).bfloat16()
    check_attend(q * 2.0 ** 100, cache, rows, scale=2.0 ** -104)
    check_attend(q * 2.0 ** -100, cache, rows, scale=2.0 ** 96)
    check_attend(q * 0, cache, rows)
    # scales of the blocks that differ by far, that are no powers of two, blocks of zeros
    cache.k_scale.mul_(torch.rand(cache.k_scale.shape, generator=gen(5), device=DEV) + 0.5)
    cache.v_scale.mul_(torch.exp2(torch.randint(-30, 30, cache.v_scale.shape, generator=gen(6), device=DEV).float()) * 1.3)
    check_attend(q, cache, rows)
    cache.v.view(torch.uint8)[::2] = 0
    cache.v_scale[::2] = 2.0 ** -126
    check_attend(q, cache, rows)


def test_attend_results_head_by_head():
    """Tokens inside heads in the result, and a result between the queries' rows."""
    rows = U.make_rows([100, 33], [1, 20], 16)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 2, 16, 128))
    both = torch.randn(21, 6, 256, generator=gen(2), device=DEV).half()
    q, plan = both[:, :, :128], lb.StepPlan(*rows[2:5])
    want = lb.attend(q, cache, rows[1], plan)
    out = torch.zeros(6, 21, 128, dtype=torch.float16, device=DEV).transpose(0, 1)
    assert torch.equal(lb.attend(q, cache, rows[1], plan, out=out), want)
    keep = q.clone()
    assert torch.equal(lb.attend(q, cache, rows[1], plan, out=both[:, :, 128:]), want) and torch.equal(q, keep)
    flat = torch.zeros(40 * 6 * 128, dtype=torch.float16, device=DEV)
    for sizes in ((128 * 5, 128, 1), (128, 128 * 20, 1), (0, 128, 1)):
        with pytest.raises(ValueError):
            lb.attend(q, cache, rows[1], plan, out=flat.as_strided((21, 6, 128), sizes))
    with pytest.raises(lb.SamplerError):
        lb.attend(q, cache, rows[1], plan, out=both[:, :, 64:192])


# few query rows (each group size of that kernel, one and two tiles a step), prompt chunks
SCORES = [([700, 900], [1, 1], 2, 4, 128), ([1500], [1], 2, 4, 128), ([700], [4], 2, 4, 64), ([700], [7], 2, 4, 128), ([700], [3], 1, 4, 256),
          ([700, 1000], [900, 300], 8, 4, 128), ([650], [1300], 8, 2, 64)]


@pytest.mark.parametrize("ctx,new,heads,per,dim", SCORES)
def test_attend_scores_that_are_all_minus_infinity(ctx, new, heads, per, dim):
    """A query whose products are all -inf has no softmax: NaN, not the 0 of one that sees nothing."""
    rows = U.make_rows(ctx, new, 16, seed=dim)
    table, t, starts, granted, lens, blocks = rows
    k, v, ks, vs = U.random_cache(blocks, heads, 16, dim, seed=per)
    k.view(torch.uint8)[..., 0] = 0x38  # 1
    cache = lb.KVCache8(k, v, ks, vs)
    q = torch.randn(sum(new), heads * per, dim, generator=gen(dim), device=DEV).bfloat16()
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    hit[0, 0] = hit[-1, -1] = hit[sum(new) // 2, heads] = True
    q[..., 0][hit] = -math.inf
    lse = torch.full(q.shape[:2], 77.0, device=DEV)
    y = lb.attend(q, cache, t, lb.StepPlan(starts, granted, lens), lse_out=lse)
    assert bool(y[hit].isnan().all()) and bool((lse[hit] == -math.inf).all())
    want, mag, wl = U.attend_reference(q, k, v, ks, vs, table, starts.tolist(), granted.tolist(), lens.tolist(), dim ** -0.5)
    tol = 1.25 * 2.0 ** -11 * mag + 2.0 ** -8 * want.abs()
    assert bool(((y.double() - want).abs() <= tol)[~hit].all()) and bool(((lse.double() - wl).abs() <= 2.0 ** -16 * (1 + wl.abs()))[~hit].all())


@pytest.mark.parametrize("ctx,new,heads,per,dim", SCORES)
def test_attend_scores_that_overflow_to_minus_infinity(ctx, new, heads, per, dim):
    """Tokens whose scores fall below the range of f32 have no weight, wherever they lie."""
    rows = U.make_rows(ctx, new, 16, seed=dim)
    table, t, starts, granted, lens, blocks = rows
    k, v, ks, vs = U.random_cache(blocks, heads, 16, dim, seed=per)
    k.view(torch.uint8)[:] = 0
    for a, b in ((0, 600), (40, 100), (620, 640)):  # from the first token on, in the middle, near the end
        k.view(torch.uint8)[:] = 0
        for row in table:
            for p in range(a, b):
                k.view(torch.uint8)[row[p // 16], :, p % 16, 0] = 0x7E  # 448
        q = torch.zeros(sum(new), heads * per, dim, dtype=torch.bfloat16, device=DEV)
        q[..., 0] = -2.0 ** 127
        y, lse = check_attend(q, lb.KVCache8(k, v, torch.ones_like(ks), vs), rows, scale=1.0)
        assert bool(y.isfinite().all()) and bool(lse.isfinite().all())


@pytest.mark.parametrize("ctx,new,heads,per,dim", SCORES)
def test_attend_smallest_value_scales(ctx, new, heads, per, dim):
    """Values near the smallest scale of a block (2^-126): bf16 results hold them."""
    rows = U.make_rows(ctx, new, 16, seed=dim)
    k, v, ks, vs = U.random_cache(rows[-1], heads, 16, dim, seed=per)
    q = torch.randn(sum(new), heads * per, dim, generator=gen(dim), device=DEV).bfloat16()
    for lo, hi in ((-126, -126), (-126, -100), (-126, 100), (110, 118)):
        scales = torch.exp2(torch.randint(lo, hi + 1, vs.shape, generator=gen(lo + hi), device=DEV).float())
        y, _ = check_attend(q, lb.KVCache8(k, v, ks, scales), rows)
        assert bool((y != 0).any())


def test_attend_small_weights_are_not_lost():
    """One token far above 60,000 others: together they hold a good part of the sum."""
    n, dim = 60000, 64
    rows = U.make_rows([n - 1], [1], 32)
    k = torch.zeros(rows[-1], 1, 32, dim, device=DEV)
    k[rows[0][0][0], 0, 0, 0] = 14.0
    v = torch.randn(rows[-1], 1, 32, dim, generator=gen(1), device=DEV) * 0.1 + 2.0
    one = torch.ones(rows[-1], 1, device=DEV)
    cache = lb.KVCache8(k.to(E4M3), v.to(E4M3), one, one.clone())
    q = torch.zeros(1, 1, dim, dtype=torch.float16, device=DEV)
    q[0, 0, 0] = 1.0
    for scale in (0.5, 0.8, 1.2):
        check_attend(q, cache, rows, scale=scale)


def test_attend_masked_places_and_bad_blocks():
    table, t, starts, granted, lens, blocks = U.make_rows([20, 37, 9], [1, 30, 1], 16)
    k, v, ks, vs = U.random_cache(blocks, 1, 16, 64, seed=3)
    nan, q = 0x7F, torch.randn(32, 4, 64, generator=gen(7), device=DEV).bfloat16()
    for name, x in (("k", k), ("v", v)):
        for b, ln in enumerate(lens.tolist()):  # behind each row's end, in its last block
            if ln % 16:
                x.view(torch.uint8)[table[b][ln // 16], :, ln % 16:] = nan
    cache = lb.KVCache8(k, v, ks, vs)
    y, _ = check_attend(q, cache, (table, t, starts, granted, lens, blocks))
    assert bool(y.isfinite().all())
    # a NaN that later queries of the same row see and earlier ones do not
    v.view(torch.uint8)[table[1][50 // 16], 0, 50 % 16, 5] = nan
    y, _ = check_attend(q, cache, (table, t, starts, granted, lens, blocks))
    seen = (torch.arange(37, 67, device=DEV) >= 50)
    assert torch.equal(y[1:31, 0, 5].isnan(), seen) and not bool(y[1:31, 0, 4].isnan().any())
    v.view(torch.uint8)[table[1][50 // 16], 0, 50 % 16, 5] = 0
    k.view(torch.uint8)[table[1][44 // 16], 0, 44 % 16, 5] = nan
    y, _ = check_attend(q, cache, (table, t, starts, granted, lens, blocks))
    assert torch.equal(y[1:31, 0, 0].isnan(), torch.arange(37, 67, device=DEV) >= 44)
    k.view(torch.uint8)[table[1][44 // 16], 0, 44 % 16, 5] = 0
    # blocks outside the cache are not seen: some, and all of a row
    for edits in ([(1, 0, -1)], [(1, 1, blocks), (2, 0, -9)], [(0, 0, -1), (0, 1, 2 ** 31 - 1)]):
        tb = [list(r) for r in table]
        for b, j, p in edits:
            tb[b][j] = p
        check_attend(q, cache, (tb, ints(tb), starts, granted, lens, blocks))
    # rows whose numbers do not fit are left out
    check_attend(q, cache, (table, t, starts, ints([1, 30, 11]), lens, blocks))
    check_attend(q, cache, (table, t, starts, granted, ints([21, 9999, 10]), blocks))
    check_attend(q[:10], cache, (table, t, starts, granted, lens, blocks))


def test_attend_far_blocks():
    """Blocks whose values lie behind 2^31 bytes of the cache."""
    blocks, heads, bs, dim = 40000, 8, 64, 128
    cache = lb.KVCache8(*(torch.zeros(blocks, heads, bs, dim, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2)),
                        torch.ones(blocks, heads, device=DEV), torch.ones(blocks, heads, device=DEV))
    pages = [39999, 5, 39000, 33000, 20001]
    x, y = (torch.randn(300, heads, dim, generator=gen(i), device=DEV).bfloat16() for i in (1, 2))
    t, plan = ints([pages]), lb.StepPlan(ints([0, 300]), ints([300]), ints([300]))
    lb.append_kv(cache, x, y, t, plan)
    q = torch.randn(300, heads, dim, generator=gen(3), device=DEV).bfloat16()
    got = lb.attend(q, cache, t, plan)
    small = lb.KVCache8.empty(5, heads, bs, dim)
    t2 = ints([[0, 1, 2, 3, 4]])
    lb.append_kv(small, x, y, t2, plan)
    assert torch.equal(got, lb.attend(q, small, t2, plan))
    for i, p in enumerate(pages):
        n = min(64, 300 - 64 * i)  # what lies behind the tokens of a block is nobody's
        assert torch.equal(cache.k[p, :, :n].view(torch.uint8), small.k[i, :, :n].view(torch.uint8))


# ---------------------------------------------------------------------------------- run together
class Loop:
    """A decode loop of one attention layer between two 4-bit projections, all state on the device."""

    def __init__(self, rows=6, blocks=40, bs=16, heads=2, per=3, dim=64, vocab=500, hidden=128):
        g = gen(77)
        r = lambda *s: torch.randn(*s, generator=g, device=DEV)
        self.rows, self.bs, self.heads, self.per, self.dim, self.width = rows, bs, heads, per, dim, 8
        self.embed = r(vocab, hidden)
        self.qkv = lb.Int4Weight.quantize(r((heads * (per + 2)) * dim, hidden) / 8, 32)
        self.proj = lb.Int4Weight.quantize(r(hidden, heads * per * dim) / 8, 64)
        self.head = lb.Int4Weight.quantize(r(vocab, hidden), 128)
        self.cache = lb.KVCache8.empty(blocks, heads, bs, dim)
        self.table = torch.full((rows, self.width), -1, dtype=torch.int32, device=DEV)
        self.lens, self.free, self.n_free = ints([0] * rows), torch.arange(blocks, dtype=torch.int32, device=DEV), ints([blocks])
        self.new = ints([5, 1, 17, 0, 3, 1])
        self.tokens = torch.randint(0, vocab, (32,), generator=g, device=DEV)
        self.prm = S.RowParams.from_params([S.SamplingParams(temperature=0.0)] * rows, DEV)
        self.u = torch.rand(rows, generator=g, device=DEV)

    def step(self, capacity):
        plan = lb.plan_blocks(self.table, self.lens, self.new, self.free, self.n_free, self.bs, capacity, lens_out=self.lens, n_free_out=self.n_free)
        x = self.embed[self.tokens[:capacity]].bfloat16()
        hq, hk = self.heads * self.per, self.heads
        qkv = lb.int4_matvec(x, self.qkv).view(capacity, hq + 2 * hk, self.dim)
        lb.append_kv(self.cache, qkv[:, hq: hq + hk], qkv[:, hq + hk:], self.table, plan)
        o = torch.zeros(capacity, hq, self.dim, dtype=x.dtype, device=DEV)
        lse = torch.zeros(capacity, hq, device=DEV)
        lb.attend(qkv[:, :hq], self.cache, self.table, plan, out=o, lse_out=lse)
        h = x + lb.int4_matvec(o.view(capacity, -1), self.proj)
        last = (plan.starts[1:] - 1).clamp(min=0)
        tok = lb.sample_hidden(h[last.long()], self.head, self.prm, uniforms=self.u)
        return plan, qkv, o, h, last, tok


def test_decode_loop_against_64_bits():
    m = Loop()
    plan, qkv, o, h, last, tok = m.step(27)
    hq, hk = m.heads * m.per, m.heads
    # what the step did, in 64 bits from its own rounded intermediate values
    table = m.table.tolist()
    k, ks = torch.zeros(m.cache.k.shape, dtype=torch.float64, device=DEV), torch.ones(m.cache.k_scale.shape, dtype=torch.float64, device=DEV)
    U.append_reference(k, ks, qkv[:, hq: hq + hk], table, plan.starts.tolist(), plan.granted.tolist(), plan.lens.tolist())
    assert torch.equal(m.cache.k.double(), k) and torch.equal(m.cache.k_scale.double(), ks)
    want, mag, _ = U.attend_reference(qkv[:, :hq], m.cache.k, m.cache.v, m.cache.k_scale, m.cache.v_scale, table, plan.starts.tolist(), plan.granted.tolist(), plan.lens.tolist(), m.dim ** -0.5)
    off = (o.double() - want).abs()
    assert bool((off <= 1.25 * 2.0 ** -11 * mag + 2.0 ** -8 * want.abs()).all())
    logits = h[last.long()].double() @ m.head.dequantize().double().t()
    best = logits.topk(2, -1).values
    sure = best[:, 0] - best[:, 1] > 1e-3 * best.abs().amax(-1)
    assert bool((tok.long() == logits.argmax(-1))[sure].all()) and int(sure.sum()) >= 4
    # stop some rows, give their blocks back, decode on
    codes = S.check_stop_batch(tok, None, [[int(tok[0])], [], [int(tok[2])], [], [], []])
    held = {p for b in range(m.rows) for p in table[b][: -(-int(plan.lens[b]) // m.bs)]}
    lb.release_blocks(m.table, m.lens, codes, m.free, m.n_free, m.bs, lens_out=m.lens, n_free_out=m.n_free)
    assert [int(c) for c in codes[:2]] == [S.STOP_TOKEN, S.STOP_NONE] and m.lens[0] == 0 and m.lens[2] == 0
    left = set(m.free[: int(m.n_free)].tolist())
    live = {p for b in (1, 3, 4, 5) for p in table[b][: -(-int(m.lens[b]) // m.bs)]}
    assert len(left) == int(m.n_free) and left | live == set(range(40)) and not left & live and held >= live


def test_loop_keeps_rows_that_had_no_token_of_their_own():
    """An idle row, a refused one and one inside its prompt behind rows that sample their EOS: the codes of the
    tokens that stand in their places would free them."""
    m = Loop()
    m.step(27)
    before = m.lens.clone()
    m.new = ints([1, 0, 4, 1, 200, 0])  # row 4 does not fit the step
    plan, _, _, _, last, tok = m.step(27)
    assert plan.granted.tolist() == [1, 0, 4, 1, 0, 0] and int(last[1]) == int(last[0]) and int(tok[1]) == int(tok[0])
    codes = S.check_stop_batch(tok, tok.tolist())  # whatever stands there is the row's EOS
    assert bool((codes == S.STOP_EOS).all())
    prompts = before.clone()
    prompts[2] = int(plan.lens[2]) + 1
    codes = plan.stops(codes, prompts)
    assert codes.tolist() == [S.STOP_EOS, 0, 0, S.STOP_EOS, 0, 0]
    held = [m.table[b, : -(-int(plan.lens[b]) // m.bs)].tolist() for b in range(m.rows)]
    lb.release_blocks(m.table, m.lens, codes, m.free, m.n_free, m.bs, lens_out=m.lens, n_free_out=m.n_free)
    left = set(m.free[: int(m.n_free)].tolist())
    assert m.lens.tolist() == [0, int(before[1]), int(before[2]) + 4, 0, int(before[4]), int(before[5])]
    for b in (1, 2, 4, 5):
        assert not left & set(held[b])
    assert set(held[0]) | set(held[3]) <= left


def test_decode_loop_captured_and_replayed():
    """The captured step against eager ones, several steps on: state in place, no host reads."""
    eager, graph = Loop(), Loop()
    for m in (eager, graph):
        m.step(27)
        m.new.fill_(1)
    tokens = eager.tokens.clone()

    def step(m):
        plan, _, o, h, _, tok = m.step(6)
        m.tokens[:6] = tok.long()
        codes = (tok % 7 == 0).int()
        lb.release_blocks(m.table, m.lens, codes, m.free, m.n_free, m.bs, lens_out=m.lens, n_free_out=m.n_free)
        return tok, o, plan.slots

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    keep = [t.clone() for t in (graph.tokens, graph.table, graph.lens, graph.free, graph.n_free)]
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            got = step(graph)
    torch.cuda.current_stream().wait_stream(side)
    for t, was in zip((graph.tokens, graph.table, graph.lens, graph.free, graph.n_free), keep):
        assert torch.equal(t, was)  # capturing ran nothing
    for _ in range(25):
        want = step(eager)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    for name in ("table", "lens", "free", "n_free"):
        assert torch.equal(getattr(eager, name), getattr(graph, name)), name
    assert torch.equal(eager.cache.k.view(torch.uint8), graph.cache.k.view(torch.uint8)) and tokens.numel() == 32


def test_two_streams_at_once():
    rows = U.make_rows([3000, 77], [1, 1], 16)
    cache = lb.KVCache8(*U.random_cache(rows[-1], 2, 16, 128))
    w, x = int4_case(2, 3001, 512, 64, seed=1)
    qs = [torch.randn(2, 8, 128, generator=gen(i), device=DEV).half() for i in range(2)]
    plan = lb.StepPlan(*rows[2:5])
    want = [(lb.attend(q, cache, rows[1], plan), lb.int4_matvec(x, w)) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = []
    for _ in range(20):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append((lb.attend(q, cache, rows[1], plan), lb.int4_matvec(x, w)))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# -------------------------------------------------------------------------------------- refusals
def test_refusals():
    w, x = int4_case(2, 20, 64, 32, seed=1)
    bad = lambda exc, f, *a, **k: pytest.raises(exc, f, *a, **k)
    bad(RuntimeError, lb.int4_matvec, x.cpu(), w)
    bad(ValueError, lb.int4_matvec, x[:, :32], w)
    bad(TypeError, lb.int4_matvec, x.double(), w)
    bad(TypeError, lb.int4_matvec, x, w, out_dtype=torch.int32)
    bad(ValueError, lb.int4_matvec, x, lb.Int4Weight(w.packed[:, ::2], w.scales))
    bad(ValueError, lb.int4_matvec, x, lb.Int4Weight(w.packed, w.scales.float()))
    bad(ValueError, lb.int4_matvec, x, lb.Int4Weight(w.packed, w.scales[:10]))
    bad(ValueError, lb.int4_matvec, x, lb.Int4Weight(w.packed.cpu(), w.scales))
    bad(ValueError, lb.int4_matvec, x, w, out=torch.empty(2, 21, device=DEV))
    bad(lb.SamplerError, lb.int4_matvec, torch.zeros(1, 96, device=DEV), lb.Int4Weight(torch.zeros(4, 48, dtype=torch.uint8, device=DEV), torch.zeros(4, 1, device=DEV).half()))
    rows = U.make_rows([5], [2], 16)
    cache, plan = lb.KVCache8(*U.random_cache(rows[-1], 2, 16, 64)), lb.StepPlan(*rows[2:5])
    k = torch.zeros(2, 2, 64, device=DEV)
    q = torch.zeros(2, 4, 64, device=DEV).half()
    bad(ValueError, lb.append_kv, cache, k[:, :1], k, rows[1], plan)
    bad(TypeError, lb.append_kv, cache, k.double(), k.double(), rows[1], plan)
    bad(ValueError, lb.append_kv, cache, k, k, rows[1].long(), plan)
    bad(ValueError, lb.append_kv, cache, k, k, rows[1], lb.StepPlan(rows[2][:1], *rows[3:5]))
    bad(ValueError, lb.append_kv, lb.KVCache8(cache.k, cache.v, cache.k_scale, cache.v_scale.double()), k, k, rows[1], plan)
    bad(TypeError, lb.attend, q.float(), cache, rows[1], plan)
    bad(ValueError, lb.attend, q[:, :3], cache, rows[1], plan)
    bad(ValueError, lb.attend, q, cache, rows[1], plan, out=torch.empty(2, 4, 64, device=DEV))
    bad(ValueError, lb.attend, q, cache, rows[1], plan, lse_out=torch.empty(4, 2, device=DEV))
    odd = lb.KVCache8(*U.random_cache(rows[-1], 2, 16, 96))
    bad(lb.SamplerError, lb.attend, torch.zeros(2, 4, 96, device=DEV).half(), odd, rows[1], plan)
    odd = lb.KVCache8(*U.random_cache(rows[-1], 2, 24, 64))
    bad(lb.SamplerError, lb.attend, q, odd, rows[1], plan)
    bad(lb.SamplerError, lb.append_kv, odd, k, k, rows[1], plan)
    args = (ints([[0, 1]]), ints([3]), ints([1]), ints([1, 2]), ints([2]))
    bad(ValueError, lb.plan_blocks, *args, 16, -1)
    bad(lb.SamplerError, lb.plan_blocks, *args, 0, 4)
    bad(ValueError, lb.plan_blocks, args[0], args[1].long(), *args[2:], 16, 4)
    bad(ValueError, lb.plan_blocks, args[0], args[1], args[2], args[3], ints([1, 1]), 16, 4)
    bad(ValueError, lb.release_blocks, args[0], args[1], ints([1, 1]), args[3], args[4], 16)
    bad(RuntimeError, lb.plan_blocks, args[0].cpu(), *args[1:], 16, 4)
    # no tokens, no rows
    lb.append_kv(cache, k[:0], k[:0], rows[1], plan)
    assert lb.attend(q[:0], cache, rows[1], plan).shape == (0, 4, 64)
