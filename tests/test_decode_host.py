"""CPU-only checks of the decode-step operators: refusals of the C entries before any device work,
and the plain forms that the GPU tests compare with."""
import pytest
import torch

import localstrm_b200 as lb
from localstrm_b200 import _lib
from tests import decode_util as U

OK, INVALID, WORKSPACE, UNSUPPORTED = 0, 1, 2, 4


def int4(**kw):
    a = dict(x=16, xd=1, rows=1, K=64, xs=64, packed=16, scales=16, sd=2, N=4, group=32, y=16, yd=0, ys=4, ws=None, wsb=0, stream=None)
    a.update(kw)
    return _lib.load().lss_int4_matvec(*a.values())


def test_int4_refusals():
    assert int4(rows=0) == OK
    for bad in (dict(rows=-1), dict(K=48), dict(K=0), dict(N=0), dict(xs=63), dict(ys=3), dict(xd=3), dict(yd=-1), dict(sd=0),
                dict(group=16), dict(group=96), dict(group=128), dict(K=320, xs=320, group=128), dict(x=None), dict(packed=None),
                dict(packed=8), dict(scales=17), dict(scales=None), dict(y=None)):
        assert int4(**bad) == INVALID, bad
    lib = _lib.load()
    assert lib.lss_int4_workspace_bytes(8, 64, 1, 4) == 0
    need = lib.lss_int4_workspace_bytes(9, 64, 1, 4)
    assert 0 < need < lib.lss_int4_workspace_bytes(9, 64, 0, 4)
    for bad in (dict(rows=9), dict(rows=9, ws=16, wsb=need - 1), dict(rows=9, ws=8, wsb=need)):
        assert int4(**bad) == WORKSPACE, bad


def plan(fn="lss_block_plan", **kw):
    a = dict(table=16, ts=4, width=4, lens=16, new=16, B=1, bs=16, free=16, blocks=8, n_free=16, cap=4, slots=16, pos=16, starts=16,
             granted=16, lens_out=16, n_free_out=16, stream=None)
    if fn == "lss_block_release":
        for k in ("cap", "slots", "pos", "starts", "granted"):
            del a[k]
    a.update(kw)
    return getattr(_lib.load(), fn)(*a.values())


@pytest.mark.parametrize("fn", ["lss_block_plan", "lss_block_release"])
def test_block_refusals(fn):
    for bad in (dict(table=None), dict(ts=3), dict(width=0), dict(B=-1), dict(bs=0), dict(blocks=0), dict(lens=None), dict(new=None),
                dict(free=None), dict(n_free=None), dict(lens_out=None), dict(n_free_out=None), dict(width=1 << 20, ts=1 << 20, bs=2048)):
        assert plan(fn, **bad) == INVALID, bad
    assert plan(fn, B=16385) == UNSUPPORTED
    if fn == "lss_block_plan":
        for bad in (dict(cap=-1), dict(slots=None), dict(pos=None), dict(starts=None), dict(granted=None)):
            assert plan(fn, **bad) == INVALID, bad


def append(**kw):
    a = dict(k=16, kt=128, kh=64, v=16, vt=128, vh=64, dt=1, T=2, heads=2, dim=64, kc=16, vc=16, ks=16, vs=16, blocks=8, bs=16, table=16,
             ts=4, width=4, starts=16, granted=16, lens=16, B=1, stream=None)
    a.update(kw)
    return _lib.load().lss_kv_append(*a.values())


def test_append_refusals():
    assert append(T=0) == OK and append(B=0) == OK
    for bad in (dict(dt=5), dict(T=-1), dict(heads=0), dict(dim=60), dict(dim=0), dict(bs=24), dict(bs=512), dict(bs=8), dict(kt=-1),
                dict(vh=-64), dict(table=None), dict(ts=3), dict(blocks=0), dict(k=None), dict(v=None), dict(kc=None), dict(vc=24),
                dict(ks=None), dict(vs=None), dict(starts=None), dict(granted=None), dict(lens=None)):
        assert append(**bad) == INVALID, bad
    assert append(B=16385) == UNSUPPORTED


def attend(**kw):
    a = dict(q=16, qt=256, qh=64, dt=1, T=2, hq=4, heads=2, dim=64, kc=16, vc=16, ks=16, vs=16, blocks=8, bs=16, table=16, ts=4, width=4,
             starts=16, granted=16, lens=16, B=1, scale=0.1, out=16, ot=256, oh=64, lse=None, ws=16, wsb=1 << 30, stream=None)
    a.update(kw)
    return _lib.load().lss_attend(*a.values())


def test_attend_refusals():
    lib = _lib.load()
    assert attend(T=0) == OK and attend(B=0) == OK
    for bad in (dict(dt=0), dict(dt=7), dict(T=-1), dict(heads=0), dict(hq=1), dict(hq=5), dict(bs=20), dict(qt=-1), dict(oh=63),
                dict(table=None), dict(width=5), dict(q=None), dict(out=None), dict(kc=8), dict(vs=None), dict(starts=None), dict(lens=None)):
        assert attend(**bad) == INVALID, bad
    assert attend(dim=96, oh=96) == UNSUPPORTED and attend(T=1 << 29) == UNSUPPORTED
    assert attend(ws=None) == WORKSPACE and attend(ws=24) == WORKSPACE
    assert attend(wsb=lib.lss_attend_workspace_bytes(64) - 1) == WORKSPACE
    assert 0 < lib.lss_attend_workspace_bytes(64) < lib.lss_attend_workspace_bytes(256) and lib.lss_attend_workspace_bytes(80) == 0


def test_cpu_tensors_fail_loudly():
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    w = lb.Int4Weight.quantize(torch.randn(8, 64), group=32)
    with pytest.raises(RuntimeError):
        lb.int4_matvec(torch.zeros(1, 64), w)
    with pytest.raises(RuntimeError):
        lb.sample_hidden(torch.zeros(1, 64), w, [])
    table = i(0, 1).view(1, 2)
    with pytest.raises(RuntimeError):
        lb.plan_blocks(table, i(3), i(1), i(1, 2), i(2), 16, 4)
    with pytest.raises(RuntimeError):
        lb.release_blocks(table, i(3), i(1), i(1, 2), i(2), 16)
    cache = lb.KVCache8.empty(4, 1, 16, 64, device="cpu")
    p = lb.StepPlan(i(0, 1), i(1), i(1))
    with pytest.raises(RuntimeError):
        lb.append_kv(cache, torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), table, p)
    with pytest.raises(RuntimeError):
        lb.attend(torch.zeros(1, 1, 64).half(), cache, table, p)


def test_quantize_round_trip():
    w = torch.randn(33, 128, generator=torch.Generator().manual_seed(0))
    w[5] = 0
    for group in (32, 64, 128):
        for dt, eps in ((torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -8)):
            q = lb.Int4Weight.quantize(w, group, dt)
            assert q.shape == (33, 128) and q.group == group and q.packed.shape == (33, 64)
            step = q.scales.float().repeat_interleave(group, 1)
            # half a step, and where the scale was rounded down the largest values end at code 7
            assert bool(((q.dequantize() - w).abs() <= step * (0.5 + 7 * 2 * eps) + 1e-30).all())
    assert bool((q.dequantize()[5] == 0).all())
    for group in (48, 16, 96, 192):
        with pytest.raises(ValueError):
            lb.Int4Weight.quantize(torch.randn(4, 192), group=group)
    with pytest.raises(ValueError):
        lb.Int4Weight.quantize(torch.randn(4, 40), group=40)


def test_plain_forms_on_known_values():
    # a row that needs a block, one that needs none, one that the free list does not hold any more, an idle one
    want, table = U.plan_reference([[7, -1], [3, -1], [4, -1], [5, -1]], [16, 3, 16, 9], [1, 2, 1, 0], [2, 6, 0, 0, 0, 0, 0, 0], 1, 16, 5)
    assert want == dict(slots=[2 * 16, 51, 52, -1, -1], positions=[16, 3, 4, 16, 0], starts=[0, 1, 3, 4, 4], granted=[1, 2, 0, 0],
                        lens=[17, 5, 16, 9], n_free=[0])
    assert table == [[7, 2], [3, -1], [4, -1], [5, -1]]
    assert U.scale_for(448.0) == 1.0 and U.scale_for(448.1) == 2.0 and U.scale_for(0.0) == 2.0 ** -126 and U.scale_for(7.0) == 2.0 ** -6
    x = torch.tensor([0.0, 1.0625, 1.1875, 448.0, 500.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -17.0], dtype=torch.float64)
    assert U.to_e4m3(x).tolist() == [0.0, 1.0, 1.25, 448.0, 448.0, 2.0 ** -9, 0.0, 2.0 ** -8, -16.0]
    assert torch.equal(U.to_e4m3(x), x.clamp(-448, 448).float().to(torch.float8_e4m3fn).double())


def test_int4_refuses_overlap_and_asks_for_workspace_for_long_rows():
    a = dict(x=1 << 20, xs=4000, rows=3, K=64, N=40, ys=4000)  # bf16 x, f32 y
    for bad in (dict(y=(1 << 20) + 2 * 63), dict(y=(1 << 20) - 4 * 39), dict(y=(1 << 20) + 2 * (2 * 4000 + 63)),
                dict(y=(1 << 20) + 8000 - 4 * 39, yd=0, ys=2000), dict(y=(1 << 20) + 8000 + 2 * 63, ys=2000)):
        assert int4(**{**a, **bad}) == INVALID, bad
    lib = _lib.load()
    for xd, k in ((1, 49152), (0, 16384)):
        assert lib.lss_int4_workspace_bytes(8, k, xd, 200000) == 0
        assert lib.lss_int4_workspace_bytes(1, 2 * k, xd, 200000) > 0
        assert int4(x=1 << 20, y=1 << 30, K=2 * k, xs=2 * k, xd=xd, N=200000, ys=200000) == WORKSPACE


def test_block_state_that_overlaps_in_part():
    for fn in ("lss_block_plan", "lss_block_release"):
        assert plan(fn, B=3, lens_out=20) == INVALID and plan(fn, B=3, lens=64, new=20) == INVALID


def test_stops_leaves_out_rows_without_a_token_of_their_own():
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    # rows: a token, idle, refused, the middle of a prompt, the end of a prompt, a token and no stop
    p = lb.StepPlan(i(0, 1, 1, 4, 6, 9, 10), i(1, 0, 0, 2, 3, 1), i(8, 5, 0, 6, 7, 9))
    codes = i(1, 1, 2, 1, 2, 0)
    assert p.stops(codes).tolist() == [1, 0, 0, 1, 2, 0]
    got = p.stops(codes, i(3, 3, 9, 7, 7, 9))
    assert got.tolist() == [1, 0, 0, 0, 2, 0] and got.dtype is torch.int32 and got.is_contiguous()
    for bad in ((codes.long(),), (codes[:5],), (codes, i(1, 2)), (codes, codes.float())):
        with pytest.raises(ValueError):
            p.stops(*bad)


def test_attend_refuses_results_shifted_over_the_queries():
    """Every row of a small layout against brute force: q at 4096 (bytes), 16-bit values."""
    rows = lambda at, st, sh, T, H: [at + 2 * (t * st + h * sh) for t in range(T) for h in range(H)]
    kinds = [(2, 4, 256, 64), (2, 4, 64, 128), (3, 2, 384, 64), (1, 4, 7, 64), (2, 2, 256, 64), (3, 4, 512, 128)]
    for T, hq, st, sh in kinds:
        for ot, oh in {(st, sh), (256, 64), (300, 72), (512, 128)}:
            if oh < 64 or (T > 1 and ot < (hq - 1) * oh + 64 and oh < (T - 1) * ot + 64):
                continue
            q = rows(4096, st, sh, T, hq)
            for at in [4096 + 16 * i for i in range(-200, 201, 3)] + [4096, 4096 + 2 * sh, 4096 + 2 * st, 4096 - 2 * st, 4096 + 128, 4096 + 126]:
                o = rows(at, ot, oh, T, hq)
                meet = any(abs(a - b) < 128 for a in q for b in o)
                apart = max(q) + 128 <= min(o) or max(o) + 128 <= min(q)
                got = attend(q=4096, qt=st, qh=sh, T=T, hq=hq, out=at, ot=ot, oh=oh, ws=None)
                if o == q or not meet and (apart or (ot, oh) == (st, sh)):
                    assert got == WORKSPACE, (T, hq, st, sh, ot, oh, at)
                elif meet:
                    assert got == INVALID, (T, hq, st, sh, ot, oh, at)


def test_attend_takes_results_head_by_head():
    for bad in (dict(ot=255), dict(ot=0), dict(ot=64, oh=127), dict(ot=65, oh=128), dict(T=3, ot=64, oh=191)):
        assert attend(out=1 << 20, ws=None, **bad) == INVALID, bad
    for good in (dict(ot=256), dict(ot=64, oh=128), dict(T=3, ot=70, oh=204), dict(T=1, ot=0), dict(hq=2, ot=128)):
        assert attend(out=1 << 20, ws=None, **good) == WORKSPACE, good


def test_int4_workspace_of_one_pass():
    """148 SMs: two to eight rows that fit some split of an SM's shared memory need none; others the other kernel's."""
    f = _lib.load().lss_int4_workspace_one_pass_bytes
    bf16, f32 = 1, 0
    for rows, k, dt, n in ((1, 49152, bf16, 200000), (1, 16384, f32, 200000), (8, 4096, bf16, 151936), (4, 4096, f32, 151936), (8, 14336, bf16, 4096),
                           (8, 14336, f32, 4096), (8, 11008, bf16, 4096), (8, 28672, bf16, 4096), (6, 8192, bf16, 151936)):
        assert f(rows, k, dt, n) == 0, (rows, k, dt, n)
    for rows, k, dt, n in ((8, 8192, bf16, 151936), (8, 8192, f32, 151936), (8, 4096, f32, 151936), (2, 49152, bf16, 200000), (8, 16384, f32, 128256)):
        assert f(rows, k, dt, n) > 0 and _lib.load().lss_int4_workspace_bytes(rows, k, dt, n) == 0, (rows, k, dt, n)
    for rows, k, dt, n in ((9, 4096, bf16, 128256), (64, 896, f32, 2000), (1, 98304, bf16, 200000)):
        assert f(rows, k, dt, n) == _lib.load().lss_int4_workspace_bytes(rows, k, dt, n) > 0
    assert f(0, 64, bf16, 4) == f(1, 0, bf16, 4) == f(1, 64, bf16, 0) == 0


def test_quantize_refuses_what_its_scales_cannot_hold():
    w = torch.ones(3, 64)
    w[1, 40] = 7 * 65504.0
    assert bool(lb.Int4Weight.quantize(w, 32).dequantize().isfinite().all())
    for bad in (7 * 65600.0, float("inf"), float("nan")):
        w[1, 40] = bad
        with pytest.raises(ValueError):
            lb.Int4Weight.quantize(w, 32)
    w[1, 40] = 7 * 65600.0
    assert bool(lb.Int4Weight.quantize(w, 32, torch.bfloat16).dequantize().isfinite().all())
