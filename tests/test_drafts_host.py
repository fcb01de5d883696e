"""CPU-only checks of the operators around drafted tokens and shared blocks: refusals of the C entries
before any device work, and the plain forms that the GPU tests compare with."""
import random

import pytest
import torch

import localstrm_b200 as lb
from localstrm_b200 import _lib
from tests import drafts_util as D

OK, INVALID, WORKSPACE, UNSUPPORTED = 0, 1, 2, 4


def rotate(**kw):
    # bf16, 2 tokens: 4 query heads and 2 key heads of 64; results apart from the inputs
    a = dict(q=1 << 20, qt=384, qh=64, qo=1 << 24, qot=256, qoh=64, hq=4, k=(1 << 20) + 512, kt=384, kh=64, ko=1 << 25, kot=128, koh=64, hk=2,
             dt=1, T=2, dim=64, pos=16, freqs=16, rot=64, inter=0, qw=16, kw=16, wd=1, eps=1e-6, stream=None)
    a.update(kw)
    return _lib.load().lss_norm_rotate(*a.values())


def test_rotate_refusals():
    assert rotate(T=0) == OK
    for bad in (dict(dt=3), dict(T=-1), dict(hq=0), dict(hk=0), dict(dim=63), dict(dim=0), dict(rot=33), dict(rot=-2), dict(rot=66), dict(qt=-1),
                dict(kh=-64), dict(wd=4), dict(q=None), dict(k=None), dict(pos=None), dict(freqs=None), dict(qo=None), dict(ko=None),
                dict(qoh=63), dict(koh=32), dict(qot=255), dict(kot=100)):
        assert rotate(**bad) == INVALID, bad
    assert rotate(dim=514, qoh=514, koh=514, qot=4 * 514, kot=2 * 514) == UNSUPPORTED and rotate(hq=70000) == UNSUPPORTED
    # results that lie over the inputs or each other in another way than exactly in place
    at = 1 << 20
    for bad in (dict(qo=at + 2), dict(qo=at, qot=256), dict(qo=at + 128), dict(ko=at + 512 + 128), dict(qo=at + 512, qot=384), dict(ko=at, kot=384),
                dict(qo=1 << 25), dict(ko=(1 << 24) + 64), dict(qo=at - 2 * 256, qot=384, qoh=64)):
        assert rotate(**bad) == INVALID, bad


def tree(**kw):
    a = dict(starts=16, granted=16, lens=16, B=2, parents=16, T=4, span=16, pos=16, stream=None)
    a.update(kw)
    return _lib.load().lss_tree_plan(*a.values())


def accept(**kw):
    a = dict(starts=16, granted=32, lens=64, B=2, parents=16, drafts=16, targets=16, codes=None, given=None, T=4, path=16, tokens=16, counts=16,
             lens_out=128, last=16, codes_out=16, stream=None)
    a.update(kw)
    return _lib.load().lss_tree_accept(*a.values())


def test_tree_refusals():
    assert tree(T=0) == OK and accept(T=0, B=0) == OK
    for bad in (dict(B=-1), dict(T=-1), dict(parents=None), dict(span=None), dict(span=20), dict(pos=None), dict(starts=None), dict(granted=None), dict(lens=None)):
        assert tree(**bad) == INVALID, bad
    for bad in (dict(B=-1), dict(T=-1), dict(parents=None), dict(drafts=None), dict(targets=None), dict(path=None), dict(tokens=None), dict(starts=None),
                dict(granted=None), dict(lens=None), dict(counts=None), dict(lens_out=None), dict(last=None), dict(codes_out=None),
                dict(lens_out=68), dict(lens_out=32), dict(lens_out=36)):
        assert accept(**bad) == INVALID, bad
    assert tree(B=16385) == UNSUPPORTED and accept(B=16385) == UNSUPPORTED


def attend_tree(**kw):
    a = dict(q=16, qt=256, qh=64, dt=1, T=2, hq=4, heads=2, dim=64, kc=16, vc=16, ks=16, vs=16, blocks=8, bs=16, table=16, ts=4, width=4,
             starts=16, granted=16, lens=16, B=1, scale=0.1, out=16, ot=256, oh=64, lse=None, ws=16, wsb=1 << 30, span=16, stream=None)
    a.update(kw)
    return _lib.load().lss_attend_tree(*a.values())


def test_attend_tree_refusals():
    assert attend_tree(T=0) == OK and attend_tree(B=0) == OK
    for bad in (dict(dt=0), dict(T=-1), dict(hq=5), dict(bs=20), dict(qt=-1), dict(oh=63), dict(q=None), dict(kc=8), dict(lens=None), dict(span=None),
                dict(span=20), dict(out=1 << 20, q=(1 << 20) + 128)):
        assert attend_tree(**bad) == INVALID, bad
    assert attend_tree(dim=96, oh=96) == UNSUPPORTED
    assert attend_tree(ws=None) == WORKSPACE and attend_tree(wsb=_lib.load().lss_attend_workspace_bytes(64) - 1) == WORKSPACE


def compact(**kw):
    a = dict(kc=16, vc=16, ks=16, vs=16, blocks=8, heads=2, bs=16, dim=64, table=16, ts=4, width=4, starts=16, granted=16, lens=16, B=1, path=16,
             counts=16, T=2, stream=None)
    a.update(kw)
    return _lib.load().lss_kv_compact(*a.values())


def copy(**kw):
    a = dict(kc=16, vc=16, ks=16, vs=16, blocks=8, heads=2, bs=16, dim=64, copies=16, n=1, stream=None)
    a.update(kw)
    return _lib.load().lss_kv_copy(*a.values())


def test_move_refusals():
    assert compact(T=0) == OK and compact(B=0) == OK and copy(n=0) == OK
    shared = (dict(heads=0), dict(bs=24), dict(dim=60), dict(dim=0), dict(blocks=0), dict(kc=None), dict(vc=None), dict(kc=24), dict(ks=None), dict(vs=None))
    for bad in shared + (dict(T=-1), dict(table=None), dict(ts=3), dict(B=-1), dict(starts=None), dict(granted=None), dict(lens=None), dict(path=None), dict(counts=None)):
        assert compact(**bad) == INVALID, bad
    for bad in shared + (dict(n=-1), dict(copies=None)):
        assert copy(**bad) == INVALID, bad
    assert compact(B=16385) == UNSUPPORTED and compact(heads=65537) == UNSUPPORTED
    assert copy(heads=65537) == UNSUPPORTED and copy(heads=65536, dim=65536, bs=256, n=1000) == UNSUPPORTED


def fork(**kw):
    a = dict(table=16, ts=4, width=4, lens=64, B=3, bs=16, src=16, dst=16, upto=None, n=1, shares=16, free=16, blocks=8, n_free=16, granted=16,
             copies=16, lens_out=64, n_free_out=16, stream=None)
    a.update(kw)
    return _lib.load().lss_block_fork(*a.values())


def give(**kw):
    a = dict(table=16, ts=4, width=4, lens=64, codes=128, keep=256, B=3, bs=16, shares=16, free=16, blocks=8, n_free=16, lens_out=64, n_free_out=16, stream=None)
    a.update(kw)
    return _lib.load().lss_block_give(*a.values())


def test_share_refusals():
    for bad in (dict(table=None), dict(ts=3), dict(width=0), dict(B=-1), dict(bs=0), dict(n=-1), dict(blocks=0), dict(lens=None), dict(lens_out=None),
                dict(src=None), dict(dst=None), dict(shares=None), dict(free=None), dict(n_free=None), dict(n_free_out=None), dict(granted=None),
                dict(copies=None), dict(lens_out=68)):
        assert fork(**bad) == INVALID, bad
    for bad in (dict(table=None), dict(ts=3), dict(width=0), dict(B=-1), dict(bs=0), dict(blocks=0), dict(lens=None), dict(lens_out=None), dict(free=None),
                dict(n_free=None), dict(n_free_out=None), dict(lens_out=72), dict(lens_out=132), dict(lens_out=252)):
        assert give(**bad) == INVALID, bad
    assert fork(B=16385) == UNSUPPORTED and fork(n=16385) == UNSUPPORTED and give(B=16385) == UNSUPPORTED
    assert give(B=16384, width=65537, ts=65537, lens=1 << 20, lens_out=1 << 20, codes=1 << 21, keep=1 << 22) == UNSUPPORTED


def test_cpu_tensors_fail_loudly():
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    table, cache = i(0, 1).view(1, 2), lb.KVCache8.empty(4, 1, 16, 64, device="cpu")
    p, x = lb.StepPlan(i(0, 1), i(1), i(1)), torch.zeros(1, 1, 64).half()
    t = lb.TreePlan(i(0, 1).view(1, 2), i(0), i(-1))
    for call in (lambda: lb.norm_rotate(x, x, i(0), torch.ones(32)), lambda: lb.plan_tree(p, i(-1)), lambda: lb.accept_drafts(p, t, i(3), i(4)),
                 lambda: lb.attend(x, cache, table, p, tree=t), lambda: lb.compact_kv(cache, table, p, i(0), i(1)),
                 lambda: lb.fork_blocks(table, i(3), i(0), i(0), i(0, 0), i(1, 2), i(2), 16), lambda: lb.copy_blocks(cache, i(0, 1).view(1, 2)),
                 lambda: lb.release_blocks(table, i(3), i(1), i(1, 2), i(2), 16, keep=i(1), shares=i(0, 0))):
        with pytest.raises(RuntimeError):
            call()


def test_plain_forms_on_known_values():
    #      0        two children, of which the second has two of its own; a second root
    #    1   2
    #       3 4
    parents = [-1, 0, 0, 2, 2, -1]
    span, positions = D.tree_reference(parents, [0, 6], [6], [16], 6)
    assert span == [[0, 5], [1, 1], [2, 3], [3, 1], [4, 1], [5, 1]] and positions == [10, 11, 11, 12, 12, 10]
    up = D.ancestors(parents)
    for i in range(6):
        for j in range(6):
            assert up[i][j] == (0 <= span[i][0] - span[j][0] < span[j][1])
    tokens, targets = [50, 7, 8, 9, 9, 1], [8, 0, 9, 33, 34, 2]
    assert D.accept_reference(parents, tokens, targets, None, None, [0, 6], [6], [16], 6) == ([0, 2, 3, -1, -1, -1], [8, 9, 33, -1, -1, -1], [3], [13], [33], [0])
    # a stop code behind token 2 ends the walk there; a given second token is kept although it was not sampled
    assert D.accept_reference(parents, tokens, targets, [0, 0, 2, 0, 0, 0], None, [0, 6], [6], [16], 6) == ([0, 2, -1, -1, -1, -1], [8, 9, -1, -1, -1, -1], [2], [12], [9], [2])
    assert D.accept_reference(parents, tokens, targets, None, [2], [0, 6], [6], [16], 6) == ([0, 1, -1, -1, -1, -1], [0, -1, -1, -1, -1, -1], [2], [12], [0], [0])
    # two samples of 20 tokens in blocks of 16; the second one's block that is not full is a copy
    want, table, shares = D.fork_reference([[3, 5], [-1, -1], [-1, -1]], [20, 0, 0], [0, 0], [1, 2], [20, 16], [0] * 8, [7, 6, 0, 0, 0, 0, 0, 0], 2, 16)
    assert want == dict(lens=[20, 20, 16], n_free=[1], granted=[20, 16], copies=[[5, 6], [-1, -1]])
    assert table == [[3, 5], [3, 6], [3, -1]] and shares == [0, 0, 0, 2, 0, 0, 0, 0]
    # rows 0 and 2 stop, row 1 keeps 16 tokens: block 3 stays with it
    assert D.give_reference(table, [20, 20, 16], [1, 0, 2], [0, 16, 0], shares, [7, 0, 0, 0, 0, 0, 0, 0], 1, 16) == \
        ([0, 16, 0], [3], [7, 5, 6, 0, 0, 0, 0, 0], [0, 0, 0, 0, 0, 0, 0, 0])


def test_random_trees_against_their_ancestors():
    rng = random.Random(3)
    for n in (1, 2, 17, 60):
        parents = D.random_tree(n, rng)
        span, positions = D.tree_reference(parents, [0, n], [n], [n + 5], n)
        up = D.ancestors(parents)
        assert sorted(s[0] for s in span) == list(range(n))
        for i in range(n):
            assert positions[i] == 5 + sum(up[i]) - 1
            assert [0 <= span[i][0] - span[j][0] < span[j][1] for j in range(n)] == up[i]
