"""Attention over paged K/V caches, every group of 16 keys counted: V holds a mark in one dim for each group, so that an output
shows how much of each group's weight arrived.  The tolerance stays below what any one group brings (asserted on the plain
form before the kernel runs), so a group that is left out, or taken twice, where parts of the keys meet or the page ids of a
long part are read anew, fails."""
import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import LAYOUTS, SUB, U32, Cache, append, attend, dev, num, u_of

pytestmark = pytest.mark.gpu


def marked(rng, kv, qt, page, nkv, g, hd, lens, nq):
    """K of small random values, V[key] = 1 in the dim of the key's group and 0 elsewhere (both exact in every type of page)"""
    c = Cache(rng, kv, page, nkv, hd, lens)
    q_start = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
    q = dev(rng.standard_normal((int(q_start[-1]), nkv * g * hd)).astype(np.float32), qt)
    seq = np.concatenate([np.full(n, s) for s, n in enumerate(lens)]).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    v = np.zeros((len(seq), nkv, hd), np.float32)
    v[np.arange(len(seq)), :, pos // 16 % hd] = 1
    k = dev(rng.standard_normal((len(seq), nkv * hd)).astype(np.float32))
    append(c, k, dev(v.reshape(len(seq), -1)), "f32", seq, pos)
    return c, q, q_start, np.asarray(lens, np.int32)


def check(c, q, o, q_start, kv_len, nh, causal, window, scale, qt, ot, rows=None, values=None):
    """against the plain form; `rows`: only these"""
    n = q.shape[0]
    qn = num(q).reshape(n, nh, c.hd)
    k, v = values or c.values()
    want, mag, total = ref.attend(qn, k, v, q_start, kv_len, c.table_h, scale, causal, window, np.full(qn.shape, 9.0))
    # the largest score times 8 of its 2^-24; the output's half step; two half steps of the weights (V is 0 or 1: mag is the
    # output itself); 64 steps of 32 bits; f16 weights off by up to 2^-37 of the largest
    worst = np.abs(qn).sum(-1).max() * np.abs(k[np.isfinite(k)]).max() * abs(scale) * U32 * 8
    tol = u_of(ot) * np.abs(want) * 1.01 + mag * (2 * u_of(qt) + 2 * worst + 64 * U32) + (SUB if ot == "f16" else 1e-30)
    tol += 2.0 ** -37 * total if qt == "f16" else 0
    # what a group brings to each sequence's last row: more than twice the tolerance of its dim
    for s in range(len(kv_len)):
        keys, r = int(kv_len[s]), int(q_start[s + 1]) - 1
        at = np.arange(max(0, keys - window if window else 0) // 16 * 16, keys // 16 * 16)
        ids = c.table_h[s][at // c.page]
        at = at[(ids >= 0) & (ids < c.n_pages) & ((at >= keys - window) | (window == 0))]
        for h in range(nh):
            kk = k[c.table_h[s][at // c.page], h // (nh // c.nkv), at % c.page]
            p = np.exp(kk @ qn[r, h] * scale)
            p /= p.sum()
            groups, first = np.unique(at // 16, return_inverse=True)
            whole = np.bincount(first) == 16
            brings = np.bincount(first, p)
            assert (brings > 2 * tol[r, h, groups % c.hd])[whole].all()
    got = num(o)[:, : nh * c.hd].reshape(qn.shape)
    bad = ~(np.abs(got - want) <= tol)
    if rows is not None:
        bad &= rows[:, None, None]
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("page,hd", [(16, 128), (64, 128), (32, 64), (16, 256)])
def test_one_workgroup_walks_a_long_sequence(torch_dev, kv, qt, page, hd):
    """understated lengths: a few workgroups take hundreds of key tiles each, whose page ids come 64 tiles at a time; then a
    last key whose V is no number, which only one of two rows sees and which starts those long parts over"""
    rng = np.random.default_rng(page + hd)
    lens = [20011, 9000]
    c, q, qs, kl = marked(rng, kv, qt, page, 1, 2, hd, lens, [2, 2])
    o = attend(c, q, qs, kl, 2, True, 0, 0.02, max_q=1, max_kv=1)
    check(c, q, o, qs, kl, 2, True, 0, 0.02, qt, qt)
    clean = c.values()
    where = int(c.table_h[0, 20010 // page]), 20010 % page
    if kv == "mxfp4":
        c.pools[1][where[0], :, dev(ref.fp4_offsets(hd, page, True)[1][where[1]])] = 255
    else:
        c.pools[1][where[0], :, where[1]] = float("inf")
    o = attend(c, q, qs, kl, 2, True, 0, 0.02, max_q=1, max_kv=1)
    check(c, q, o, qs, kl, 2, True, 0, 0.02, qt, qt, rows=np.array([True, False, True, True]), values=clean)
    assert not np.isfinite(num(o)[1]).any()


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (False, 1500), (True, 1500)])
@pytest.mark.parametrize("max_q", [1, 1000])
def test_parts_of_long_keys(torch_dev, kv, qt, hd, causal, window, max_q):
    """items whose keys several workgroups share, in either kernel, causal and not, with and without a window"""
    rng = np.random.default_rng(hd)
    c, q, qs, kl = marked(rng, kv, qt, 32, 1, 2, hd, [3100, 5003, 40], [70, 9, 3])
    o = attend(c, q, qs, kl, 2, causal, window, 0.02, max_q=max_q)
    check(c, q, o, qs, kl, 2, causal, window, 0.02, qt, qt)


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("max_q", [1, 1000])
def test_parts_with_holes_and_odd_rows(torch_dev, kv, qt, hd, max_q):
    """the same with pages that are not there, f32 output in rows of odd stride, and a last key that is no number"""
    import torch

    rng = np.random.default_rng(hd + 1)
    c, q, qs, kl = marked(rng, kv, qt, 16, 1, 2, hd, [3000, 2900], [70, 5])
    full = c.table_h.copy()
    c.table_h[0, [0, 50, 101]], c.table_h[1, [60, 181]] = -1, c.n_pages
    c.table = dev(c.table_h)
    o = torch.full((75, 2 * hd + 3), 9.0, device="cuda:0")
    attend(c, q, qs, kl, 2, True, 0, 0.02, ot="f32", o=o, max_q=max_q)
    check(c, q, o, qs, kl, 2, True, 0, 0.02, qt, "f32")
    assert (num(o)[:, 2 * hd:] == 9).all()
    clean, last = c.values(), (int(full[0, 2999 // 16]), 2999 % 16)
    for j, p in enumerate(c.pools):
        if kv == "mxfp4":
            p[last[0], :, dev(ref.fp4_offsets(hd, 16, j == 1)[1][last[1]])] = 255
        elif j == 1:
            p[last[0], :, last[1]] = float("inf")
    attend(c, q, qs, kl, 2, True, 0, 0.02, ot="f32", o=o, max_q=max_q)
    check(c, q, o, qs, kl, 2, True, 0, 0.02, qt, "f32", rows=np.arange(75) != 69, values=clean)
    assert not np.isfinite(num(o)[69, : 2 * hd]).any()


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("max_q", [1, 1000])
def test_output_in_place_of_q(torch_dev, kv, qt, hd, max_q):
    """o written over q gives what a second buffer gets, bit for bit: whole items and shared ones, rows without a key, and rows
    of no sequence as they were"""
    rng = np.random.default_rng(hd)
    lens, nq = [3100, 0, 5003, 40, 1], [70, 2, 9, 60, 1]
    c, q, qs, kl = marked(rng, kv, qt, 32, 2, 3, hd, lens, nq)
    q = c.torch.cat((q, q[:3]))
    want = attend(c, q, qs, kl, 6, True, 0, 0.05, max_q=max_q)
    for _ in range(3):
        x = q.clone()
        attend(c, x, qs, kl, 6, True, 0, 0.05, o=x, max_q=max_q)
        assert c.torch.equal(x[:-3], want[:-3]) and c.torch.equal(x[-3:], q[-3:])


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("max_q", [1, 1000])
def test_long_sequences_among_many(torch_dev, kv, qt, max_q):
    """more sequences than a wave holds at once, long ones (shared out) beside short and empty ones in each stretch of 64"""
    rng = np.random.default_rng(21)
    lens, nq = rng.integers(0, 60, 150), rng.integers(0, 3, 150)
    for s, n in ((3, 2500), (63, 4100), (64, 3000), (100, 5000), (149, 2000)):
        lens[s], nq[s] = n, 2
    c, q, qs, kl = marked(rng, kv, qt, 16, 1, 2, 64, lens, nq)
    o = attend(c, q, qs, kl, 2, True, 0, 0.02, max_q=max_q)
    got, rows = num(o), np.concatenate([np.arange(qs[s], qs[s + 1]) for s in (3, 63, 64, 100, 149)])
    # every row against the plain form; the groups' shares of the long ones
    c2, q2 = c, q[dev(rows)]
    c2.table_h = c.table_h[[3, 63, 64, 100, 149]]
    long = c.torch.from_numpy(got[rows])
    check(c2, q2, long, np.arange(0, 11, 2), kl[[3, 63, 64, 100, 149]], 2, True, 0, 0.02, qt, qt)
    short = np.setdiff1d(np.arange(len(got)), rows)
    assert np.isfinite(got[short]).all() and (got[short] <= 1.01).all() and (got[short] >= 0).all()
    total = got[short].reshape(len(short), 2, 64).sum(-1)      # V has one mark a key: 1 a row, 0 without keys
    keys = np.repeat(kl, np.diff(qs))[short]
    sees = keys > np.maximum(np.repeat(np.diff(qs), np.diff(qs))[short] - 1 - (short - np.repeat(qs[:-1], np.diff(qs))[short]), 0)
    assert (np.abs(total - sees[:, None]) <= 4 * u_of(qt)).all()
