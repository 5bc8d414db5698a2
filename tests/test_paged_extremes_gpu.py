"""Attention over paged K/V caches where numbers are extreme but finite, against the 64-bit plain form."""
import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import LAYOUTS, SUB, U32, append, attend, dev, make, num, u_of

pytestmark = pytest.mark.gpu


def check(c, q, o, q_start, kv_len, nh, scale, qt, ot, score_error=0.0, rest=0.0):
    """As check_attend of test_paged_gpu.py counts it, the scores' own error given by the case (0: they are exact in 32 bits):
    the output's half step, twice that of the weights' type on the weighted mean of |v|, 64 steps of 32 bits besides, and f16
    weights off by up to 2^-37 of the largest.  `rest`: how much of the largest |v| keys bring whose weights are not counted so."""
    rows = q.shape[0]
    qn = num(q).reshape(rows, nh, c.hd)
    want, mag, total = ref.attend(qn, *c.values(), q_start, kv_len, c.table_h, scale, True, 0, np.full(qn.shape, 9.0))
    tol = u_of(ot) * np.abs(want) * 1.01 + mag * (2 * u_of(qt) + 2 * score_error + 64 * U32) + (SUB if ot == "f16" else 1e-30)
    tol += 2.0 ** -37 * total if qt == "f16" else 0
    tol += rest * np.abs(c.values()[1]).max() if rest else 0
    got = num(o).reshape(qn.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("ot", ["bf16", "f32"])
@pytest.mark.parametrize("top", [1e37, 1e38, 3.3e38])
def test_largest_values_of_v(torch_dev, top, ot, hd):
    """bf16 V near the type's largest, one sign a dim: a mean of them is finite, whatever the number of keys.  (At 3.3e38 the
    output, off by at most two half steps of bf16, stays below 3.36e38 and so below the largest bf16, 3.39e38.)"""
    rng = np.random.default_rng(hd)
    lens, nq = [1, 700, 90, 6000, 17], [1, 3, 90, 2, 1]
    c, q, qs, kl = make(rng, "bf16", 32, 2, 2, hd, lens, nq, "bf16")
    sign = rng.choice([-1.0, 1.0], hd)
    c.pools[1].copy_(dev((rng.uniform(0.5, 1, tuple(c.pools[1].shape)) * sign * top).astype(np.float32), "bf16"))
    # |q . k| <= max |q|_1 max |k|, off by at most 8 of its 2^-24 (hd <= 256 products added in the matrix unit, and the scaling)
    reach = np.abs(num(q)).reshape(-1, 4, hd).sum(-1).max() * np.abs(c.values()[0]).max()
    for scale in (0.0, 0.09):
        for max_q in (1, 1000):     # either way of splitting the work
            o = attend(c, q, qs, kl, 4, True, 0, scale, ot=ot, max_q=max_q)
            check(c, q, o, qs, kl, 4, scale, "bf16", ot, reach * scale * U32 * 8)


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("power", [4, 12, 20, 40, 100])
def test_scores_of_any_size(torch_dev, kv, qt, hd, power):
    """Small whole q, K whole (or multiples of 2^-6 in 4-bit pages): every q . k is exact in 32 bits.  Scaled by a power of two
    and log2 e, and less the row's maximum, a score is off by at most 4 * 2^-24 of the largest (two products, two maxima
    before and after one has moved).  Where scores that differ at all then differ by 40, only those equal to a row's largest
    have a weight to speak of, and equal ones are equal: no error of scores is left.  The up to 6,000 others bring at most
    6,000 e^-40 of the largest |v|, exactly and as computed (an output is that small where the largest keys' v is 0: there
    their weights' own errors show, which the scores' rounding leaves relative to themselves), so that much is let pass."""
    rng = np.random.default_rng(hd + power)
    lens, nq = [1, 700, 90, 6000, 17], [1, 3, 90, 2, 1]
    c, q, qs, kl = make(rng, kv, 32, 2, 2, hd, lens, nq, qt)
    q.copy_((2 * q).round().clamp_(-8, 8))
    if kv != "mxfp4":
        c.pools[0].copy_((3 * c.pools[0]).round())
    k = c.values()[0].transpose(0, 2, 1, 3).reshape(-1, 2, hd)
    top = max(np.abs(num(q).reshape(-1, 2, 2, hd)[:, h].reshape(-1, hd) @ k[:, h].T).max() for h in (0, 1))
    assert top < 2 ** 16 and (k * 2.0 ** 6 == np.round(k * 2.0 ** 6)).all()
    err, gap = 4 * U32 * top * 2.0 ** power, (2.0 ** -6 if kv == "mxfp4" else 1.0) * 2.0 ** power
    rest = 0.0
    if gap - 2 * err > 40:
        err, rest = 0.0, 6000 * np.exp(-40.0)
    for scale in (2.0 ** power, -2.0 ** power):
        for max_q in (1, 1000):     # either way of splitting the work
            o = attend(c, q, qs, kl, 4, True, 0, scale, max_q=max_q)
            check(c, q, o, qs, kl, 4, scale, qt, qt, err, rest)


@pytest.mark.parametrize("size", [1.5e19, -1.5e19])
def test_scores_near_the_largest_f32(torch_dev, size):
    """one product of +-2.25e38 a score, the same for every key (times log2 e 3.25e38, which f32 still holds): the plain mean"""
    rng = np.random.default_rng(5)
    lens, nq = [1, 700, 90, 6000], [1, 3, 90, 2]
    c, q, qs, kl = make(rng, "bf16", 32, 2, 2, 128, lens, nq, "bf16")
    q.zero_()
    q.view(-1, 4, 128)[..., 5] = 1.5e19
    c.pools[0].zero_()
    c.pools[0][..., 5] = size
    for max_q in (1, 1000):
        o = attend(c, q, qs, kl, 4, True, 0, 1.0, max_q=max_q)
        check(c, q, o, qs, kl, 4, 1.0, "bf16", "bf16")


@pytest.mark.parametrize("kv", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_the_largest_value_of_the_type(torch_dev, kv, hd):
    """V at the type's largest value, one sign a dim: any mean of it is that value.  All keys but each sequence's first have
    the weight (1 + 1.1 u) / 2, which is rounded up by 0.9 of its u: that must not carry the output to infinity."""
    rng = np.random.default_rng(hd)
    lens, nq = [1, 3, 700, 90, 6000, 17], [1, 2, 30, 90, 2, 1]
    c, q, qs, kl = make(rng, kv, 32, 2, 2, hd, lens, nq, kv)
    top, u = float(c.torch.finfo(q.dtype).max), u_of(kv)
    sign = dev(rng.choice([-1.0, 1.0], hd).astype(np.float32), kv)
    c.pools[1].copy_((sign * top).expand_as(c.pools[1]))
    for p, x in ((c.pools[0], -1.0), (q.view(-1, 4, hd), 1.0)):
        p.zero_()
        p[..., 0] = x
    for s in range(len(lens)):
        c.pools[0][int(c.table_h[s, 0]), :, 0] = 0
    scale = float(-np.log((1 + 1.1 * u) / 2))
    for max_q in (1, 1000):     # either way of splitting the work
        o = attend(c, q, qs, kl, 4, True, 0, scale, max_q=max_q)
        # the weights' rounding and the output's half step, all of the value itself
        got, want = num(o).reshape(-1, 4, hd), num(sign) * top
        assert (np.abs(got - want) <= top * (2 * u + 64 * U32 + u * 1.01)).all()


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_means_of_one_value(torch_dev, kv, qt, hd):
    """V the same for every key: its mean is that value whatever the weights are rounded to, for they are divided by the sum of
    what they were rounded to.  At random scores, and with one key before 20,000 of 2^-27 of its weight, where f16 has no
    leading one left.  32-bit sums are off by 2^-24 for each of up to keys / 32 steps, twice, and 64 besides."""
    rng = np.random.default_rng(hd)
    lens, nq = [1, 700, 90, 20000], [1, 3, 90, 2]
    c, q, qs, kl = make(rng, kv, 32, 2, 2, hd, lens, nq, qt)
    seq = np.concatenate([np.full(n, s) for s, n in enumerate(lens)]).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    v = dev(np.full((len(seq), 2 * hd), 1.5, np.float32))
    k = rng.standard_normal((len(seq), 2, hd)).astype(np.float32)
    for scale in (0.09, float(27 * np.log(2))):
        if scale > 1:
            k[:] = 0
            k[..., 0] = np.where(pos == 0, 0, -1)[:, None]
            q.zero_()
            q.view(-1, 4, hd)[..., 0] = 1
        append(c, dev(k.reshape(len(seq), -1)), v, "f32", seq, pos)
        for max_q in (1, 1000):     # either way of splitting the work
            o = num(attend(c, q, qs, kl, 4, True, 0, scale, ot="f32", max_q=max_q))
            steps = 64 + 2 * np.repeat(kl, nq)[:, None] / 32
            assert (np.abs(o - 1.5) <= 1.5 * U32 * steps).all()
