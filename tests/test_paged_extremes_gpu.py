"""Attention over paged K/V caches where numbers are extreme but finite, against the 64-bit plain form."""
import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import LAYOUTS, SUB, U32, Cache, attend, dev, make, num, u_of

pytestmark = pytest.mark.gpu


def check(c, q, o, q_start, kv_len, nh, scale, qt, ot, score_error=0.0):
    """As check_attend of test_paged_gpu.py counts it, the scores' own error given by the case (0: they are exact in 32 bits):
    the output's half step, twice that of the weights' type on the weighted mean of |v|, 64 steps of 32 bits besides, and f16
    weights off by up to 2^-37 of the largest."""
    rows = q.shape[0]
    qn = num(q).reshape(rows, nh, c.hd)
    want, mag, total = ref.attend(qn, *c.values(), q_start, kv_len, c.table_h, scale, True, 0, np.full(qn.shape, 9.0))
    tol = u_of(ot) * np.abs(want) * 1.01 + mag * (2 * u_of(qt) + 2 * score_error + 64 * U32) + (SUB if ot == "f16" else 1e-30)
    tol += 2.0 ** -37 * total if qt == "f16" else 0
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
