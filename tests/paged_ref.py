"""Plain 64-bit forms of the paged K/V cache operators (include/qasr.h), for the tests: numpy, one element at a time where
that is the plainest."""
import numpy as np

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def rotate(x, pos, cs, rot, inter, norm_w=None, eps=0.0):
    """x [rows][heads][hd] f64, cs [n_pos][rot/2][2] -> normed and rotated"""
    y = x.astype(np.float64).copy()
    if norm_w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * norm_w.astype(np.float64)
    if cs is None:
        return y
    z = y.copy()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        c, s = (cs[pos, i, j].astype(np.float64)[:, None] for j in (0, 1))
        z[..., a] = y[..., a] * c - y[..., b] * s
        z[..., b] = y[..., b] * c + y[..., a] * s
    return z


def fp4(x):
    """f32 [..., hd] -> codes uint8 [..., hd], scale bytes uint8 [..., hd / 32]"""
    b = x.astype(np.float32).astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    ok = np.isfinite(b).all(-1)
    b = np.where(ok[..., None], b, 0)
    amax = np.abs(b).max(-1)
    e = np.full(amax.shape, 13)
    for k in range(12, -24, -1):
        e = np.where(amax <= 6.0 * 2.0 ** k, k, e)
    a = np.minimum(np.abs(b) / 2.0 ** e[..., None], 6.0)
    d = np.abs(a[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    code = np.where(near[..., ::2].any(-1), 2 * near[..., ::2].argmax(-1), near.argmax(-1))
    code = np.where(ok[..., None], code | 8 * np.signbit(b), 0)
    return code.astype(np.uint8).reshape(x.shape), np.where(ok, e + 127, 255).astype(np.uint8)


def fp4_value(code, scale):
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7]
    e = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127))
    return v * np.repeat(e, 32, -1)


def fp4_offsets(hd, page, is_v):
    """byte offset of every (token, dim)'s code and of every (token, block)'s scale in a block"""
    t, d = np.arange(page)[:, None], np.arange(hd)[None]
    blk = np.arange(hd // 32)[None]
    if is_v:
        nd = hd // 16
        code = (t // 16) * 8 * hd + ((((t % 16) // 4) * 16 + d // nd) * 4 + t % 4) * nd // 2 + (d % nd) // 2
        scale = (t // 16) * (hd // 2) + blk * 16 + t % 16
    else:
        code = t * hd // 2 + ((d % 32) // 8) * (hd // 8) + (d // 32) * 4 + (d % 8) // 2
        scale = t * (hd // 32) + blk
    return code, page * hd // 2 + scale


class Pool:
    """One pool of MXFP4 pages as bytes [pages][heads][block]."""

    def __init__(self, raw, heads, page, hd, is_v):
        self.raw, self.page, self.hd = raw.reshape(-1, heads, page * hd * 17 // 32), page, hd
        self.code_at, self.scale_at = fp4_offsets(hd, page, is_v)

    def write(self, p, t, x):
        """x [heads][hd] f32 at token t of page p"""
        code, scale = fp4(x)
        at = self.code_at[t]
        for h in range(x.shape[0]):
            row = self.raw[p, h]
            for half in (0, 1):
                mask = 0xF0 if half == 0 else 0x0F
                row[at[half::2]] = (row[at[half::2]] & mask) | (code[h, half::2] << (4 * half))
            row[self.scale_at[t]] = scale[h]

    def values(self):
        """f64 [pages][heads][page][hd]"""
        b = self.raw[:, :, self.code_at]
        code = np.where(np.arange(self.hd) % 2, b >> 4, b & 15)
        return fp4_value(code, self.raw[:, :, self.scale_at])


def attend(q, k, v, q_start, kv_len, table, scale, causal, window, out):
    """q [rows][nh][hd]; k, v [pages][nkv][page][hd] values (f64) -> out (filled for rows of a sequence), and the
    weighted mean and the plain sum of |v| that the tolerances go by."""
    nh, nkv, page, n_pages = q.shape[1], k.shape[1], k.shape[2], k.shape[0]
    mag, total = np.zeros_like(out), np.zeros_like(out)
    edge = np.maximum.accumulate(np.clip(q_start, 0, len(q)))     # rows of sequences lie side by side
    for s in range(len(kv_len)):
        r0, n = edge[s], edge[s + 1] - edge[s]
        length = min(max(0, kv_len[s]), table.shape[1] * page)
        pos = np.arange(length)
        ids = table[s][pos // page]
        pos = pos[(ids >= 0) & (ids < n_pages)]
        ids = table[s][pos // page]
        for i in range(n):
            at = length - n + i
            ok = np.ones(len(pos), bool)
            if causal:
                ok &= pos <= at
            if window:
                ok &= pos > at - window
            for h in range(nh):
                kk, vv = (x[ids[ok], h // (nh // nkv), pos[ok] % page].astype(np.float64) for x in (k, v))
                if not len(kk):
                    out[r0 + i, h] = mag[r0 + i, h] = 0
                    continue
                x = kk @ q[r0 + i, h].astype(np.float64) * scale
                p = np.exp(x - x.max())
                p /= p.sum()
                out[r0 + i, h], mag[r0 + i, h], total[r0 + i, h] = p @ vv, p @ np.abs(vv), np.abs(vv).sum(0)
    return out, mag, total
