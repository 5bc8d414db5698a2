"""The paged K/V cache operators against plain 64-bit forms (paged_ref.py).

Tolerances count roundings: a result rounded to a type is off by at most half a step, u = eps / 2 relative; 32-bit
arithmetic in between adds a few 2^-24 of the terms' magnitudes.  Codes and scales of 4-bit pages are equal, byte for byte."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as ref
from qasr import _lib

pytestmark = pytest.mark.gpu
IDS = {"f32": 0, "f16": 1, "bf16": 2, "mxfp4": 3}
U32 = 2.0 ** -24
SUB = 2.0 ** -25     # half of f16's step below 2^-14, where steps no longer shrink with the value


def T(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "mxfp4": torch.uint8}[name]


def u_of(name):
    import torch

    return torch.finfo(T(name)).eps / 2


def dev(x, t=None):
    import torch

    x = torch.from_numpy(np.ascontiguousarray(x)).to("cuda:0")
    return x if t is None else x.to(T(t))


def num(t):
    return t.double().cpu().numpy()


def stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


def table(n_pos, rot, theta=1e4):
    a = np.arange(n_pos)[:, None] * theta ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    return np.stack((np.cos(a), np.sin(a)), -1).astype(np.float32)


def rope_args(cs, rot, inter, w, eps=1e-6):
    return _lib.Rope(cs=cs.data_ptr() if cs is not None else None, n_pos=cs.shape[0] if cs is not None else 0,
                     rot_dim=rot, interleaved=int(inter), norm_w=w.data_ptr() if w is not None else None, eps=eps)


def rope_tol(x, w, ut):
    """per element: the rounding to the output's type, and in 32 bits: the norm's factor (sum, division, root: < hd / 2 + 8
    steps), the two products and the sum, each relative to the head's largest normed magnitude"""
    m = np.abs(x).max(-1, keepdims=True)
    if w is not None:
        m = m / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * np.abs(w).max()
    return 2 * m * U32 * (x.shape[-1] / 2 + 16) + ut * 2 * m * (1 + 1e-3) + SUB


# ------------------------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("xt,yt", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"),
                                   ("f32", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("heads,hd,rot", [(16, 128, 128), (3, 64, 32), (5, 256, 64), (2, 80, 20), (1, 96, 96),
                                          (7, 2, 2), (1, 1024, 1024), (4, 48, 16), (1, 128, 0)])
def test_rope(torch_dev, xt, yt, heads, hd, rot):
    import torch

    for inter, normed, rows, pad in [(False, True, 1, 0), (True, False, 37, 8), (True, True, 5, 3), (False, False, 130, 1)]:
        rng = np.random.default_rng(heads * hd + rows)
        x = dev(rng.standard_normal((rows, heads * hd + pad)).astype(np.float32) * 3, xt)
        w = dev(1 + 0.2 * rng.standard_normal(hd).astype(np.float32)) if normed else None
        cs_h = table(50, rot)
        cs, pos_h = dev(cs_h), rng.integers(0, 50, rows).astype(np.int32)
        pos_h[0] = 49
        pos = dev(pos_h)
        y = torch.full((rows, heads * hd + 2 * pad), 7.0, device="cuda:0", dtype=T(yt))
        r = rope_args(cs, rot, inter, w)
        _lib.check(_lib.load().qasr_op_rope(x.data_ptr(), IDS[xt], x.shape[1], pos.data_ptr(), rows, heads, hd,
                                            C.byref(r), y.data_ptr(), IDS[yt], y.shape[1], stream()))
        xs = num(x)[:, : heads * hd].reshape(rows, heads, hd)
        wn = num(w) if normed else None
        want = ref.rotate(xs, pos_h, cs_h, rot, inter, wn, float(np.float32(1e-6)))
        got = num(y)
        assert (got[:, heads * hd:] == 7).all()
        assert (np.abs(got[:, : heads * hd].reshape(want.shape) - want) <= rope_tol(xs, wn, u_of(yt))).all()


def test_rope_padding_rows_and_in_place(torch_dev):
    rng = np.random.default_rng(1)
    x_h = rng.standard_normal((6, 4 * 128)).astype(np.float16)
    cs_h, pos_h = table(20, 128), np.array([3, -1, 19, 20, 0, -2 ** 31], np.int32)
    x, cs, pos = dev(x_h), dev(cs_h), dev(pos_h)
    r = rope_args(cs, 128, False, None)
    _lib.check(_lib.load().qasr_op_rope(x.data_ptr(), 1, 512, pos.data_ptr(), 6, 4, 128, C.byref(r), x.data_ptr(), 1,
                                        512, stream()))
    got, xs = num(x), x_h.astype(np.float64).reshape(6, 4, 128)
    for i, p in enumerate(pos_h):
        if 0 <= p < 20:
            want = ref.rotate(xs[i:i + 1], pos_h[i:i + 1], cs_h, 128, False)
            assert (np.abs(got[i].reshape(1, 4, 128) - want) <= rope_tol(xs[i:i + 1], None, u_of("f16"))).all()
        else:
            assert np.array_equal(got[i], x_h[i].astype(np.float64))


@pytest.mark.parametrize("rows,heads,hd,rot,inter", [(700, 7, 128, 128, False), (700, 7, 128, 64, True),
                                                     (9, 3, 80, 20, False), (1500, 16, 256, 128, False)])
def test_rope_in_place_many_rows(torch_dev, rows, heads, hd, rot, inter):
    """in place gives what a second buffer gets, bit for bit, in every form of the kernel"""
    import torch

    rng = np.random.default_rng(rows + rot)
    x = dev(rng.standard_normal((rows, heads * hd)).astype(np.float32), "bf16")
    cs, w = dev(table(rows, rot)), dev(1 + 0.2 * rng.standard_normal(hd).astype(np.float32))
    pos, y = dev(rng.permutation(rows).astype(np.int32)), torch.empty_like(x)
    r = rope_args(cs, rot, inter, w)
    for out in (y, x):
        _lib.check(_lib.load().qasr_op_rope(x.data_ptr(), 2, heads * hd, pos.data_ptr(), rows, heads, hd, C.byref(r),
                                            out.data_ptr(), 2, heads * hd, stream()))
    torch.cuda.synchronize()
    assert torch.equal(x, y)


@pytest.mark.parametrize("rot", [2, 20, 64, 128])
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("first,n", [(0, 1), (0, 700), (131072 - 65, 65), ((1 << 40) - 3, 4), (5, 0)])
def test_rope_table_scaled(torch_dev, rot, kind, first, n):
    import torch

    if kind == 2 and rot == 2:
        return
    theta, factor, orig = 1e6, 4.0, 32768.0
    r = _lib.RopeScaling(rot_dim=rot, kind=kind, theta=theta, factor=factor, orig_ctx=orig, beta_fast=32.0, beta_slow=1.0)
    out = torch.full((n + 1, rot // 2, 2), 9.0, device="cuda:0")
    _lib.check(_lib.load().qasr_op_rope_table_scaled(C.byref(r), first, n, out.data_ptr(), stream()))
    ld = np.longdouble
    j = np.arange(rot // 2).astype(ld)
    th = ld(theta) * ld(factor) ** (ld(rot) / (rot - 2)) if kind == 2 else ld(theta)
    f, m = th ** (-2 * j / rot), ld(1)
    if kind == 1:
        f = f / factor
    if kind == 3:
        lo, hi = (rot * np.log(orig / (b * 2 * np.pi)) / (2 * np.log(theta)) for b in (32.0, 1.0))
        lo, hi = max(np.floor(lo), 0), min(np.ceil(hi), rot - 1)
        ramp = np.clip((j - lo) / max(hi - lo, 1e-3), 0, 1)
        f, m = f * (1 - ramp) + f / factor * ramp, ld(0.1) * np.log(ld(factor)) + 1
    a = (first + np.arange(n).astype(ld))[:, None] * f
    want = np.stack((np.cos(a) * m, np.sin(a) * m), -1)
    # half a step of f32, and the 64-bit angle: a frequency off by a few 2^-53 turns position p by p times that
    tol = U32 * 1.2 + 2.0 ** -50 * (first + n)
    got = num(out)
    assert (got[n:] == 9).all()
    if n:
        assert np.abs(got[:n] - want.astype(np.float64)).max() <= tol


# ------------------------------------------------------------------------------------------------ pages
class Cache:
    """A paged cache on the device with a page table of shuffled pages (unused entries -1)."""

    def __init__(self, rng, kv, page, nkv, hd, lens, spare=2, fill=True):
        import torch

        self.kv, self.page, self.nkv, self.hd = kv, page, nkv, hd
        per = [-(-n // page) for n in lens]
        self.n_pages = sum(per) + spare
        ids = rng.permutation(self.n_pages)
        self.table_h = np.full((len(lens), max(1, max(per))), -1, np.int32)
        at = 0
        for s, n in enumerate(per):
            self.table_h[s, :n] = ids[at:at + n]
            at += n
        self.table = dev(self.table_h)
        shape = (self.n_pages, nkv, page * hd * 17 // 32) if kv == "mxfp4" else (self.n_pages, nkv, page, hd)
        self.pools = []
        for i in range(2):
            if kv == "mxfp4":
                p = ref.Pool(np.zeros(shape, np.uint8), nkv, page, hd, i == 1)
                if fill:
                    p.raw[:] = rng.integers(0, 256, shape)
                    p.raw[:, :, page * hd // 2:] = rng.integers(122, 130, (*shape[:2], page * hd // 32))
                self.pools.append(dev(p.raw))
            else:
                self.pools.append(dev(rng.standard_normal(shape).astype(np.float32), kv))
        self.torch = torch

    def desc(self):
        return _lib.KvCache(k=self.pools[0].data_ptr(), v=self.pools[1].data_ptr(), page_table=self.table.data_ptr(),
                            n_seq=self.table_h.shape[0], max_pages=self.table_h.shape[1], n_pages=self.n_pages,
                            page_size=self.page, n_kv_heads=self.nkv, head_dim=self.hd, type=IDS[self.kv])

    def values(self):
        if self.kv == "mxfp4":
            return [ref.Pool(p.cpu().numpy(), self.nkv, self.page, self.hd, i == 1).values()
                    for i, p in enumerate(self.pools)]
        return [num(p) for p in self.pools]


def append(c, k, v, xt, seq, pos, r=None):
    keep = [dev(seq), dev(pos)]      # referenced until the kernel has finished
    _lib.check(_lib.load().qasr_op_kv_append(C.byref(c.desc()), k.data_ptr(), v.data_ptr(), IDS[xt], k.stride(0),
                                             v.stride(0), keep[0].data_ptr(), keep[1].data_ptr(), len(seq),
                                             C.byref(r) if r is not None else None, stream()))
    c.torch.cuda.synchronize()


def gather(c, seq, pos, k, v, yt):
    keep, ld = [dev(seq), dev(pos)], (k if k is not None else v).stride(0)
    _lib.check(_lib.load().qasr_op_kv_gather(C.byref(c.desc()), keep[0].data_ptr(), keep[1].data_ptr(), len(seq),
                                             k.data_ptr() if k is not None else None,
                                             v.data_ptr() if v is not None else None, IDS[yt], ld, ld, stream()))
    c.torch.cuda.synchronize()


@pytest.mark.parametrize("kv", ["f16", "bf16", "mxfp4"])
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,nkv,hd,rot", [(16, 1, 64, 64), (64, 8, 128, 128), (32, 3, 256, 64), (16, 2, 128, 20),
                                             (128, 5, 64, 16), (1024, 2, 128, 0)])
def test_append_and_gather(torch_dev, kv, xt, page, nkv, hd, rot):
    import torch

    for inter, normed, pad, lens in [(False, True, 0, [page, 3, 2 * page + 1]), (True, False, 5, [1]), (True, True, 8, [17, 40])]:
        rng = np.random.default_rng(hd + rot + page)
        c = Cache(rng, kv, page, nkv, hd, lens)
        had = [n // 3 for n in lens]
        seq = np.concatenate([np.full(n - h, s) for s, (h, n) in enumerate(zip(had, lens))]).astype(np.int32)
        pos = np.concatenate([np.arange(h, n) for h, n in zip(had, lens)]).astype(np.int32)
        order = rng.permutation(len(seq))
        seq, pos = seq[order], pos[order]
        # padding rows of each kind among the others
        seq = np.concatenate([seq, [-1, len(lens), 0, 0, 0]]).astype(np.int32)
        pos = np.concatenate([pos, [0, 0, -1, c.table_h.shape[1] * page, 2 ** 31 - 1]]).astype(np.int32)
        rows, width = len(seq), nkv * hd
        k = dev(rng.standard_normal((rows, width + pad)).astype(np.float32) * 2, xt)
        v = dev(rng.standard_normal((rows, width + 2 * pad)).astype(np.float32), xt)
        w = dev(1 + 0.2 * rng.standard_normal(hd).astype(np.float32)) if normed else None
        cs_h = table(max(lens), rot)
        cs = dev(cs_h)
        before = c.values()
        raw = [p.cpu().numpy().copy() for p in c.pools] if kv == "mxfp4" else None
        append(c, k, v, xt, seq, pos, rope_args(cs if rot else None, rot, inter, w))
        ks, vs = (num(t)[:, :width].reshape(rows, nkv, hd) for t in (k, v))
        real = rows - 5
        wn = num(w) if normed else None
        kk = ref.rotate(ks[:real], pos[:real], cs_h if rot else None, rot, inter, wn, float(np.float32(1e-6)))
        out = [torch.full((rows, width + 4), 9.0, device="cuda:0") for _ in range(2)]
        gather(c, seq, pos, *out, "f32")
        after = c.values()
        for j, x in enumerate((kk, vs[:real])):
            if kv == "mxfp4":
                p = ref.Pool(raw[j], nkv, page, hd, j == 1)
                for i in range(real):
                    p.write(c.table_h[seq[i], pos[i] // page], pos[i] % page, x[i].astype(np.float32))
                assert np.array_equal(p.raw.ravel(), c.pools[j].cpu().numpy().ravel())
            else:
                for i in range(real):
                    at = (c.table_h[seq[i], pos[i] // page], slice(None), pos[i] % page)
                    tol = rope_tol(ks[i], wn, u_of(kv)) if j == 0 else u_of(kv) * np.abs(x[i]) * 1.0001 + SUB
                    assert (np.abs(after[j][at] - x[i]) <= tol).all()
                    before[j][at] = after[j][at]
                assert np.array_equal(before[j], after[j])      # nothing else was touched
            got = num(out[j])
            assert (got[:, width:] == 9).all() and (got[real:] == 9).all()
            page_of = c.table_h[seq[:real], pos[:real] // page]
            assert np.array_equal(got[:real, :width].reshape(real, nkv, hd), after[j][page_of, :, pos[:real] % page])


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_append_fp4_borders(torch_dev, hd):
    """zeros, ties between codes, saturation, infinities and NaN, blocks that differ by many powers of two"""
    rng = np.random.default_rng(3)
    x = rng.choice([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6], (40, hd)).astype(np.float32)
    x *= rng.choice([-1, 1], x.shape) * 2.0 ** rng.integers(-30, 18, (40, 1))
    x[0] = 0
    x[1] = -0.0
    x[2, 3], x[3, 33], x[4, :] = np.inf, np.nan, 1e38
    x[5] *= np.float32(1 + 2.0 ** -20)
    x[6] = 1e-40
    for xt in ("f32", "bf16"):
        c = Cache(rng, "mxfp4", 16, 1, hd, [40], fill=False)
        k, v = dev(x, xt), dev(x[::-1], xt)
        append(c, k, v, xt, np.zeros(40, np.int32), np.arange(40, dtype=np.int32))
        for j, t in enumerate((k, v)):
            p = ref.Pool(np.zeros(tuple(c.pools[j].shape), np.uint8), 1, 16, hd, j == 1)
            for i in range(40):
                p.write(c.table_h[0, i // 16], i % 16, t[i:i + 1].float().cpu().numpy())
            assert np.array_equal(p.raw.ravel(), c.pools[j].cpu().numpy().ravel())


def test_gather_of_one_side_and_types(torch_dev):
    import torch

    rng = np.random.default_rng(4)
    for kv in ("f16", "bf16", "mxfp4"):
        c = Cache(rng, kv, 32, 2, 64, [50, 9])
        seq, pos = np.array([0, 1, 0, 1], np.int32), np.array([49, 8, 0, 9], np.int32)
        for yt in ("f32", "f16", "bf16"):
            out = torch.full((4, 128), 9.0, device="cuda:0", dtype=T(yt))
            for j in range(2):
                gather(c, seq, pos, out if j == 0 else None, out if j == 1 else None, yt)
                vals = c.values()[j]
                want = vals[c.table_h[seq, pos // 32], :, pos % 32].reshape(4, 128)
                assert (np.abs(num(out) - want) <= (0 if yt == "f32" else u_of(yt) * np.abs(want) + SUB)).all()


# ------------------------------------------------------------------------------------------------ attention
def attend(c, q, q_start, kv_len, nh, causal, window, scale, ot=None, o=None, max_q=None, max_kv=None, ws=None, qt=None,
           ldq=None):
    import torch

    qt = qt or ("f16" if q.dtype == torch.float16 else "bf16")
    ot = ot or qt
    rows = q.shape[0]
    if o is None:
        o = torch.full((rows, nh * c.hd), 9.0, device="cuda:0", dtype=T(ot))
    n = np.diff(q_start)
    a = _lib.PagedAttn(n_heads=nh, q_type=IDS[qt], o_type=IDS[ot], causal=int(causal), window=window, scale=scale,
                       max_q=int(n.max()) if max_q is None else max_q,
                       max_kv=int(max(kv_len)) if max_kv is None else max_kv)
    d, size = c.desc(), C.c_size_t()
    _lib.check(_lib.load().qasr_paged_attention_workspace(C.byref(d), C.byref(a), C.byref(size)))
    if ws is None:
        ws = torch.zeros(max(16, size.value), dtype=torch.uint8, device="cuda:0")
    keep = [dev(np.asarray(q_start, np.int32)), dev(np.asarray(kv_len, np.int32))]
    _lib.check(_lib.load().qasr_op_paged_attention(C.byref(d), C.byref(a), q.data_ptr(), q.stride(0), keep[0].data_ptr(),
                                                   keep[1].data_ptr(), rows, o.data_ptr(), o.stride(0), ws.data_ptr(),
                                                   ws.numel(), stream()))
    torch.cuda.synchronize()
    return o


def check_attend(c, q, o, q_start, kv_len, nh, causal, window, scale, qt, ot, values=None):
    """|o - exact| <= the output's half step of it, plus, of the weighted mean of |v|: twice the half step of the weights'
    type (each weight, and their sum), twice the 32-bit error of a score (hd products and sums of at most max |q|.|k|) and
    a few 2^-22 of exp and the running sums.  f16 weights below 2^-14 are multiples of 2^-24, off by up to 2^-25 where the
    largest is 2^12 at least: 2^-37 of the plain sum of |v| besides"""
    rows = q.shape[0]
    qn = num(q)[:, : nh * c.hd].reshape(rows, nh, c.hd)
    k, v = values or c.values()
    want = np.full(qn.shape, 9.0)
    want, mag, total = ref.attend(qn, k, v, q_start, kv_len, c.table_h, scale, causal, window, want)
    worst = np.abs(qn).sum(-1).max() * np.nanmax(np.abs(np.where(np.isfinite(k), k, 0))) * abs(scale) * U32 * 8
    tol = u_of(ot) * np.abs(want) * 1.01 + mag * (2 * u_of(qt) + 2 * worst + 64 * U32) + (SUB if ot == "f16" else 1e-30)
    tol += 2.0 ** -37 * total if qt == "f16" else 0
    got = num(o)[:, : nh * c.hd].reshape(qn.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], np.abs(got - want)[bad].max())


def make(rng, kv, page, nkv, g, hd, lens, nq, qt):
    c = Cache(rng, kv, page, nkv, hd, lens)
    q_start = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
    q = dev(rng.standard_normal((max(1, q_start[-1]), nkv * g * hd)).astype(np.float32), qt)
    return c, q, q_start, np.asarray(lens, np.int32)


LAYOUTS = [("f16", "f16"), ("bf16", "bf16"), ("mxfp4", "f16"), ("mxfp4", "bf16")]


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("nkv,g,hd,page", [(2, 2, 128, 16), (1, 1, 64, 64), (3, 5, 128, 32), (1, 20, 64, 128),
                                           (2, 4, 256, 16), (1, 2, 128, 1024)])
def test_attention_single_tokens(torch_dev, kv, qt, nkv, g, hd, page):
    rng = np.random.default_rng(nkv * hd + g)
    for lens in ([1], [15, 16, 17, 31, 32, 33], [130, 1, 0, 700, 64, 129, 2], [1500]):
        c, q, qs, kl = make(rng, kv, page, nkv, g, hd, lens, [1] * len(lens), qt)
        o = attend(c, q, qs, kl, nkv * g, True, 0, hd ** -0.5)
        check_attend(c, q, o, qs, kl, nkv * g, True, 0, hd ** -0.5, qt, qt)


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 20), (True, 1), (False, 50)])
@pytest.mark.parametrize("nkv,g,hd,page", [(2, 2, 128, 16), (1, 3, 64, 64), (1, 5, 256, 32)])
def test_attention_prompts(torch_dev, kv, qt, causal, window, nkv, g, hd, page):
    """ragged prompts, chunks on a context, verify passes; more queries than keys leaves rows empty"""
    rng = np.random.default_rng(nkv * hd + g)
    for lens, nq in (([5], [5]), ([40, 200, 3, 70], [40, 33, 3, 9]), ([10, 0, 90], [17, 4, 90]), ([300], [131])):
        c, q, qs, kl = make(rng, kv, page, nkv, g, hd, lens, nq, qt)
        for hints in ((None, None), (1000, 1 << 20)):     # either way of splitting the work
            o = attend(c, q, qs, kl, nkv * g, causal, window, hd ** -0.5, max_q=hints[0], max_kv=hints[1])
            check_attend(c, q, o, qs, kl, nkv * g, causal, window, hd ** -0.5, qt, qt)


@pytest.mark.parametrize("kv,qt", LAYOUTS)
def test_attention_long(torch_dev, kv, qt):
    """a long sequence beside short ones (the keys split over workgroups), alone and as a verify pass"""
    rng = np.random.default_rng(8)
    for lens, nq in (([9001], [1]), ([5000, 3, 40, 1], [1, 1, 1, 1]), ([4097, 700], [6, 5]), ([6000] + [30] * 40, [1] * 41)):
        c, q, qs, kl = make(rng, kv, 64, 2, 2, 128, lens, nq, qt)
        for max_q in (None, 1000):     # either way of splitting the work
            o = attend(c, q, qs, kl, 4, True, 0, 0.09, max_q=max_q)
            check_attend(c, q, o, qs, kl, 4, True, 0, 0.09, qt, qt)
            again = attend(c, q, qs, kl, 4, True, 0, 0.09, max_q=max_q)
            assert c.torch.equal(o, again)


@pytest.mark.parametrize("kv,qt", LAYOUTS)
def test_attention_f32_output_and_strides(torch_dev, kv, qt):
    import torch

    rng = np.random.default_rng(9)
    c, _, qs, kl = make(rng, kv, 32, 2, 2, 128, [100, 7], [40, 1], qt)
    for ldq, ldo in ((4 * 128 + 8, 4 * 128 + 4), (4 * 128 + 1, 4 * 128 + 3)):
        q = dev(rng.standard_normal((41, ldq)).astype(np.float32), qt)
        for ot, max_q in (("f32", 1), (qt, 1), ("f32", 1000), (qt, 1000)):
            o = torch.full((41, ldo), 9.0, device="cuda:0", dtype=T(ot))
            attend(c, q, qs, kl, 4, True, 0, 0.1, ot=ot, o=o, max_q=max_q)
            check_attend(c, q, o, qs, kl, 4, True, 0, 0.1, qt, ot)
            assert (num(o)[:, 512:] == 9).all()


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("nq", [1, 3, 60])
def test_attention_nothing_outside_the_keys(torch_dev, kv, qt, nq):
    """NaN in free pages, behind the last key, and in keys that a row does not see; bad page ids; rows of no sequence;
    understated sizes"""
    import torch

    rng = np.random.default_rng(10)
    lens = [70, 0, 200, 33]
    n = [min(nq, x) for x in lens]
    c, _, qs, kl = make(rng, kv, 16, 2, 2, 128, lens, n, qt)
    rows = int(qs[-1])
    q = dev(rng.standard_normal((rows + 4, 512)).astype(np.float32), qt)
    clean = c.values()
    for j, p in enumerate(c.pools):
        keep = torch.zeros((c.n_pages, 16), dtype=torch.bool)
        for s, length in enumerate(lens):
            for t in range(length):
                keep[c.table_h[s, t // 16], t % 16] = True
        if kv == "mxfp4":
            code_at, scale_at = ref.fp4_offsets(128, 16, j == 1)
            raw = p.cpu().numpy()
            for pg in range(c.n_pages):
                for t in range(16):
                    if not keep[pg, t]:
                        raw[pg, :, scale_at[t]] = 255
            p.copy_(torch.from_numpy(raw))
        else:
            p[~keep.to("cuda:0")[:, None].expand(-1, 2, -1)] = float("nan")
    for hints in ((None, None), (0, 0), (1 << 20, 1 << 30), (1000, 10 ** 4)):
        o = attend(c, q, qs, kl, 4, True, 0, 0.09, max_q=hints[0], max_kv=hints[1])
        check_attend(c, q, o, qs, kl, 4, True, 0, 0.09, qt, qt, values=clean)
        assert (num(o)[rows:] == 9).all()
    # NaN in the last key: only the rows that see it take it (in either way of splitting the work)
    before = [num(attend(c, q, qs, kl, 4, True, 0, 0.09, max_q=m)) for m in (1, 1000)]     # 1,000: as prompts
    ids, t = c.table_h[2, 199 // 16], 199 % 16
    for j, p in enumerate(c.pools):
        if kv == "mxfp4":
            p[int(ids), :, dev(ref.fp4_offsets(128, 16, j == 1)[1][t])] = 255
        else:
            p[int(ids), :, t] = float("inf") if j else float("nan")
    last = int(qs[3]) - 1
    same = np.arange(rows) != last
    for m, was in zip((1, 1000), before):
        o2 = num(attend(c, q, qs, kl, 4, True, 0, 0.09, max_q=m))
        assert np.isnan(o2[last]).all()
        assert np.array_equal(o2[:rows][same], was[:rows][same])


@pytest.mark.parametrize("kv,qt", LAYOUTS)
def test_attention_bad_entries(torch_dev, kv, qt):
    """page ids outside the pool are keys left out; lengths and row ranges outside the buffers are cut"""
    rng = np.random.default_rng(11)
    c, q, qs, kl = make(rng, kv, 16, 1, 2, 64, [100, 50, 64], [1, 20, 3], qt)
    c.table_h[0, 2], c.table_h[1, 0], c.table_h[1, 3], c.table_h[2, :] = c.n_pages, -5, 2 ** 31 - 1, -1
    c.table = dev(c.table_h)
    o = attend(c, q, qs, kl, 2, True, 0, 0.1)
    check_attend(c, q, o, qs, kl, 2, True, 0, 0.1, qt, qt)
    for qs2, kl2 in (([0, 1, 21, 30], [10 ** 9, -7, 64]), ([-3, 1, 1, 24], [20, 3, 64]), ([5, 3, 10, 12], [20, 50, 1]),
                     ([20, 0, 20, 0], [20, 50, 1]), ([7, 2 ** 31 - 1, -2 ** 31, 9], [20, 50, 1])):
        for max_q in (30, 1000):
            o = attend(c, q, qs2, kl2, 2, True, 0, 0.1, max_q=max_q, max_kv=100)
            check_attend(c, q, o, qs2, kl2, 2, True, 0, 0.1, qt, qt)


@pytest.mark.parametrize("kv,qt", LAYOUTS)
def test_attention_no_pages_and_odd_rows(torch_dev, kv, qt):
    """a cache without pages gives zeros; a row of q that is no number stays the only one"""
    import torch

    rng = np.random.default_rng(18)
    c, q, qs, kl = make(rng, kv, 16, 2, 2, 128, [90, 40], [37, 1], qt)
    want = [num(attend(c, q, qs, kl, 4, True, 0, 0.1, max_q=m)) for m in (1, 1000)]
    q[5, 128:256] = float("nan")
    q[20, 300] = float("inf")
    for m, was in zip((1, 1000), want):
        got = num(attend(c, q, qs, kl, 4, True, 0, 0.1, max_q=m)).reshape(38, 4, 128)
        was = was.reshape(38, 4, 128)
        assert np.isnan(got[5, 1]).all()
        same = np.ones((38, 4), bool)
        same[5, 1] = same[20, 2] = False
        assert np.array_equal(got[same], was[same])
    d = c.desc()
    for kw in (dict(n_pages=0, k=None, v=None), dict(max_pages=0, page_table=None)):
        for name, value in kw.items():
            setattr(d, name, value)
        c.desc = lambda: d
        for m in (1, 1000):
            o = attend(c, q, qs, kl, 4, True, 0, 0.1, max_q=m)
            assert (num(o) == 0).all()


@pytest.mark.parametrize("kv,qt", LAYOUTS)
def test_attention_extreme_scores(torch_dev, kv, qt):
    """one key far above the others, scores of the same size, a zero scale, large values"""
    rng = np.random.default_rng(12)
    c, q, qs, kl = make(rng, kv, 32, 2, 2, 128, [400, 90], [1, 50], qt)
    for scale, max_q in ((0.0, 1), (30.0, 1), (-2.0, 1), (0.0, 1000), (30.0, 1000), (-2.0, 1000)):
        o = attend(c, q, qs, kl, 4, True, 0, scale, max_q=max_q)
        check_attend(c, q, o, qs, kl, 4, True, 0, scale, qt, qt)
    if kv == "mxfp4":
        hd, page = 128, 32
        c.pools[1][:, :, page * hd // 2:] = dev(rng.choice([104, 127, 139, 140], (c.n_pages, 2, page * hd // 32)).astype(np.uint8))
    else:
        c.pools[1].mul_(20000.0 if kv == "f16" else 1e30)
        c.pools[1].clamp_(-60000 if kv == "f16" else -1e38, 60000 if kv == "f16" else 1e38)
    for scale, max_q in ((0.01, 1), (0.3, 1), (0.01, 1000), (0.3, 1000)):
        o = attend(c, q, qs, kl, 4, True, 0, scale, ot="f32", max_q=max_q)
        check_attend(c, q, o, qs, kl, 4, True, 0, scale, qt, "f32")


@pytest.mark.parametrize("kv,qt", LAYOUTS)
def test_attention_small_values(torch_dev, kv, qt):
    """K and V in the range where f16 has no leading one left (and the smallest scales of 4-bit pages): nothing is flushed"""
    rng = np.random.default_rng(17)
    c, q, qs, kl = make(rng, kv, 32, 2, 2, 128, [300, 45], [1, 45], qt)
    if kv == "mxfp4":
        for p in c.pools:
            p[:, :, 32 * 64:] = dev(rng.integers(104, 108, (c.n_pages, 2, 32 * 4)).astype(np.uint8))
    else:
        for p in c.pools:
            p.mul_(2.0 ** -16)
    for max_q in (1, 1000):
        o = attend(c, q, qs, kl, 4, True, 0, 3e4, ot="f32", max_q=max_q)
        check_attend(c, q, o, qs, kl, 4, True, 0, 3e4, qt, "f32")
        assert (o[kl.argmax()] != 0).any()


@pytest.mark.parametrize("kv,qt", LAYOUTS)
def test_attention_many_sequences(torch_dev, kv, qt):
    rng = np.random.default_rng(13)
    lens = rng.integers(0, 90, 300)
    nq = rng.integers(0, 4, 300)
    c, q, qs, kl = make(rng, kv, 16, 1, 2, 64, lens, nq, qt)
    for max_q in (None, 1000):
        o = attend(c, q, qs, kl, 2, True, 0, 0.12, max_q=max_q)
        check_attend(c, q, o, qs, kl, 2, True, 0, 0.12, qt, qt)


@pytest.mark.parametrize("kv", ["f16", "mxfp4"])
def test_offsets_past_32_bits(torch_dev, kv):
    """pages whose bytes lie more than 2^32 into their pool"""
    import torch

    hd, nkv, page = 128, 8, 1024
    block = page * hd * (17 / 32 if kv == "mxfp4" else 2)
    n_pages = int(2 ** 32 * 1.01 / (block * nkv)) + 2
    rng = np.random.default_rng(14)
    c = Cache(rng, kv, 16, nkv, hd, [1])
    c.page, c.n_pages = page, n_pages
    c.pools = [torch.empty(int(n_pages * nkv * block), dtype=torch.uint8, device="cuda:0") for _ in range(2)]
    c.table_h = np.array([[n_pages - 1, 0, n_pages - 2]], np.int32)
    c.table = dev(c.table_h)
    n = 2 * page + 5
    k = dev(rng.standard_normal((n, nkv * hd)).astype(np.float32))
    v = dev(rng.standard_normal((n, nkv * hd)).astype(np.float32))
    seq, pos = np.zeros(n, np.int32), np.arange(n, dtype=np.int32)
    append(c, k, v, "f32", seq, pos)
    out = [torch.empty_like(k) for _ in range(2)]
    gather(c, seq, pos, *out, "f32")
    ks, vs = (num(t) for t in (k, v))
    if kv == "mxfp4":
        ks, vs = (ref.fp4_value(*ref.fp4(x.reshape(n, nkv, hd).astype(np.float32))).reshape(n, -1) for x in (ks, vs))
    else:
        ks, vs = (x.astype(np.float16).astype(np.float64) for x in (ks, vs))
    assert np.array_equal(num(out[0]), ks) and np.array_equal(num(out[1]), vs)
    for nq in (1, 200):
        q = dev(rng.standard_normal((nq, 16 * hd)).astype(np.float32), "f16")
        o = attend(c, q, [0, nq], [n], 16, True, 0, 0.09)
        c2 = Cache(rng, "f16", page, nkv, hd, [1])      # the same values in three pages near the start, for the oracle
        c2.table_h = np.arange(3, dtype=np.int32)[None]
        vals = [np.zeros((3, nkv, page, hd)) for _ in range(2)]
        for x, y in zip(vals, (ks, vs)):
            x[pos // page, :, pos % page] = y.reshape(n, nkv, hd)
        check_attend(c2, q, o, [0, nq], [n], 16, True, 0, 0.09, "f16", "f16", values=vals)


# ------------------------------------------------------------------------------------------------ as they are used
@pytest.mark.parametrize("kv", ["f16", "mxfp4"])
def test_steps_of_a_session_batch(torch_dev, kv):
    """two prompts of different lengths and then single tokens: rotate q, append K and V, attend; against the plain forms
    over the values that the cache holds, and for f16 against the framework's contiguous cache"""
    import torch

    nh, nkv, hd, page = 4, 2, 128, 16
    rng = np.random.default_rng(15)
    lens, steps = np.array([37, 5]), 14
    c = Cache(rng, kv, page, nkv, hd, list(lens + steps))
    cs_h = table(64, hd, 1e6)
    cs, qw, kw = dev(cs_h), dev(1 + 0.1 * rng.standard_normal(hd).astype(np.float32)), dev(
        1 + 0.1 * rng.standard_normal(hd).astype(np.float32))
    had = np.zeros(2, np.int64)
    slots = int((lens + steps).sum())
    flat = [torch.zeros((slots, nkv * hd), dtype=torch.float16, device="cuda:0") for _ in range(2)]
    base = np.array([0, lens[0] + steps])
    ws = torch.zeros(1 << 27, dtype=torch.uint8, device="cuda:0")
    for step in range(steps + 1):
        new = lens if step == 0 else np.ones(2, np.int64)
        rows = int(new.sum())
        qkv = dev(rng.standard_normal((rows, (nh + 2 * nkv) * hd)).astype(np.float32))
        seq = np.repeat(np.arange(2), new).astype(np.int32)
        pos = np.concatenate([np.arange(h, h + n) for h, n in zip(had, new)]).astype(np.int32)
        q = torch.empty((rows, nh * hd), dtype=torch.float16, device="cuda:0")
        lib, ld = _lib.load(), qkv.shape[1]
        p_dev, s_dev = dev(pos), dev(seq)
        _lib.check(lib.qasr_op_rope(qkv.data_ptr(), 0, ld, p_dev.data_ptr(), rows, nh, hd,
                                    C.byref(rope_args(cs, hd, False, qw)), q.data_ptr(), 1, nh * hd, stream()))
        _lib.check(lib.qasr_op_kv_append(C.byref(c.desc()), qkv.data_ptr() + 4 * nh * hd,
                                         qkv.data_ptr() + 4 * (nh + nkv) * hd, 0, ld, ld, s_dev.data_ptr(),
                                         p_dev.data_ptr(), rows, C.byref(rope_args(cs, hd, False, kw)), stream()))
        had = had + new
        qs = np.concatenate([[0], np.cumsum(new)])
        o = attend(c, q, qs, had, nh, True, 0, hd ** -0.5, ws=ws)
        xs = num(qkv)[:, : nh * hd].reshape(rows, nh, hd)
        want = ref.rotate(xs, pos, cs_h, hd, False, num(qw), float(np.float32(1e-6)))
        assert (np.abs(num(q).reshape(want.shape) - want) <= rope_tol(xs, num(qw), u_of("f16"))).all()
        check_attend(c, q, o, qs, had, nh, True, 0, hd ** -0.5, "f16", "f16")
        if kv == "f16":
            slot = dev((base[seq] + pos).astype(np.int32))
            q2 = torch.empty_like(q)
            _lib.check(lib.qasr_op_qk_norm_rope(qkv.data_ptr(), rows, nh, nkv, hd, p_dev.data_ptr(), slot.data_ptr(),
                                                qw.data_ptr(), kw.data_ptr(), cs.data_ptr(), 1e-6, q2.data_ptr(),
                                                flat[0].data_ptr(), flat[1].data_ptr(), stream()))
            o2 = torch.empty((rows, nh * hd), dtype=torch.float32, device="cuda:0")
            start, length = dev(base[seq].astype(np.int32)), dev((pos + 1).astype(np.int32))
            _lib.check(lib.qasr_op_attention(q2.data_ptr(), nh * hd, flat[0].data_ptr(), flat[1].data_ptr(), nkv * hd,
                                             start.data_ptr(), length.data_ptr(), rows, nh, nkv, hd, hd ** -0.5,
                                             o2.data_ptr(), None, None, stream()))
            # q and K of either path differ by at most a step of f16 (2^-10), which moves a score by |q||k| scale 2^-9 or
            # so; the outputs then agree to a small part of the values' size
            assert (q - q2).abs().max() <= 2.0 ** -9 * q.abs().max()
            assert (o.float() - o2).abs().max() <= 0.02 * float(flat[1].abs().max())


@pytest.mark.parametrize("kv", ["f16", "mxfp4"])
def test_graph_replays_and_streams(torch_dev, kv):
    """a captured step replayed as the lengths grow on the device, eager work between the replays, a second graph with a
    workspace of its own on another stream; the workspace is left as it was found"""
    import torch

    nh, nkv, hd, page, n = 4, 2, 128, 16, 3
    rng = np.random.default_rng(16)
    c = Cache(rng, kv, page, nkv, hd, [3000, 200, 40])
    cs_h = table(3000, hd)
    cs = dev(cs_h)
    lib, r, d = _lib.load(), rope_args(cs, hd, False, None), c.desc()
    a = _lib.PagedAttn(n_heads=nh, q_type=1, o_type=1, causal=1, window=0, scale=0.09, max_q=1, max_kv=3000)
    size = C.c_size_t()
    _lib.check(lib.qasr_paged_attention_workspace(C.byref(d), C.byref(a), C.byref(size)))
    seq, qs = dev(np.arange(n, dtype=np.int32)), dev(np.arange(n + 1, dtype=np.int32))
    pos, kl = dev(np.array([2980, 180, 20], np.int32)), dev(np.array([2981, 181, 21], np.int32))
    qkv = dev(rng.standard_normal((n, (nh + 2 * nkv) * hd)).astype(np.float32))

    def step(q, o, ws, s):
        _lib.check(lib.qasr_op_rope(qkv.data_ptr(), 0, qkv.shape[1], pos.data_ptr(), n, nh, hd, C.byref(r), q.data_ptr(),
                                    1, nh * hd, s))
        _lib.check(lib.qasr_op_kv_append(C.byref(d), qkv.data_ptr() + 4 * nh * hd, qkv.data_ptr() + 4 * (nh + nkv) * hd,
                                         0, qkv.shape[1], qkv.shape[1], seq.data_ptr(), pos.data_ptr(), n, C.byref(r), s))
        _lib.check(lib.qasr_op_paged_attention(C.byref(d), C.byref(a), q.data_ptr(), nh * hd, qs.data_ptr(),
                                               kl.data_ptr(), n, o.data_ptr(), nh * hd, ws.data_ptr(), ws.numel(), s))

    bufs = [[torch.empty((n, nh * hd), dtype=torch.float16, device="cuda:0") for _ in range(2)]
            + [torch.zeros(max(16, size.value), dtype=torch.uint8, device="cuda:0")] for _ in range(3)]
    graphs = []
    for b in bufs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(*b, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    side = torch.cuda.Stream()
    for i in range(8):
        qkv.copy_(dev(rng.standard_normal(tuple(qkv.shape)).astype(np.float32)))
        torch.cuda.synchronize()
        graphs[0].replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        step(*bufs[2], stream())
        torch.cuda.synchronize()
        assert torch.equal(bufs[0][1], bufs[2][1]) and torch.equal(bufs[1][1], bufs[2][1])
        check_attend(c, bufs[2][0], bufs[2][1], qs.cpu().numpy(), kl.cpu().numpy(), nh, True, 0, 0.09, "f16", "f16")
        pos.add_(1)
        kl.add_(1)


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("hd", [64, 256])
def test_one_workspace_for_prompts_and_tokens(torch_dev, kv, qt, hd):
    """a captured prompt whose keys are shared out between workgroups, then single tokens, alternating on one workspace:
    each replay gives what an eager call on a fresh one does, and the workspace's counters end as they began"""
    import torch

    nkv, g, page = 2, 2, 32
    nh, scale = nkv * g, hd ** -0.5
    rng = np.random.default_rng(hd)
    lens = [2900, 4100]
    c, q, qs, kl = make(rng, kv, page, nkv, g, hd, lens, [150, 70], qt)
    lib, d, size = _lib.load(), c.desc(), C.c_size_t()
    a = [_lib.PagedAttn(n_heads=nh, q_type=IDS[qt], o_type=IDS[qt], causal=1, window=0, scale=scale, max_q=m, max_kv=4100)
         for m in (150, 1)]
    most = 0
    for x in a:
        _lib.check(lib.qasr_paged_attention_workspace(C.byref(d), C.byref(x), C.byref(size)))
        most = max(most, size.value)
    ws = torch.zeros(most, dtype=torch.uint8, device="cuda:0")
    starts, klen = [dev(qs), dev(np.arange(3, dtype=np.int32))], dev(kl)
    outs = [torch.empty((n, nh * hd), dtype=T(qt), device="cuda:0") for n in (220, 2)]
    g_ = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g_):
        for x, st, o in zip(a, starts, outs):
            _lib.check(lib.qasr_op_paged_attention(C.byref(d), C.byref(x), q.data_ptr(), nh * hd, st.data_ptr(),
                                                   klen.data_ptr(), o.shape[0], o.data_ptr(), nh * hd, ws.data_ptr(),
                                                   most, torch.cuda.current_stream().cuda_stream))
    for i in range(4):
        for o in outs:
            o.fill_(9.0)
        torch.cuda.synchronize()
        g_.replay()
        torch.cuda.synchronize()
        want = [attend(c, q, qs, kl, nh, True, 0, scale), attend(c, q[:2], [0, 1, 2], kl, nh, True, 0, scale)]
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
        check_attend(c, q, outs[0], qs, kl, nh, True, 0, scale, qt, qt)
        check_attend(c, q[:2], outs[1], [0, 1, 2], kl, nh, True, 0, scale, qt, qt)
        q.copy_(dev(rng.standard_normal(tuple(q.shape)).astype(np.float32), qt))
    assert int(ws[:4096].sum()) == 0


@pytest.mark.parametrize("kv,qt", LAYOUTS)
@pytest.mark.parametrize("nq,lens,window,max_kv,max_q", [
    ([70, 1, 128], [900, 3000, 2100], 0, None, None), ([70, 1, 128], [900, 3000, 2100], 100, None, None),
    ([300, 17], [2600, 30], 64, None, None), ([300, 17], [2600, 1900], 0, 1, None), ([200], [5000], 0, 64, None),
    ([128] * 6, [700] * 6, 0, None, None), ([65, 65], [17000, 100], 0, None, None), ([400], [3000], 300, None, 40),
    ([100, 0, 90], [6000, 9, 90], 5900, 1 << 30, 1 << 20)])
def test_attention_split_choices(torch_dev, kv, qt, nq, lens, window, max_kv, max_q):
    """every way in which rows, keys, windows and what was announced of them share a call out"""
    rng = np.random.default_rng(sum(nq) + window)
    c, q, qs, kl = make(rng, kv, 64, 2, 2, 128, lens, nq, qt)
    o = attend(c, q, qs, kl, 4, True, window, 0.09, max_kv=max_kv, max_q=max_q)
    check_attend(c, q, o, qs, kl, 4, True, window, 0.09, qt, qt)
