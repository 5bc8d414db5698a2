"""The paged K/V cache operators without a GPU: pool sizes, the 4-bit format's plain form, refused calls."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as ref
from qasr import _lib

A = 1 << 20     # a well-aligned address that no refused call follows


def cache(**kw):
    return _lib.KvCache(**{**dict(k=A, v=A, page_table=A, n_seq=2, max_pages=4, n_pages=8, page_size=16, n_kv_heads=2,
                                  head_dim=128, type=_lib.T_F16), **kw})


def attn(**kw):
    return _lib.PagedAttn(**{**dict(n_heads=4, q_type=_lib.T_F16, o_type=_lib.T_F16, causal=1, window=0, scale=0.1,
                                    max_q=1, max_kv=64), **kw})


def rope(**kw):
    return _lib.Rope(**{**dict(cs=A, n_pos=64, rot_dim=128, interleaved=0, norm_w=None, eps=0.0), **kw})


def refused(rc, code=1):
    assert rc == code, rc
    assert _lib.load().qasr_last_error()


@pytest.mark.parametrize("t,page,hd,block", [(1, 16, 64, 2048), (2, 64, 128, 16384), (3, 16, 64, 544),
                                             (3, 64, 128, 4352), (3, 1024, 256, 139264)])
def test_pool_bytes(t, page, hd, block):
    n = C.c_size_t()
    _lib.check(_lib.load().qasr_kv_pool_bytes(C.byref(cache(type=t, page_size=page, head_dim=hd, n_pages=70000,
                                                            n_kv_heads=8)), C.byref(n)))
    assert n.value == 70000 * 8 * block


BAD_CACHE = [dict(type=0), dict(type=4), dict(head_dim=96), dict(head_dim=0), dict(page_size=8), dict(page_size=48),
             dict(page_size=2048), dict(n_kv_heads=0), dict(n_pages=-1), dict(n_seq=-1), dict(max_pages=-1),
             dict(page_size=1024, max_pages=1 << 21)]
BAD_POOLS = [dict(k=None), dict(v=None), dict(k=A + 8), dict(page_table=None), dict(page_table=A + 2)]


@pytest.mark.parametrize("kw", BAD_CACHE + BAD_POOLS)
def test_cache_refused(kw):
    lib, c = _lib.load(), cache(**kw)
    n = C.c_size_t()
    if kw in BAD_CACHE:
        refused(lib.qasr_kv_pool_bytes(C.byref(c), C.byref(n)))
        refused(lib.qasr_paged_attention_workspace(C.byref(c), C.byref(attn()), C.byref(n)))
    refused(lib.qasr_op_kv_append(C.byref(c), A, A, 1, 256, 256, A, A, 3, None, None))
    refused(lib.qasr_op_kv_gather(C.byref(c), A, A, 3, A, A, 1, 256, 256, None))
    refused(lib.qasr_op_paged_attention(C.byref(c), C.byref(attn()), A, 512, A, A, 3, A, 512, A, 1 << 40, None))


@pytest.mark.parametrize("kw", [dict(rot_dim=130), dict(rot_dim=7), dict(rot_dim=-2), dict(n_pos=-1), dict(cs=A + 4),
                                dict(norm_w=A + 1), dict(norm_w=A, eps=-1.0), dict(norm_w=A, eps=float("nan"))])
def test_rope_refused(kw):
    lib, r = _lib.load(), rope(**kw)
    refused(lib.qasr_op_rope(A, 1, 256, A, 3, 2, 128, C.byref(r), A, 1, 256, None))
    refused(lib.qasr_op_kv_append(C.byref(cache()), A, A, 1, 256, 256, A, A, 3, C.byref(r), None))


def test_rope_arguments_refused():
    lib, r = _lib.load(), rope()
    ok = [A, 1, 256, A, 3, 2, 128, C.byref(r), A, 1, 256, None]
    for at, bad in [(0, None), (0, A + 1), (1, 3), (1, -1), (2, 255), (2, 1 << 62), (3, None), (3, A + 1), (4, -1),
                    (5, 0), (6, 127), (6, 0), (6, 2048), (7, None), (8, None), (9, 3), (9, 0), (10, 255)]:
        refused(lib.qasr_op_rope(*ok[:at], bad, *ok[at + 1:]))
    refused(lib.qasr_op_rope(A, 1, 256, A, 1 << 30, 65536, 2, C.byref(r), A, 1, 1 << 20, None))
    refused(lib.qasr_op_rope(A, 1, 256, A, 3, 2, 128, C.byref(r), A, 1, 512, None))     # in place, another stride
    _lib.check(lib.qasr_op_rope(None, 1, 256, None, 0, 2, 128, C.byref(r), None, 1, 256, None))   # no rows: nothing


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=3), dict(kind=4), dict(kind=-1), dict(theta=0.0),
                                dict(theta=float("inf")), dict(kind=1, factor=0.5), dict(kind=2, rot_dim=2),
                                dict(kind=3, orig_ctx=0.0), dict(kind=3, theta=1.0), dict(kind=3, beta_fast=0.5)])
def test_rope_table_refused(kw):
    r = _lib.RopeScaling(**{**dict(rot_dim=64, kind=0, theta=1e6, factor=2.0, orig_ctx=4096, beta_fast=32.0,
                                   beta_slow=1.0), **kw})
    refused(_lib.load().qasr_op_rope_table_scaled(C.byref(r), 0, 16, A, None))


def test_rope_table_arguments_refused():
    lib, r = _lib.load(), _lib.RopeScaling(rot_dim=64, kind=0, theta=1e6, factor=1.0)
    for a in [(None, 0, 16, A), (C.byref(r), -1, 16, A), (C.byref(r), 0, -1, A), (C.byref(r), 0, 16, None),
              (C.byref(r), 0, 16, A + 4)]:
        refused(lib.qasr_op_rope_table_scaled(*a, None))


def test_append_gather_arguments_refused():
    lib, c = _lib.load(), cache()
    ok = [C.byref(c), A, A, 1, 256, 256, A, A, 3, None, None]
    for at, bad in [(0, None), (1, None), (1, A + 1), (2, None), (3, 3), (4, 255), (5, 255), (6, None), (6, A + 2),
                    (7, None), (8, -1), (8, 1 << 30)]:
        refused(lib.qasr_op_kv_append(*ok[:at], bad, *ok[at + 1:]))
    ok = [C.byref(c), A, A, 3, A, A, 1, 256, 256, None]
    for at, bad in [(0, None), (1, None), (2, None), (3, -1), (4, A + 1), (6, 3), (7, 255), (8, 255)]:
        refused(lib.qasr_op_kv_gather(*ok[:at], bad, *ok[at + 1:]))
    _lib.check(lib.qasr_op_kv_gather(C.byref(c), A, A, 3, None, None, 1, 0, 0, None))
    _lib.check(lib.qasr_op_kv_append(C.byref(c), None, None, 1, 256, 256, None, None, 0, None, None))


@pytest.mark.parametrize("kw", [dict(n_heads=3), dict(n_heads=0), dict(q_type=2, o_type=2), dict(q_type=0, o_type=0),
                                dict(o_type=2), dict(scale=float("inf")), dict(window=-1), dict(max_q=-1),
                                dict(max_kv=-1)])
def test_attention_refused(kw):
    lib, n = _lib.load(), C.c_size_t()
    refused(lib.qasr_paged_attention_workspace(C.byref(cache()), C.byref(attn(**kw)), C.byref(n)))
    refused(lib.qasr_op_paged_attention(C.byref(cache()), C.byref(attn(**kw)), A, 512, A, A, 3, A, 512, A, 1 << 40,
                                        None))


@pytest.mark.parametrize("scale,ok", [(2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False),
                                      (float("nan"), False)])
def test_attention_scale_fits_with_log2e(scale, ok):
    """scores are taken to base 2: a scale that is no longer finite then is refused, not answered with NaN"""
    lib, n = _lib.load(), C.c_size_t()
    rc = lib.qasr_paged_attention_workspace(C.byref(cache()), C.byref(attn(scale=scale)), C.byref(n))
    assert (rc == 0) == ok
    if not ok:
        refused(rc)
        refused(lib.qasr_op_paged_attention(C.byref(cache()), C.byref(attn(scale=scale)), A, 512, A, A, 3, A, 512, A,
                                            1 << 40, None))


def test_attention_arguments_refused():
    lib, n = _lib.load(), C.c_size_t()
    refused(lib.qasr_paged_attention_workspace(C.byref(cache()), C.byref(attn()), None))
    ok = [C.byref(cache()), C.byref(attn()), A, 512, A, A, 3, A, 512, A, 1 << 40, None]
    for at, bad in [(0, None), (1, None), (2, None), (2, A + 1), (3, 511), (4, None), (5, None), (6, -1), (6, 1 << 30),
                    (7, None), (8, 511), (8, 1 << 62)]:
        refused(lib.qasr_op_paged_attention(*ok[:at], bad, *ok[at + 1:]))
    _lib.check(lib.qasr_paged_attention_workspace(C.byref(cache()), C.byref(attn()), C.byref(n)))
    if n.value:
        for ws, size in ((None, n.value), (A, n.value - 1), (A + 8, n.value), (A + 64, n.value)):
            refused(lib.qasr_op_paged_attention(*ok[:9], ws, size, None), 6)
    _lib.check(lib.qasr_op_paged_attention(C.byref(cache()), C.byref(attn()), None, 512, None, None, 0, None, 512, None,
                                           0, None))


@pytest.mark.parametrize("kw,ld", [(dict(o_type=_lib.T_F32), (512, 512)), (dict(), (512, 520))])
def test_attention_in_place_of_another_type_or_stride(kw, ld):
    refused(_lib.load().qasr_op_paged_attention(C.byref(cache()), C.byref(attn(**kw)), A, ld[0], A, A, 3, A, ld[1], A, 1 << 40,
                                                None))


def test_fp4_plain_form():
    """borders between codes go to the even code, the exponent is the smallest that holds the block's maximum"""
    x = np.zeros((1, 32), np.float32)
    x[0, :15] = [6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -5, np.nextafter(np.float32(.25), np.float32(1)),
                 np.nextafter(np.float32(5), np.float32(9)), 0, -6]
    code, scale = ref.fp4(x)
    assert scale[0, 0] == 127
    assert code[0, :15].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 8, 10, 14, 1, 7, 0, 15]
    for amax, e in ((6.0, 0), (np.nextafter(np.float32(6), np.float32(7)), 1), (12, 1), (3, -1), (1e-9, -23), (0, -23),
                    (49152, 13), (1e30, 13)):
        assert ref.fp4(np.full((1, 32), amax, np.float32))[1][0, 0] == 127 + e
    assert ref.fp4_value(*ref.fp4(np.full((1, 32), 1e30, np.float32)))[0, 0] == 49152
    for bad in (np.nan, np.inf):
        x[0, 3] = bad
        assert np.isnan(ref.fp4_value(*ref.fp4(x))).all()
    for is_v in (False, True):
        for hd, page in ((64, 16), (128, 64), (256, 32)):
            code, scale = ref.fp4_offsets(hd, page, is_v)
            assert np.array_equal(np.unique(code), np.arange(page * hd // 2))     # each byte twice, low half first
            assert np.array_equal(np.sort(scale.ravel()), page * hd // 2 + np.arange(page * hd // 32))
            assert np.array_equal(code[:, 0::2], code[:, 1::2])
