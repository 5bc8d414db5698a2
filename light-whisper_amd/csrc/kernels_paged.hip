// Rotary positions, their table, and moving rows into and out of paged K/V caches (include/qasr.h, "paged K/V cache").
#include <algorithm>
#include <type_traits>

#include "paged_dev.h"

namespace qasr {

// ------------------------------------------------------------------------------------------------ table
// A thread takes one frequency and `run` positions: the angle's sine and cosine once, in 64 bits, and from there each next
// position by one rotation (4 multiply-adds in 64 bits; after 32 of them off by 2^-48 at most, the result is rounded to
// 24 bits).  Bound by the stores: neighbouring lanes hold neighbouring frequencies.  131,072 positions of 64: 67 MB in 13 us,
// 5.1 TB/s (an angle's own sine for each: 40 us).
__global__ __launch_bounds__(256) void k_rope_table(RopeFreqs f, int64_t first, int n_pos, int run, float2* __restrict__ cs) {
    const int half = f.rot / 2;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, p0 = i / half * run;
    if (p0 >= n_pos) return;
    const int j = (int)(i % half);
    double w = exp2(-2.0 * j / f.rot * f.log2_theta);
    const double ramp = f.kind == 3 ? fmin(fmax((j - f.lo) * f.inv_span, 0.0), 1.0) : f.kind == 1 ? 1.0 : 0.0;
    w = w * (1.0 - ramp) + w * f.inv_factor * ramp;
    double s, c, ds, dc;
    sincos((double)(first + p0) * w, &s, &c);
    sincos(w, &ds, &dc);
    float2* out = cs + p0 * half + j;
    for (int k = 0; k < run && p0 + k < n_pos; k++, out += half) {
        *out = make_float2((float)(c * f.mscale), (float)(s * f.mscale));
        const double t = fma(c, dc, -(s * ds));
        s = fma(s, dc, c * ds);
        c = t;
    }
}

void rope_table_scaled(const RopeFreqs& f, int64_t first, int n_pos, float* cs, hipStream_t s) {
    if (n_pos <= 0) return;
    // long runs once the chip is full without them
    const int64_t n = (int64_t)n_pos * (f.rot / 2);
    const int run = n >= 32 * 131072 ? 32 : n >= 8 * 65536 ? 8 : 1;
    k_rope_table<<<(unsigned)cdiv64(cdiv64(n_pos, run) * (f.rot / 2), 256), 256, 0, s>>>(f, first, n_pos, run, (float2*)cs);
}

// ------------------------------------------------------------------------------------------------ rows
template <typename A>
__device__ __forceinline__ A shfl_xor_t(A v, int o);
template <>
__device__ __forceinline__ float shfl_xor_t<float>(float v, int o) { return __shfl_xor(v, o); }
template <>
__device__ __forceinline__ double shfl_xor_t<double>(double v, int o) { return __shfl_xor(v, o); }

template <typename A>
__device__ __forceinline__ A fma_t(A a, A b, A c) {
    if constexpr (sizeof(A) == 8) return fma(a, b, c);
    else return fmaf(a, b, c);
}

__device__ __forceinline__ void lds_sync_wave() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// one head by one wave: x → buf[hd], normed and rotated in A's arithmetic
template <int XT, typename A>
__device__ void head_to_lds(const void* x, int64_t off, int hd, const RopeArgs& r, int pos, int lane, A* buf) {
    const auto* p = (const typename Elem<XT>::type*)x + off;
    A ss = 0;
    for (int d = lane; d < hd; d += 64) {
        const A v = (A)(float)p[d];
        buf[d] = v;
        ss += v * v;
    }
    lds_sync_wave();
    A inv = 1;
    if (r.norm_w) {
        for (int o = 32; o > 0; o >>= 1) ss += shfl_xor_t<A>(ss, o);
        inv = (A)1 / sqrt(ss / (A)hd + (A)r.eps);
        for (int d = lane; d < hd; d += 64) buf[d] = buf[d] * inv * (A)r.norm_w[d];
        lds_sync_wave();
    }
    if (r.cs)
        for (int i = lane; i < r.rot / 2; i += 64) {
            const int a = r.interleaved ? 2 * i : i, b = r.interleaved ? 2 * i + 1 : i + r.rot / 2;
            const A c = r.cs[((int64_t)pos * (r.rot / 2) + i) * 2], s = r.cs[((int64_t)pos * (r.rot / 2) + i) * 2 + 1];
            const A u = buf[a], v = buf[b];
            buf[a] = u * c - v * s;
            buf[b] = v * c + u * s;
        }
    lds_sync_wave();
}

// ---- the fast form: a thread takes 16 dims of a head, as two runs of 8 with 16-byte accesses: dims 8 u and rot/2 + 8 u in
// the half layout (each pair in one thread), 8 u and hd/2 + 8 u in the interleaved one, and the two halves of the dims that
// do not rotate likewise.  The head's hd / 16 threads are neighbours, so a run of lanes reads a run of bytes (a lane's 16
// dims in one piece: a third slower) and the norm's sum is a few xor-shuffles.  A thread takes up to four heads of its row
// with one read of the table.  Bound by memory: 8,192 rows of 16 heads, bf16, half of each turned, 69 MB in 18 us (3.9 TB/s;
// a copy of 2 GiB runs at 4.8).

// 8 elements as they were loaded; they are widened only when they are used, so that many loads are in flight
template <int T>
struct Raw8 {
    uint4 d[T == T_F32 ? 2 : 1];
};
template <int T>
__device__ __forceinline__ Raw8<T> raw8(const void* p, int64_t at) {
    Raw8<T> r;
    const uint4* s = (const uint4*)((const uint8_t*)p + at * (T == T_F32 ? 4 : 2));
    r.d[0] = s[0];
    if constexpr (T == T_F32) r.d[1] = s[1];
    return r;
}
template <int T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&v)[8]) {
    if constexpr (T == T_F32) {
        const float4 a = __builtin_bit_cast(float4, r.d[0]), b = __builtin_bit_cast(float4, r.d[1]);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else if constexpr (T == T_F16) {
        const f16x8 a = __builtin_bit_cast(f16x8, r.d[0]);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)a[i];
    } else {
        const bf16x8 a = __builtin_bit_cast(bf16x8, r.d[0]);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)a[i];
    }
}
template <int T>
__device__ __forceinline__ void load8(const void* p, int64_t at, float (&v)[8]) { widen8<T>(raw8<T>(p, at), v); }
template <int T>
__device__ __forceinline__ void store8(void* p, int64_t at, const float (&v)[8]) {
    if constexpr (T == T_F32) {
        *(float4*)((float*)p + at) = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)((float*)p + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else if constexpr (T == T_F16) {
        f16x8 a;
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = (_Float16)v[i];
        *(f16x8*)((uint16_t*)p + at) = a;
    } else {
        bf16x8 a;
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = (__bf16)v[i];
        *(bf16x8*)((uint16_t*)p + at) = a;
    }
}
// whether rows can be read and written 16 bytes at a time
static bool rows16(const Rows& r) { return ((uintptr_t)r.p & 15) == 0 && r.ld * elem_bytes(r.type) % 16 == 0; }
static bool units_ok(int hd, const RopeArgs& r) {
    return hd % 16 == 0 && (!r.cs || (r.rot % (r.interleaved ? 8 : 16) == 0 && ((uintptr_t)r.cs & 15) == 0)) && ((uintptr_t)r.norm_w & 15) == 0;
}

// a thread's place in a head, the same for all rows
struct Unit {
    int a, b;      // its two runs' first dims
    bool ta, tb;   // which of them rotate
};
__device__ __forceinline__ Unit unit_of(int u, int hd, const RopeArgs& r) {
    const int n = r.cs ? r.rot / 16 : 0;
    if (r.interleaved || n == 0) return Unit{8 * u, hd / 2 + 8 * u, r.cs && 8 * u < r.rot, r.cs && hd / 2 + 8 * u < r.rot};
    if (u < n) return Unit{8 * u, r.rot / 2 + 8 * u, true, true};
    return Unit{r.rot + 8 * (u - n), r.rot + (hd - r.rot) / 2 + 8 * (u - n), false, false};
}
// norm and rotation of the 16 dims; cs: the row's table entries of the unit (8 of cos, sin), w: its norm weights.
// `lanes`: threads of a head rounded up to a power of two; those without dims hold zeros
template <typename A>
__device__ __forceinline__ void turn16(A (&x)[2][8], const Unit& un, const RopeArgs& r, int hd, int lanes,
                                       const float (&cs)[16], const float (&w)[2][8]) {
    if (r.norm_w) {
        A ss = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fma_t<A>(x[0][i], x[0][i], fma_t<A>(x[1][i], x[1][i], ss));
        for (int o = lanes >> 1; o > 0; o >>= 1) ss += shfl_xor_t<A>(ss, o);
        A inv;
        if constexpr (sizeof(A) == 8) inv = 1.0 / sqrt(ss / (double)hd + (double)r.eps);
        else inv = rsqrtf(ss / (float)hd + r.eps);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[0][i] = x[0][i] * inv * (A)w[0][i];
            x[1][i] = x[1][i] * inv * (A)w[1][i];
        }
    }
    if (r.interleaved) {
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (k ? un.tb : un.ta)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const A c = cs[8 * k + 2 * i], s = cs[8 * k + 2 * i + 1], u = x[k][2 * i], v = x[k][2 * i + 1];
                x[k][2 * i] = fma_t<A>(u, c, -(v * s));
                x[k][2 * i + 1] = fma_t<A>(v, c, u * s);
            }
    } else if (un.ta) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const A c = cs[2 * i], s = cs[2 * i + 1], u = x[0][i], v = x[1][i];
            x[0][i] = fma_t<A>(u, c, -(v * s));
            x[1][i] = fma_t<A>(v, c, u * s);
        }
    }
}
__device__ __forceinline__ void load_unit_consts(const Unit& un, const RopeArgs& r, int p, float (&cs)[16],
                                                 float (&w)[2][8]) {
    const float4* row = (const float4*)(r.cs + (int64_t)p * r.rot);   // cos, sin of two pairs each
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float4 v = {};
        if (i < 2 ? un.ta : un.tb) v = row[r.interleaved ? (i < 2 ? un.a : un.b) / 4 + i % 2 : un.a / 2 + i];
        cs[4 * i] = v.x, cs[4 * i + 1] = v.y, cs[4 * i + 2] = v.z, cs[4 * i + 3] = v.w;
    }
    if (r.norm_w) {
        load8<T_F32>(r.norm_w, un.a, w[0]);
        load8<T_F32>(r.norm_w, un.b, w[1]);
    }
}

// grid: (row, group of HP heads) items, 256 / lanes of them a workgroup
template <int XT, int YT, int HP>
__global__ __launch_bounds__(256) void k_rope_units(const void* x, int64_t ldx, const int* __restrict__ pos, int rows,
                                                    int heads, int hd, int lanes_log2, RopeArgs r, void* y, int64_t ldy) {
    const int lanes = 1 << lanes_log2, u = threadIdx.x & (lanes - 1), groups = (heads + HP - 1) / HP;
    const bool mine = u < hd / 16;
    const Unit un = unit_of(u, hd, r);
    const int64_t items = (int64_t)rows * groups, step = (int64_t)gridDim.x * (256 >> lanes_log2);
    for (int64_t it = (int64_t)blockIdx.x * (256 >> lanes_log2) + (threadIdx.x >> lanes_log2); it < items; it += step) {
        const int row = (int)(it / groups), h0 = (int)(it % groups) * HP;
        const int p = r.cs ? pos[row] : 0;
        if (r.cs && (unsigned)p >= (unsigned)r.n_pos) continue;   // the whole group of lanes
        float cs[16], w[2][8];
        Raw8<XT> raw[HP][2];
        if (mine) {
#pragma unroll
            for (int k = 0; k < HP; k++) {   // (a head past the last one: the last one again, not stored)
                const int64_t at = row * ldx + (int64_t)min(h0 + k, heads - 1) * hd;
                raw[k][0] = raw8<XT>(x, at + un.a);
                raw[k][1] = raw8<XT>(x, at + un.b);
            }
            load_unit_consts(un, r, p, cs, w);
        }
#pragma unroll
        for (int k = 0; k < HP; k++) {
            float v[2][8] = {};
            if (mine) {
                widen8<XT>(raw[k][0], v[0]);
                widen8<XT>(raw[k][1], v[1]);
            }
            turn16<float>(v, un, r, hd, lanes, cs, w);
            if (mine && h0 + k < heads) {
                const int64_t at = row * ldy + (int64_t)(h0 + k) * hd;
                store8<YT>(y, at + un.a, v[0]);
                store8<YT>(y, at + un.b, v[1]);
            }
        }
    }
}
static int log2_up(int n) {
    int l = 0;
    while (1 << l < n) l++;
    return l;
}
static unsigned unit_grid(int64_t items, int lanes_log2) {   // enough workgroups to fill the chip several times over
    return (unsigned)std::min<int64_t>(cdiv64(items, 256 >> lanes_log2), 256 * 32);
}

// ---- any other: a head a wave, through LDS, element by element
constexpr int kRopeMaxHd = 1024;

template <int XT, int YT>
__global__ __launch_bounds__(64) void k_rope_any(const void* x, int64_t ldx, const int* __restrict__ pos, int rows, int heads,
                                                 int hd, RopeArgs r, void* y, int64_t ldy) {
    __shared__ float buf[kRopeMaxHd];
    const int lane = threadIdx.x;
    for (int64_t it = blockIdx.x; it < (int64_t)rows * heads; it += gridDim.x) {
        const int row = (int)(it / heads), head = (int)(it % heads);
        const int p = r.cs ? pos[row] : 0;
        if (r.cs && (unsigned)p >= (unsigned)r.n_pos) continue;
        head_to_lds<XT, float>(x, row * ldx + (int64_t)head * hd, hd, r, p, lane, buf);
        auto* o = (typename Elem<YT>::type*)y + row * ldy + (int64_t)head * hd;
        for (int d = lane; d < hd; d += 64) o[d] = (typename Elem<YT>::type)buf[d];
        lds_sync_wave();
    }
}

template <class F>
static void by_type(int t, F&& f) {
    if (t == T_F32) f(std::integral_constant<int, T_F32>{});
    else if (t == T_F16) f(std::integral_constant<int, T_F16>{});
    else f(std::integral_constant<int, T_BF16>{});
}

void rope_rows(const Rows& x, const int* pos, int rows, int heads, int hd, const RopeArgs& r, const Rows& y,
               hipStream_t s) {
    if (rows <= 0) return;
    by_type(x.type, [&](auto xt) {
        by_type(y.type, [&](auto yt) {
            constexpr int XT = xt(), YT = yt();
            if (units_ok(hd, r) && rows16(x) && rows16(y)) {
                const int ll = log2_up(hd / 16);
                // a head a thread while all of them fit the chip at once (900 x 16 heads, f32: 5.6 against 7.0 us with four);
                // past that, as many heads as 64 registers hold of x (8,192 x 16: f32 two, 28 us, one or four 30; f16 four,
                // 18 us, one 20)
                constexpr int HP = XT == T_F32 ? 2 : 4;
                const int64_t all = (int64_t)rows * heads;
                if (all << ll < 8 * 65536)
                    k_rope_units<XT, YT, 1><<<unit_grid(all, ll), 256, 0, s>>>(x.p, x.ld, pos, rows, heads, hd, ll, r,
                                                                               (void*)y.p, y.ld);
                else
                    k_rope_units<XT, YT, HP><<<unit_grid((int64_t)rows * cdiv(heads, HP), ll), 256, 0, s>>>(
                        x.p, x.ld, pos, rows, heads, hd, ll, r, (void*)y.p, y.ld);
            } else {
                k_rope_any<XT, YT><<<(unsigned)std::min<int64_t>((int64_t)rows * heads, 1 << 20), 64, 0, s>>>(
                    x.p, x.ld, pos, rows, heads, hd, r, (void*)y.p, y.ld);
            }
        });
    });
}

// ------------------------------------------------------------------------------------------------ append / gather
// 8 codes of values that share a scale byte (255: none)
__device__ __forceinline__ uint32_t fp4_codes8(const float (&v)[8], int scale) {
    if (scale == 255) return 0;
    const float f = __uint_as_float((uint32_t)scale << 23);   // v / f to the nearest code, ties to the even one, saturating
    uint32_t d = 0;
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[0], v[1], f, 0);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[2], v[3], f, 1);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[4], v[5], f, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[6], v[7], f, 3);
    return d;
}
__device__ __forceinline__ uint32_t top8(const float (&v)[8]) {   // the largest |v| by its bits, so that NaN counts
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}
// two runs of 8 dims (first dims a and b) of token t into an MXFP4 block; four neighbouring threads' runs are a block of 32
__device__ __forceinline__ void fp4_put(uint8_t* blk, uint32_t codes, int hd, int t, bool is_v, int a, int b,
                                        const float (&x)[2][8]) {
    uint32_t m[2] = {top8(x[0]), top8(x[1])};
#pragma unroll
    for (int k = 0; k < 2; k++) {
        m[k] = max(m[k], (uint32_t)__shfl_xor((int)m[k], 1));
        m[k] = max(m[k], (uint32_t)__shfl_xor((int)m[k], 2));
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int d = k ? b : a, sc = fp4_scale(__uint_as_float(m[k]));
        const uint32_t w = fp4_codes8(x[k], sc);
        if (is_v && hd == 64) {   // 4 dims lie together
            *(uint16_t*)(blk + fp4_v_code(hd, t, d)) = (uint16_t)w;
            *(uint16_t*)(blk + fp4_v_code(hd, t, d + 4)) = (uint16_t)(w >> 16);
        } else {
            *(uint32_t*)(blk + (is_v ? fp4_v_code(hd, t, d) : fp4_k_code(hd, t, d))) = w;
        }
        if (d % 32 == 0) blk[codes + (is_v ? fp4_v_scale(hd, t, d) : fp4_k_scale(hd, t, d))] = (uint8_t)sc;
    }
}

// a thread: 16 dims of K (even waves) or V (odd ones) of one KV head, as k_rope_units; hd is a power of two, so every thread
// has dims.  f32 rows of 8 heads into bf16 pages: 8,191 rows, 101 MB in 23.5 us (4.3 TB/s).  Into 4-bit pages 39 us for 76 MB:
// there K is in 64 bits (below), and its values pass through scratch memory, 80 bytes a thread (into 16-bit pages and in
// k_rope_units 48): turn16's two layouts store to different elements of one array behind a run-time branch
template <int XT, int CT>
__global__ __launch_bounds__(256) void k_kv_append_units(KvPages c, const void* k, const void* v, int64_t ldk, int64_t ldv,
                                                         const int* __restrict__ seq, const int* __restrict__ pos, int rows,
                                                         RopeArgs r) {
    // 4-bit pages: K in 64 bits up to the rounding to f32, so that a value next to a border between two codes gets its own
    typedef typename std::conditional<CT == T_MXFP4, double, float>::type A;
    const int lanes = c.hd / 16, ll = 31 - __builtin_clz(lanes), u = threadIdx.x & (lanes - 1);
    const bool is_v = threadIdx.x >> 6 & 1;
    const int64_t items = (int64_t)rows * c.nkv, step = (int64_t)gridDim.x * (128 >> ll);
    const uint32_t codes = (c.hd / 2) << c.page_shift;
    const int mine = (threadIdx.x >> 7) * (64 >> ll) + ((threadIdx.x & 63) >> ll);
    for (int64_t it = (int64_t)blockIdx.x * (128 >> ll) + mine; it < items; it += step) {
        const int row = (int)(it / c.nkv), head = (int)(it % c.nkv);
        const int p = pos[row];
        const int64_t at = r.cs && (unsigned)p >= (unsigned)r.n_pos ? -1 : page_block(c, seq[row], p, head);
        if (at < 0) continue;   // the whole group of lanes
        const int t = p & ((1 << c.page_shift) - 1);
        const Unit un = is_v ? Unit{8 * u, c.hd / 2 + 8 * u, false, false} : unit_of(u, c.hd, r);
        const void* src = is_v ? v : k;
        const int64_t from = row * (is_v ? ldv : ldk) + (int64_t)head * c.hd;
        const Raw8<XT> raw[2] = {raw8<XT>(src, from + un.a), raw8<XT>(src, from + un.b)};
        float y[2][8];
        if (is_v) {
            widen8<XT>(raw[0], y[0]);
            widen8<XT>(raw[1], y[1]);
        } else {
            float cs[16], w[2][8];
            load_unit_consts(un, r, p, cs, w);
            widen8<XT>(raw[0], y[0]);
            widen8<XT>(raw[1], y[1]);
            A x[2][8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[0][i] = y[0][i], x[1][i] = y[1][i];
            turn16<A>(x, un, r, c.hd, lanes, cs, w);
#pragma unroll
            for (int i = 0; i < 8; i++) y[0][i] = (float)x[0][i], y[1][i] = (float)x[1][i];
        }
        uint8_t* blk = (is_v ? c.v : c.k) + at;
        if constexpr (CT == T_MXFP4) {
            fp4_put(blk, codes, c.hd, t, is_v, un.a, un.b, y);
        } else {
            store8<CT>(blk, (int64_t)t * c.hd + un.a, y[0]);
            store8<CT>(blk, (int64_t)t * c.hd + un.b, y[1]);
        }
    }
}

// any other alignment or rotation: one (row, KV head) by one wave, through LDS
template <int XT, int CT>
__global__ __launch_bounds__(64) void k_kv_append_any(KvPages c, const void* k, const void* v, int64_t ldk, int64_t ldv,
                                                      const int* __restrict__ seq, const int* __restrict__ pos, int rows,
                                                      RopeArgs r) {
    typedef typename std::conditional<CT == T_MXFP4, double, float>::type A;   // as above
    __shared__ A buf[256];
    const int lane = threadIdx.x;
    const RopeArgs none{};
    for (int64_t it = blockIdx.x; it < (int64_t)rows * c.nkv; it += gridDim.x) {
        const int row = (int)(it / c.nkv), head = (int)(it % c.nkv);
        const int p = pos[row];
        const int64_t at = r.cs && (unsigned)p >= (unsigned)r.n_pos ? -1 : page_block(c, seq[row], p, head);
        if (at < 0) continue;
        const int t = p & ((1 << c.page_shift) - 1);
        for (int kv = 0; kv < 2; kv++) {
            uint8_t* blk = (kv ? c.v : c.k) + at;
            head_to_lds<XT, A>(kv ? v : k, row * (kv ? ldv : ldk) + (int64_t)head * c.hd, c.hd, kv ? none : r, p, lane, buf);
            if constexpr (CT == T_MXFP4) {
                const uint32_t codes = (c.hd / 2) << c.page_shift;
                if (16 * lane < c.hd) {
                    float x[2][8];
#pragma unroll
                    for (int i = 0; i < 16; i++) x[i / 8][i % 8] = (float)buf[i / 8 * (c.hd / 2) + 8 * lane + i % 8];
                    fp4_put(blk, codes, c.hd, t, kv, 8 * lane, c.hd / 2 + 8 * lane, x);
                }
            } else {
                typedef typename Elem<CT>::type E;
                for (int d = lane; d < c.hd; d += 64) ((E*)blk)[t * c.hd + d] = (E)(float)buf[d];
            }
            lds_sync_wave();
        }
    }
}

template <int XT, int CT>
static void launch_append(const KvPages& c, const Rows& k, const Rows& v, const int* seq, const int* pos, int rows,
                          const RopeArgs& r, hipStream_t s) {
    const int64_t items = (int64_t)rows * c.nkv;
    // in the half layout 4-bit blocks of 32 dims have to fall together on either side of rot / 2
    const bool blocks = CT != T_MXFP4 || !r.cs || r.interleaved || r.rot % 64 == 0;
    if (units_ok(c.hd, r) && rows16(k) && rows16(v) && blocks)
        k_kv_append_units<XT, CT><<<unit_grid(2 * items, log2_up(c.hd / 16)), 256, 0, s>>>(c, k.p, v.p, k.ld, v.ld, seq, pos,
                                                                                       rows, r);
    else
        k_kv_append_any<XT, CT><<<(unsigned)std::min<int64_t>(items, 1 << 20), 64, 0, s>>>(c, k.p, v.p, k.ld, v.ld, seq, pos,
                                                                                         rows, r);
}

void kv_append(const KvPages& c, const Rows& k, const Rows& v, const int* seq, const int* pos, int rows,
               const RopeArgs& r, hipStream_t s) {
    if (rows <= 0) return;
    by_type(k.type, [&](auto xt) {
        if (c.type == T_MXFP4) launch_append<xt(), T_MXFP4>(c, k, v, seq, pos, rows, r, s);
        else if (c.type == T_F16) launch_append<xt(), T_F16>(c, k, v, seq, pos, rows, r, s);
        else launch_append<xt(), T_BF16>(c, k, v, seq, pos, rows, r, s);
    });
}

// 8 dims from d on of token t
template <int CT>
__device__ __forceinline__ void block_values(const KvPages& c, const uint8_t* blk, bool is_v, int t, int d, float (&v)[8]) {
    if constexpr (CT == T_MXFP4) {
        const uint32_t codes = (c.hd / 2) << c.page_shift;
        uint32_t w;
        if (is_v && c.hd == 64)
            w = *(const uint16_t*)(blk + fp4_v_code(c.hd, t, d)) | (uint32_t)*(const uint16_t*)(blk + fp4_v_code(c.hd, t, d + 4)) << 16;
        else
            w = *(const uint32_t*)(blk + (is_v ? fp4_v_code(c.hd, t, d) : fp4_k_code(c.hd, t, d)));
        const uint32_t sc = blk[codes + (is_v ? fp4_v_scale(c.hd, t, d) : fp4_k_scale(c.hd, t, d))];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = fp4_value(w >> (4 * i) & 15, sc);
    } else {
        load8<CT>(blk, (int64_t)t * c.hd + d, v);
    }
}

// a thread: 8 dims of K and of V of one KV head.  8,191 rows of 8 heads from 4-bit pages to f32: 76 MB in 18 us (4.2 TB/s)
template <int CT, int YT, bool WIDE>
__global__ __launch_bounds__(256) void k_kv_gather(KvPages c, const int* __restrict__ seq, const int* __restrict__ pos,
                                                   int rows, void* k, void* v, int64_t ldk, int64_t ldv) {
    const int lanes = c.hd / 8, ll = 31 - __builtin_clz(lanes), d = 8 * (threadIdx.x & (lanes - 1));
    const int64_t items = (int64_t)rows * c.nkv, step = (int64_t)gridDim.x * (256 >> ll);
    for (int64_t it = (int64_t)blockIdx.x * (256 >> ll) + (threadIdx.x >> ll); it < items; it += step) {
        const int row = (int)(it / c.nkv), head = (int)(it % c.nkv), p = pos[row];
        const int64_t at = page_block(c, seq[row], p, head);
        if (at < 0) continue;
        const int t = p & ((1 << c.page_shift) - 1);
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            void* y = kv ? v : k;
            if (!y) continue;
            const int64_t to = row * (kv ? ldv : ldk) + (int64_t)head * c.hd + d;
            float x[8];
            block_values<CT>(c, (kv ? c.v : c.k) + at, kv, t, d, x);
            if constexpr (WIDE) {
                store8<YT>(y, to, x);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) ((typename Elem<YT>::type*)y)[to + i] = (typename Elem<YT>::type)x[i];
            }
        }
    }
}

template <int CT, int YT>
static void launch_gather(const KvPages& c, const int* seq, const int* pos, int rows, const Rows& k, const Rows& v,
                          hipStream_t s) {
    const unsigned grid = unit_grid((int64_t)rows * c.nkv, log2_up(c.hd / 8));
    if (rows16(k) && rows16(v))
        k_kv_gather<CT, YT, true><<<grid, 256, 0, s>>>(c, seq, pos, rows, (void*)k.p, (void*)v.p, k.ld, v.ld);
    else
        k_kv_gather<CT, YT, false><<<grid, 256, 0, s>>>(c, seq, pos, rows, (void*)k.p, (void*)v.p, k.ld, v.ld);
}

void kv_gather(const KvPages& c, const int* seq, const int* pos, int rows, const Rows& k, const Rows& v,
               hipStream_t s) {
    if (rows <= 0) return;
    by_type(k.type, [&](auto yt) {
        if (c.type == T_MXFP4) launch_gather<T_MXFP4, yt()>(c, seq, pos, rows, k, v, s);
        else if (c.type == T_F16) launch_gather<T_F16, yt()>(c, seq, pos, rows, k, v, s);
        else launch_gather<T_BF16, yt()>(c, seq, pos, rows, k, v, s);
    });
}

}  // namespace qasr
