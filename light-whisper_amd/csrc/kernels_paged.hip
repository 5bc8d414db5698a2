// Rotary positions, their table, and moving rows into and out of paged K/V caches (include/qasr.h, "paged K/V cache").
#include "paged_dev.h"

namespace qasr {

// ------------------------------------------------------------------------------------------------ table
// A thread takes one frequency and `run` positions: the angle's sine and cosine once, in 64 bits, and from there each next
// position by one rotation (4 multiply-adds in 64 bits; after 32 of them off by 2^-48 at most, the result is rounded to
// 24 bits).  Bound by the stores: neighbouring lanes hold neighbouring frequencies.
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

constexpr int kRopeMaxHd = 1024;

template <int XT, int YT>
__global__ __launch_bounds__(64) void k_rope_any(const void* x, int64_t ldx, const int* __restrict__ pos, int heads,
                                                 int hd, RopeArgs r, void* y, int64_t ldy) {
    __shared__ float buf[kRopeMaxHd];
    const int row = blockIdx.x / heads, head = blockIdx.x % heads, lane = threadIdx.x;
    const int p = r.cs ? pos[row] : 0;
    if (r.cs && (unsigned)p >= (unsigned)r.n_pos) return;
    head_to_lds<XT, float>(x, row * ldx + (int64_t)head * hd, hd, r, p, lane, buf);
    auto* o = (typename Elem<YT>::type*)y + row * ldy + (int64_t)head * hd;
    for (int d = lane; d < hd; d += 64) o[d] = (typename Elem<YT>::type)buf[d];
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
            k_rope_any<xt(), yt()><<<(unsigned)rows * heads, 64, 0, s>>>(x.p, x.ld, pos, heads, hd, r, (void*)y.p, y.ld);
        });
    });
}

// ------------------------------------------------------------------------------------------------ append / gather
// one (row, KV head) by one wave
template <int XT, int CT>
__global__ __launch_bounds__(64) void k_kv_append(KvPages c, const void* k, const void* v, int64_t ldk, int64_t ldv,
                                                  const int* __restrict__ seq, const int* __restrict__ pos, RopeArgs r) {
    // 4-bit pages: K in 64 bits up to the rounding to f32, so that a value next to a border between two codes gets its own
    typedef typename std::conditional<CT == T_MXFP4, double, float>::type A;
    __shared__ A buf[256];
    const int row = blockIdx.x / c.nkv, head = blockIdx.x % c.nkv, lane = threadIdx.x;
    const int p = pos[row];
    if (r.cs && (unsigned)p >= (unsigned)r.n_pos) return;
    const int64_t at = page_block(c, seq[row], p, head);
    if (at < 0) return;
    const int t = p & ((1 << c.page_shift) - 1);
    const RopeArgs none{};
    for (int kv = 0; kv < 2; kv++) {
        uint8_t* blk = (kv ? c.v : c.k) + at;
        head_to_lds<XT, A>(kv ? v : k, row * (kv ? ldv : ldk) + (int64_t)head * c.hd, c.hd, kv ? none : r, p, lane, buf);
        if constexpr (CT == T_MXFP4) {
            const uint32_t codes = (c.hd / 2) << c.page_shift;
            if (4 * lane < c.hd) {   // four dims of one block of 32
                uint32_t am = 0;
                for (int i = 0; i < 32; i++)
                    am = max(am, __float_as_uint((float)buf[(4 * lane) / 32 * 32 + i]) & 0x7fffffffu);
                const int sc = fp4_scale(__uint_as_float(am));
                uint32_t w = 0;
                for (int i = 0; i < 4; i++) w |= fp4_code((float)buf[4 * lane + i], sc) << (4 * i);
                *(uint16_t*)(blk + (kv ? fp4_v_code : fp4_k_code)(c.hd, t, 4 * lane)) = (uint16_t)w;
                if (lane % 8 == 0) blk[codes + (kv ? fp4_v_scale : fp4_k_scale)(c.hd, t, 4 * lane)] = (uint8_t)sc;
            }
        } else {
            typedef typename Elem<CT>::type E;
            for (int d = lane; d < c.hd; d += 64) ((E*)blk)[t * c.hd + d] = (E)(float)buf[d];
        }
        lds_sync_wave();
    }
}

void kv_append(const KvPages& c, const Rows& k, const Rows& v, const int* seq, const int* pos, int rows,
               const RopeArgs& r, hipStream_t s) {
    if (rows <= 0) return;
    const unsigned grid = (unsigned)rows * c.nkv;
    by_type(k.type, [&](auto xt) {
        if (c.type == T_MXFP4)
            k_kv_append<xt(), T_MXFP4><<<grid, 64, 0, s>>>(c, k.p, v.p, k.ld, v.ld, seq, pos, r);
        else if (c.type == T_F16)
            k_kv_append<xt(), T_F16><<<grid, 64, 0, s>>>(c, k.p, v.p, k.ld, v.ld, seq, pos, r);
        else
            k_kv_append<xt(), T_BF16><<<grid, 64, 0, s>>>(c, k.p, v.p, k.ld, v.ld, seq, pos, r);
    });
}

// the value at (token, dim) of a block
template <int CT>
__device__ __forceinline__ float block_value(const KvPages& c, const uint8_t* blk, bool is_v, int t, int d) {
    if constexpr (CT == T_MXFP4) {
        const uint32_t codes = (c.hd / 2) << c.page_shift;
        const uint32_t b = blk[(is_v ? fp4_v_code : fp4_k_code)(c.hd, t, d)];
        return fp4_value(d & 1 ? b >> 4 : b & 15, blk[codes + (is_v ? fp4_v_scale : fp4_k_scale)(c.hd, t, d)]);
    } else {
        return (float)((const typename Elem<CT>::type*)blk)[t * c.hd + d];
    }
}

template <int CT, int YT>
__global__ __launch_bounds__(64) void k_kv_gather(KvPages c, const int* __restrict__ seq, const int* __restrict__ pos,
                                                  void* k, void* v, int64_t ldk, int64_t ldv) {
    const int row = blockIdx.x / c.nkv, head = blockIdx.x % c.nkv;
    const int p = pos[row];
    const int64_t at = page_block(c, seq[row], p, head);
    if (at < 0) return;
    typedef typename Elem<YT>::type Y;
    const int t = p & ((1 << c.page_shift) - 1);
    for (int d = threadIdx.x; d < c.hd; d += 64) {
        if (k) ((Y*)k)[row * ldk + head * c.hd + d] = (Y)block_value<CT>(c, c.k + at, false, t, d);
        if (v) ((Y*)v)[row * ldv + head * c.hd + d] = (Y)block_value<CT>(c, c.v + at, true, t, d);
    }
}

void kv_gather(const KvPages& c, const int* seq, const int* pos, int rows, const Rows& k, const Rows& v,
               hipStream_t s) {
    if (rows <= 0) return;
    const unsigned grid = (unsigned)rows * c.nkv;
    by_type(k.type, [&](auto yt) {
        if (c.type == T_MXFP4)
            k_kv_gather<T_MXFP4, yt()><<<grid, 64, 0, s>>>(c, seq, pos, (void*)k.p, (void*)v.p, k.ld, v.ld);
        else if (c.type == T_F16)
            k_kv_gather<T_F16, yt()><<<grid, 64, 0, s>>>(c, seq, pos, (void*)k.p, (void*)v.p, k.ld, v.ld);
        else
            k_kv_gather<T_BF16, yt()><<<grid, 64, 0, s>>>(c, seq, pos, (void*)k.p, (void*)v.p, k.ld, v.ld);
    });
}

}  // namespace qasr
