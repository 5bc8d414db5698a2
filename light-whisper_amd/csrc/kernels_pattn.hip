// Attention over a paged K/V cache (include/qasr.h, qasr_op_paged_attention), gfx950.
//
// Query rows of one sequence and KV head are numbered r = token · G + g (G query heads share a KV head), so that every K/V
// byte that is loaded serves all G heads, and are the columns of the matrix instructions:
//   Sᵀ = K·Qᵀ   (keys × rows; a lane holds scores of ONE row, so the softmax needs no cross-lane work but a vote)
//   Oᵀ = Vᵀ·Pᵀ  (dims × rows; a lane's weights are the second operand as they stand, V is brought to match)
// One pass over the keys with a running maximum that moves only where some row's rises by more than 2^kSlack: weights are
// exp2(s − m + lift), sums and Oᵀ in f32.  Roundings: the weights to q's type for the product with V (half a step each; f16
// reaches 2^-26 of the largest before its steps stop shrinking), and their sum is that of the rounded ones, so that an output
// lies between the values it is a mean of; the output to its type.  e2m1 · 2^E is exact in either type.
//
// Few rows (k_paged_attn): bound by memory.  16 / 8 heads of 128, f16: one sequence of 32,768 keys 33 us (134 MB, 4.1 TB/s),
// 64 of 17 .. 8,200 93 us (396 MB, 4.2 TB/s); over 4-bit pages 32 of 501 .. 32,768 77 us (322 MB, 4.2 TB/s; a copy of
// 2 GiB runs at 4.8).  A token of one sequence of 403 keys: 9 us, all of it round trips.
// o may be q: an item's rows of q are read by its own workgroups alone, into registers, and its o is written when all of
// them have done with them (no __restrict__ on either: the compiler must not load q again behind a store).
// Many rows (k_paged_prompt): the matrix unit is busy 38 % of the time and the vector unit 38 %, 10 % of it both at once (two
// prompts of 4,097 and 3,512 rows on 6,891 and 8,192 keys, 431 us; profiles/paged_prompt_counters.txt).  8,192 × 8,192: 620 us,
// 886 TFLOP/s, causal 836; over 4-bit pages 919 and 839; causal at head_dim 64 680, 256 795 (a large f16 product of the
// library: 1,180).
#include "lds_dma.h"
#include "paged_dev.h"
#include "wt.h"

namespace qasr {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kPieces = 32;      // parts of one item at most
constexpr int kTileKeys = 128;   // keys of one workgroup step: 32 for each of its 4 waves
constexpr int kSplitWgs = 1024;  // workgroups at most (what the scratch is sized for)
// workgroups that a CU holds by their registers
constexpr int wgs_per_cu(int hd, int ct) { return ct == T_MXFP4 ? (hd == 256 ? 2 : 3) : hd == 256 ? 1 : 2; }
// weights are exp2(s − m + lift), m at most kSlack below the running maximum.  f16 and 4-bit pages: lift = kUp, weights of at
// most 2^15 in f16, whose normal range reaches 26 bits further down, and V of at most 2^16 leaves the sums far below f32's
// largest.  bf16 pages hold V up to that: there a row's weights, one for each of its sequence's keys, sum to at most 1, so that
// no partial sum of the product with V passes the largest |V| (at the other end, over 32,768 keys, V below 2^-108 meets f32's
// smallest normal numbers)
constexpr float kSlack = 3.f, kUp = 12.f;
template <int CT>
__device__ __forceinline__ float lift(int keys) {
    return CT == T_BF16 ? -kSlack - (float)(32 - __clz(max(keys, 1) - 1)) : kUp;   // (bits of keys − 1: ⌈log2 keys⌉)
}
constexpr float kNone = -3.40282347e38f;   // running maximum before the first key: no score is less
// exp2(s · c + (lift − m)) is one multiply-add and one rounding of m, which is more than the slack in a weight's range once m
// has 24 bits before the point: where a row's |m| is past kBig (a rounding of 2^-12), s · c − m is taken first, from the product
// as m was, so that the largest gives 0 and none a larger weight than the lift and the slack allow
constexpr float kBig = 4096.f;
__device__ __forceinline__ bool is_big(float m) { return fabsf(m) > kBig && m != kNone; }

template <int QT>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (QT == T_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                       0);
}
template <int QT>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (QT == T_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                       0);
}
// two f32 → a packed pair of QT, rounded to nearest even
template <int QT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (QT == T_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
// sum + both numbers of a packed pair, in f32
template <int QT>
__device__ __forceinline__ float add2(uint32_t pair, float sum) {
    if constexpr (QT == T_F16) {
        const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), one, sum, false);
    } else {
        const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), one, sum, false);
    }
}
// byte SEL of w: two e2m1 codes · the power of two `s` → a packed pair of QT, exact
template <int QT>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float s, int sel) {
    if constexpr (QT == T_F16) {
        switch (sel) {
            case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0));
            case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1));
            case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2));
            default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3));
        }
    } else {
        switch (sel) {
            case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
            case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
            case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
            default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
        }
    }
}
__device__ __forceinline__ uint32_t lo16(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t hi16(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// inclusive prefix sum and prefix maximum (of values >= 0) over the wave, on DPP: rows of 16 by shifts, then each row's last
// lane to the rows behind it
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_0(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
    v += dpp_or_0<0x111, 0xf>(v);
    v += dpp_or_0<0x112, 0xf>(v);
    v += dpp_or_0<0x114, 0xf>(v);
    v += dpp_or_0<0x118, 0xf>(v);
    v += dpp_or_0<0x142, 0xa>(v);
    v += dpp_or_0<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ int wave_scan_max(int v) {
    v = max(v, dpp_or_0<0x111, 0xf>(v));
    v = max(v, dpp_or_0<0x112, 0xf>(v));
    v = max(v, dpp_or_0<0x114, 0xf>(v));
    v = max(v, dpp_or_0<0x118, 0xf>(v));
    v = max(v, dpp_or_0<0x142, 0xa>(v));
    return max(v, dpp_or_0<0x143, 0xc>(v));
}

// what one sequence asks for (per lane while scanning, uniform afterwards)
struct SeqWork {
    int row0, nq, len, lo;   // first row of q, rows, keys, first key that any row sees
};
// that of sequence s0 + lane; `edge`: where the rows of sequence s0 begin, becomes where those of s0 + 64 do.  (Whatever
// q_start holds, the sequences' rows lie side by side in [0, rows): the lists below cannot grow past what the host reckons)
__device__ __forceinline__ SeqWork seq_work(const KvPages& c, const AttnArgs& a, const int* q_start, const int* kv_len,
                                            int rows, int s0, int lane, int& edge) {
    SeqWork w;
    const int s = s0 + lane;
    const bool is = s < c.n_seq;
    const int end = max(wave_scan_max(is ? min(max(q_start[s + 1], 0), rows) : 0), edge);
    w.row0 = __builtin_amdgcn_update_dpp(edge, end, 0x138, 0xf, 0xf, false);   // the lane before's
    w.nq = end - w.row0;
    edge = __builtin_amdgcn_readlane(end, 63);
    w.len = is ? (int)min((int64_t)max(kv_len[s], 0), (int64_t)c.max_pages << c.page_shift) : 0;
    // the first row's window starts furthest left; with len < nq its position is negative
    w.lo = a.window > 0 ? max(w.len - w.nq - a.window + 1, 0) : 0;
    return w;
}
__device__ __forceinline__ int first_row(const int* q_start, int rows) { return uniform(min(max(q_start[0], 0), rows)); }

// the registers of one wave's 32 keys
template <int HD, int CT>
struct Slice {
    static constexpr int ND = HD / 16;
    u32x4 k[2][HD / 32], v[8 * ND / 8];   // v[j] (ND = 8); ND = 16: v[2 j], v[2 j + 1]; ND = 4: two keys each
};
template <int HD>
struct Slice<HD, T_MXFP4> {
    uint32_t k[2][HD / 32], v[2][HD / 32];
    uint32_t ks[2][HD == 256 ? 2 : 1], vs[2];
};

// One block of a page as a buffer: 32-bit lane offsets, and nothing past the block is ever read
__device__ __forceinline__ __amdgpu_buffer_rsrc_t block_rsrc(const uint8_t* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), (short)0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 load4(__amdgpu_buffer_rsrc_t r, uint32_t lane_off, uint32_t off) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, lane_off, off, 0));
}
__device__ __forceinline__ u32x2 load2(__amdgpu_buffer_rsrc_t r, uint32_t lane_off, uint32_t off) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, lane_off, off, 0));
}
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&d)[N], __amdgpu_buffer_rsrc_t r, uint32_t lane_off, uint32_t off) {
    if constexpr (N == 2) {
        const u32x2 t = load2(r, lane_off, off);
        d[0] = t[0], d[1] = t[1];
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const u32x4 t = load4(r, lane_off + 16 * i, off);
#pragma unroll
            for (int j = 0; j < 4; j++) d[4 * i + j] = t[j];
        }
    }
}

// tokens t0 .. t0 + 15 of a page's block into sub-tile u
template <int HD, int CT>
__device__ __forceinline__ void load_k(Slice<HD, CT>& s, int u, __amdgpu_buffer_rsrc_t kb, int t0, uint32_t codes, int n,
                                       int kg) {
    if constexpr (CT == T_MXFP4) {
        load_words(s.k[u], kb, n * (HD / 2) + kg * (HD / 8), t0 * (HD / 2));
        const uint32_t ks = codes + t0 * (HD / 32);
        if constexpr (HD == 64) s.ks[u][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(kb, n * 2, ks, 0);
        else if constexpr (HD == 128) s.ks[u][0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(kb, n * 4, ks, 0);
        else load_words(s.ks[u], kb, n * 8, ks);
    } else {
#pragma unroll
        for (int kk = 0; kk < HD / 32; kk++) s.k[u][kk] = load4(kb, n * (HD * 2) + kg * 16 + kk * 64, t0 * (HD * 2));
    }
}
template <int HD, int CT>
__device__ __forceinline__ void load_v(Slice<HD, CT>& s, int u, __amdgpu_buffer_rsrc_t vb, int t0, uint32_t codes, int n,
                                       int kg) {
    constexpr int ND = HD / 16;
    if constexpr (CT == T_MXFP4) {
        load_words(s.v[u], vb, (16 * kg + n) * (2 * ND), t0 * (HD / 2));
        s.vs[u] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(vb, (n * ND / 32) * 16 + 4 * kg, codes + t0 * (HD / 32), 0);
    } else {
        const uint32_t vr = 4 * kg * (HD * 2) + n * (ND * 2), off = t0 * (HD * 2);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (ND == 8) s.v[4 * u + j] = load4(vb, vr + j * (HD * 2), off);
            else if constexpr (ND == 16) {
                s.v[8 * u + 2 * j] = load4(vb, vr + j * (HD * 2), off);
                s.v[8 * u + 2 * j + 1] = load4(vb, vr + j * (HD * 2) + 16, off);
            } else {
                const u32x2 t = load2(vb, vr + j * (HD * 2), off);
                s.v[2 * u + j / 2][2 * (j & 1)] = t[0];
                s.v[2 * u + j / 2][2 * (j & 1) + 1] = t[1];
            }
        }
    }
}

// Vᵀ operands of the dims ND·m + 2 b (t0) and + 2 b + 1 (t1): register p holds the lane's keys 2 p, 2 p + 1
// (ANEW: not to be computed ahead of a loop that asks for them each time)
template <int HD, int CT, int QT, bool ANEW = false>
__device__ __forceinline__ void pair_v(const Slice<HD, CT>& s, int b, u32x4& t0, u32x4& t1) {
    auto at = [](uint32_t v) {
        if (ANEW) asm volatile("" : "+v"(v));
        return v;
    };
    constexpr int ND = HD / 16;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        uint32_t x, y;
        if constexpr (CT == T_MXFP4) {
            const int u = p >> 1, j = (2 * p) & 3;   // sub-tile, first key of the pair in it
            const float s0 = __uint_as_float(((s.vs[u] >> (8 * j)) & 255) << 23);
            const float s1 = __uint_as_float(((s.vs[u] >> (8 * j + 8)) & 255) << 23);
            const int i0 = j * (ND / 2) + b, i1 = (j + 1) * (ND / 2) + b;
            x = fp4_pair<QT>(at(s.v[u][i0 / 4]), s0, i0 % 4);
            y = fp4_pair<QT>(at(s.v[u][i1 / 4]), s1, i1 % 4);
        } else if constexpr (ND == 8) {
            x = at(s.v[2 * p][b]), y = at(s.v[2 * p + 1][b]);
        } else if constexpr (ND == 16) {
            x = at(s.v[4 * p + b / 4][b % 4]), y = at(s.v[4 * p + 2 + b / 4][b % 4]);
        } else {
            x = at(s.v[p][b]), y = at(s.v[p][2 + b]);
        }
        t0[p] = lo16(x, y);
        t1[p] = hi16(x, y);
    }
}

// zero V of the lane's keys that are not in `keep` (bit j = key j)
template <int HD, int CT>
__device__ __forceinline__ void zero_keys(Slice<HD, CT>& s, uint32_t keep) {
    constexpr int ND = HD / 16;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (keep >> j & 1) continue;
        if constexpr (CT == T_MXFP4) {
            const int u = j >> 2, i = j & 3;
            s.vs[u] = (s.vs[u] & ~(255u << (8 * i))) | 127u << (8 * i);
            if constexpr (ND == 4) s.v[u][i / 2] &= i & 1 ? 0xffffu : 0xffff0000u;
            else if constexpr (ND == 8) s.v[u][i] = 0;
            else s.v[u][2 * i] = 0, s.v[u][2 * i + 1] = 0;
        } else if constexpr (ND == 8) {
            s.v[j] = u32x4{0, 0, 0, 0};
        } else if constexpr (ND == 16) {
            s.v[2 * j] = u32x4{0, 0, 0, 0}, s.v[2 * j + 1] = u32x4{0, 0, 0, 0};
        } else {
            s.v[j / 2][2 * (j & 1)] = 0, s.v[j / 2][2 * (j & 1) + 1] = 0;
        }
    }
}
// not 0 where one of four scale bytes is 255: it alone has its two highest bits set (the others are 104 .. 140)
__device__ __forceinline__ uint32_t nan_scale(uint32_t b) { return b & (b << 1) & 0x80808080u; }
// a value that the compiler takes for new here: what follows from it is not computed ahead and held in registers
__device__ __forceinline__ int anew(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
// some V of the lane's keys is an infinity or NaN
template <int HD, int CT, int QT>
__device__ __forceinline__ bool v_not_finite(const Slice<HD, CT>& s) {
    if constexpr (CT == T_MXFP4) {
        return (nan_scale(s.vs[0]) | nan_scale(s.vs[1])) != 0;
    } else {
        constexpr uint32_t e = QT == T_F16 ? 0x7c00u : 0x7f80u;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < HD / 16; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) bad |= (s.v[j][i] & e) == e || ((s.v[j][i] >> 16) & e) == e;
        return bad;
    }
}

// four values of o
template <int QT>
__device__ __forceinline__ void store_out(void* o, int o_type, int64_t at, f32x4 v, int o_vec) {
    if (o_type == T_F32) {
        float* op = (float*)o + at;
        if (o_vec) *(f32x4*)op = v;
        else
#pragma unroll
            for (int i = 0; i < 4; i++) op[i] = v[i];
    } else {
        uint16_t* op = (uint16_t*)o + at;
        const u32x2 d = {pack2<QT>(v[0], v[1]), pack2<QT>(v[2], v[3])};
        if (o_vec) *(u32x2*)op = d;
        else
#pragma unroll
            for (int i = 0; i < 4; i++) op[i] = (uint16_t)(d[i / 2] >> (16 * (i & 1)));
    }
}
// ------------------------------------------------------------------------------------------------ few rows
// One launch over every sequence: the work is the list of (sequence, 16-row tile, KV head) items, each ⌈keys / 128⌉ tiles
// long; workgroup w takes tiles [w · per, (w + 1) · per) of the whole list, so lengths that differ a thousandfold load the
// workgroups alike.  No K/V byte passes LDS: K rows are loaded in the first operand's layout (v_mfma_f32_16x16x32: 16 keys ×
// 16 rows), a lane loads hd/16 dims of its 8 keys of V and pairs them key by key in registers (v_perm), which makes MFMA row
// m of tile t dim (hd/16) m + t; contraction slot (lane >> 4, j) stands for key 16 (j >> 2) + 4 (lane >> 4) + (j & 3), the
// order in which the lane has its weights.  A wave's next K is loaded as soon as its scores are there, V behind its product
// (two sets of registers instead: one workgroup less a CU, and spills).
// A workgroup's part of an item is a segment; a segment that is not its whole item leaves its
// (m, l, Oᵀ) in the scratch, and the last of the item's workgroups to arrive adds them up in their order (the result does
// not depend on who is last).  Slot 0 of a workgroup: the item began in an earlier one; slot 1: it goes on in a later one.
template <int HD, int CT, int QT>
__global__ __launch_bounds__(256, wgs_per_cu(HD, CT)) void k_paged_attn(KvPages c, AttnArgs a, const void* q, int64_t ldq,
                                                       const int* __restrict__ q_start, const int* __restrict__ kv_len,
                                                       int rows, void* o, int64_t ldo, float* part,
                                                       unsigned* cnt, int q_vec, int o_vec) {
    constexpr int ND = HD / 16, KK = HD / 32, LANES = 64;
    constexpr int kSlot = 16 * HD + 32;   // floats of a slot: Oᵀ as [wave][lane >> 4][row][ND], then m and l of 16 rows
    __shared__ float s_acc[4][ND * 4][LANES];
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ int s_last;
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
    const int G = a.nh / c.nkv;
    const uint32_t codes = (HD / 2) << c.page_shift;
    // a negative scale goes into q's signs; a zero one is the smallest number, so that −∞ of a masked key stays −∞
    const float sc = fmaxf(fabsf(a.scale) * 1.44269504088896340736f, 1.17549435e-38f);
    const uint32_t q_sign = a.scale < 0.f ? 0x80008000u : 0u;

    // ---- the list: tiles of every sequence, and where this workgroup's begin
    auto tiles_of = [&](const SeqWork& x) {   // key tiles of one item; an item without keys has one, which writes zeros
        return max(1, (x.len + kTileKeys - 1) / kTileKeys - x.lo / kTileKeys);
    };
    auto items_of = [&](const SeqWork& x) { return ((x.nq * G + 15) >> 4) * c.nkv; };
    int longest = 0;                        // item, in tiles
    int chunk = 0, before = 0, total = 0;   // first sequence held in the lanes, tiles before it, all tiles
    SeqWork my{};
    int scan = 0;   // tiles up to and with this lane's sequence, from `chunk` on
    const int row_first = first_row(q_start, rows);
    int edge = row_first;
    auto hold = [&](int s0) {
        chunk = s0;
        if (s0 == 0) edge = row_first;
        my = seq_work(c, a, q_start, kv_len, rows, s0, lane, edge);
        scan = wave_scan(my.nq > 0 ? items_of(my) * tiles_of(my) : 0);
    };
    for (int s0 = 0; s0 < c.n_seq; s0 += LANES) {
        hold(s0);
        total += __builtin_amdgcn_readlane(scan, 63);
        longest = max(longest, __builtin_amdgcn_readlane(wave_scan_max(my.nq > 0 ? tiles_of(my) : 0), 63));
    }
    // a long item in at most kPieces parts: their arrivals are counted one after the other, 40 to 80 ns each
    const int per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, (longest + kPieces - 1) / kPieces);
    int t = blockIdx.x * per;
    const int t_end = min(total, t + per);
    if (t >= t_end) return;
    if (c.n_seq > LANES) {
        for (int s0 = 0;; s0 += LANES) {
            hold(s0);
            const int in = __builtin_amdgcn_readlane(scan, 63);
            if (t < before + in) break;
            before += in;
        }
    }

    while (t < t_end) {
        // what follows from the lane's place is computed anew for each segment: held over the loop it takes the registers
        // of a third of the waves
        const int ln = anew(lane);
        const int n = ln & 15, kg = ln >> 4;
        // ---- the segment that tile t begins
        while (t >= before + __builtin_amdgcn_readlane(scan, 63)) {
            before += __builtin_amdgcn_readlane(scan, 63);
            hold(chunk + LANES);
        }
        const int sl = __popcll(__ballot(before + scan <= t));   // the lane that holds the sequence
        const int seq = chunk + sl;
        const SeqWork x{__builtin_amdgcn_readlane(my.row0, sl), __builtin_amdgcn_readlane(my.nq, sl),
                        __builtin_amdgcn_readlane(my.len, sl), __builtin_amdgcn_readlane(my.lo, sl)};
        const int first = before + (sl ? __builtin_amdgcn_readlane(scan, sl - 1) : 0);   // the sequence's first tile
        const int kt = tiles_of(x), item = (t - first) / kt;
        const int item_t = first + item * kt;                    // the item's first tile
        const int seg = min(item_t + kt, t_end) - t;             // tiles of this segment
        const int key0 = (x.lo / kTileKeys + (t - item_t)) * kTileKeys;
        const int rt = item / c.nkv, kvh = item % c.nkv;
        const int nrow = min(16, x.nq * G - rt * 16);

        // ---- this lane's row: its keys [lo, hi) and its q
        // (positions: lengths are at most 2^30, row counts below 2^31, so differences fit; windows are cut to 2^30)
        auto row_of = [&](int nn, int& tok, int& head) {
            const int r = rt * 16 + min(nn, nrow - 1);
            tok = r / G;
            head = kvh * G + r % G;
        };
        int tok, head;
        row_of(n, tok, head);
        const int p0 = x.len - x.nq, at = p0 + tok;
        const int hi = a.causal ? min(x.len, at + 1) : x.len;
        const int lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
        // keys [all_lo, all_hi) are seen by every row of the tile
        const int all_hi = a.causal ? max(0, min(x.len, p0 + rt * 16 / G + 1)) : x.len;
        const int all_lo = a.window > 0 ? max(0, p0 + (rt * 16 + nrow - 1) / G - a.window + 1) : 0;
        u32x4 qf[KK];
        {
            const uint16_t* qp = (const uint16_t*)q + (x.row0 + tok) * ldq + (int64_t)head * HD + 8 * kg;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                if (q_vec) qf[kk] = *(const u32x4*)(qp + 32 * kk);
                else
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        qf[kk][i] = qp[32 * kk + 2 * i] | (uint32_t)qp[32 * kk + 2 * i + 1] << 16;
#pragma unroll
                for (int i = 0; i < 4; i++) qf[kk][i] ^= q_sign;
            }
        }

        // ---- the page ids of this wave's next 64 slices, one per lane (two where pages have 16 tokens)
        const int* tab = c.table + (int64_t)seq * c.max_pages;
        int id0 = 0, id1 = 0;
        auto ids = [&](int i0, int& d0, int& d1) {
            const int64_t key = (int64_t)key0 + (i0 + lane) * (int64_t)kTileKeys + w * 32;
            d0 = key < x.len ? tab[key >> c.page_shift] : -1;
            d1 = c.page_shift > 4 ? d0 : key + 16 < x.len ? tab[(key + 16) >> c.page_shift] : -1;
        };
        ids(0, id0, id1);

        f32x4 acc[ND];
        float m, l;
        bool big = false;   // some row's m is
        auto clear = [&] {
#pragma unroll
            for (int i = 0; i < ND; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            m = kNone;
            l = 0.f;
            big = false;
        };
        clear();

        // where slice i lies: its two sub-tiles' blocks, and which have a page (the others load bytes that no row uses)
        struct At {
            int64_t b0, b1;
            int t0, t1, have;
        };
        auto place = [&](int i) {
            const int key = key0 + i * kTileKeys + w * 32, mask = (1 << c.page_shift) - 1;
            const int d0 = __builtin_amdgcn_readlane(id0, i & 63), d1 = __builtin_amdgcn_readlane(id1, i & 63);
            const bool ok0 = (unsigned)d0 < (unsigned)c.n_pages, ok1 = (unsigned)d1 < (unsigned)c.n_pages;
            return At{((int64_t)(ok0 ? d0 : 0) * c.nkv + kvh) * c.block_bytes,
                      ((int64_t)(ok1 ? d1 : 0) * c.nkv + kvh) * c.block_bytes, key & mask, (key + 16) & mask,
                      (ok0 ? 1 : 0) | (ok1 ? 2 : 0)};
        };

        // ---- the segment's slices: the next slice's K is loaded into the registers of this one's as soon as its scores
        // are there, and V's after the product
        const int mine = max(0, min(seg, (x.len - key0 - 32 * w + kTileKeys - 1) / kTileKeys));   // with keys in them
        bool careful = false;
        for (bool again = mine > 0; again;) {
            again = false;
            clear();
            Slice<HD, CT> s;
            At pl = place(0);
            load_k<HD, CT>(s, 0, block_rsrc(c.k + pl.b0, c.block_bytes), pl.t0, codes, n, kg);
            load_k<HD, CT>(s, 1, block_rsrc(c.k + pl.b1, c.block_bytes), pl.t1, codes, n, kg);
            load_v<HD, CT>(s, 0, block_rsrc(c.v + pl.b0, c.block_bytes), pl.t0, codes, n, kg);
            load_v<HD, CT>(s, 1, block_rsrc(c.v + pl.b1, c.block_bytes), pl.t1, codes, n, kg);
            for (int i = 0; i < mine; i++) {
                const int key = key0 + i * kTileKeys + w * 32, have = pl.have;
                const bool whole = have == 3 && key >= all_lo && key + 32 <= all_hi;
                float p[8];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kk = 0; kk < KK; kk++) {
                        if constexpr (CT == T_MXFP4) {
                            const float f = __uint_as_float(((s.ks[u][kk / 4] >> (8 * (kk % 4))) & 255) << 23);
                            const uint32_t wd = s.k[u][kk];
                            const u32x4 kf = {fp4_pair<QT>(wd, f, 0), fp4_pair<QT>(wd, f, 1), fp4_pair<QT>(wd, f, 2),
                                              fp4_pair<QT>(wd, f, 3)};
                            d = mfma16<QT>(kf, qf[kk], d);
                        } else {
                            d = mfma16<QT>(s.k[u][kk], qf[kk], d);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) p[4 * u + j] = d[j];
                }
                if constexpr (CT == T_MXFP4) {   // a scale byte of 255: the key (lane n's) is not a number
                    uint32_t nan[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        nan[u] = nan_scale(s.ks[u][0]);
                        if constexpr (HD == 256) nan[u] |= nan_scale(s.ks[u][1]);
                    }
                    if (__any((nan[0] | nan[1]) != 0)) {
                        const int kq = 4 * anew(kg);
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const uint32_t who = (uint32_t)__ballot(nan[u] != 0) >> kq;
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                if (who >> j & 1) p[4 * u + j] = __uint_as_float(0x7fc00000u);
                        }
                    }
                }
                if (i + 1 < mine) {
                    if (((i + 1) & 63) == 0) ids(i + 1, id0, id1);
                    pl = place(i + 1);
                    load_k<HD, CT>(s, 0, block_rsrc(c.k + pl.b0, c.block_bytes), pl.t0, codes, n, kg);
                    load_k<HD, CT>(s, 1, block_rsrc(c.k + pl.b1, c.block_bytes), pl.t1, codes, n, kg);
                }
                uint32_t see = 0xff;   // which of this lane's 8 keys its row sees
                if (!whole) {
                    see = 0;
                    uint32_t real = 0;   // … and which any row may
                    const int k4 = key + 4 * anew(kg);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int kj = k4 + 16 * (j >> 2) + (j & 3);
                        const bool h = have >> (j >> 2) & 1;
                        if (h && kj >= lo && kj < hi) see |= 1u << j;
                        else p[j] = -INFINITY;
                        if (h && kj < x.len) real |= 1u << j;
                    }
                    zero_keys<HD, CT>(s, real);
                }
                if ((!whole || CT == T_MXFP4) && !careful && __any(v_not_finite<HD, CT, QT>(s))) {
                    // 0 · V is no zero where V is no number: from the start again, with the rows one by one
                    careful = again = true;
                    ids(0, id0, id1);
                    break;
                }
                float mx = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
                mx *= sc;
                if (__any(mx > m + kSlack)) {   // some row's maximum rose: move every row to its own
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                    l *= al;
                    big = __any(is_big(m));
#pragma unroll
                    for (int t2 = 0; t2 < ND; t2++) acc[t2] *= al;
                }
                u32x4 pf;
                float c2 = sc, mk = lift<CT>(x.len) - m;
                if (__builtin_expect(big, 0) && is_big(m)) {
#pragma unroll
                    for (int j = 0; j < 8; j++) p[j] = p[j] * sc - m;
                    c2 = 1.f;
                    mk = lift<CT>(x.len);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] = __builtin_amdgcn_exp2f(fmaf(p[j], c2, mk));
#pragma unroll
                for (int j = 0; j < 4; j++) pf[j] = pack2<QT>(p[2 * j], p[2 * j + 1]);
                l += add2<QT>(pf[3], add2<QT>(pf[2], add2<QT>(pf[1], add2<QT>(pf[0], 0.f))));
                if (!careful) {
#pragma unroll
                    for (int b = 0; b < ND / 2; b++) {
                        u32x4 v0, v1;
                        pair_v<HD, CT, QT>(s, b, v0, v1);
                        acc[2 * b] = mfma16<QT>(v0, pf, acc[2 * b]);
                        acc[2 * b + 1] = mfma16<QT>(v1, pf, acc[2 * b + 1]);
                    }
                } else {
                    for (int n0 = 0; n0 < nrow; n0++) {
                        const uint32_t sees = __shfl(see, 16 * kg + n0);
#pragma unroll
                        for (int b = 0; b < ND / 2; b++) {
                            u32x4 v0, v1;
                            pair_v<HD, CT, QT, true>(s, b, v0, v1);
#pragma unroll
                            for (int pr = 0; pr < 4; pr++) {
                                if constexpr (CT == T_MXFP4) {   // a scale byte of 255 stands for NaN
                                    const uint32_t two = s.vs[pr / 2] >> (16 * (pr & 1));
                                    const uint32_t nan = ((two & 255) == 255 ? 0x7fffu : 0u) | ((two >> 8 & 255) == 255 ? 0x7fff0000u : 0u);
                                    v0[pr] |= nan, v1[pr] |= nan;
                                }
                                const uint32_t mask = (sees >> (2 * pr) & 1 ? 0xffffu : 0u) | (sees >> (2 * pr + 1) & 1 ? 0xffff0000u : 0u);
                                v0[pr] &= mask, v1[pr] &= mask;
                            }
                            const f32x4 d0 = mfma16<QT>(v0, pf, acc[2 * b]), d1 = mfma16<QT>(v1, pf, acc[2 * b + 1]);
                            if (n == n0) acc[2 * b] = d0, acc[2 * b + 1] = d1;
                        }
                    }
                }
                if (i + 1 < mine) {
                    load_v<HD, CT>(s, 0, block_rsrc(c.v + pl.b0, c.block_bytes), pl.t0, codes, n, kg);
                    load_v<HD, CT>(s, 1, block_rsrc(c.v + pl.b1, c.block_bytes), pl.t1, codes, n, kg);
                }
            }
        }

        // ---- the four waves' states, then out or into the scratch: wave w takes acc[.][w], dims ND (4 kg + w) ..
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        __syncthreads();   // the previous segment's readers are done
        if (kg == 0) s_m[w][n] = m, s_l[w][n] = l;
        if (n < nrow) {
#pragma unroll
            for (int t2 = 0; t2 < ND; t2++)
#pragma unroll
                for (int i = 0; i < 4; i++) s_acc[w][t2 * 4 + i][ln] = acc[t2][i];
        }
        __syncthreads();
        float M = fmaxf(fmaxf(s_m[0][n], s_m[1][n]), fmaxf(s_m[2][n], s_m[3][n])), Lsum = 0.f, out[ND];
#pragma unroll
        for (int t2 = 0; t2 < ND; t2++) out[t2] = 0.f;
        if (n < nrow) {
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const float f = __builtin_amdgcn_exp2f(s_m[v][n] - M);
                Lsum = fmaf(s_l[v][n], f, Lsum);
#pragma unroll
                for (int t2 = 0; t2 < ND; t2++) out[t2] = fmaf(s_acc[v][t2 * 4 + w][ln], f, out[t2]);
            }
        }
        bool write = true;
        if (seg < kt) {   // uniform: a part of its item
            const int wg0 = item_t / per, wg1 = (item_t + kt - 1) / per;   // the item's first and last workgroup
            const int pieces = wg1 - wg0 + 1;
            float* mine = part + ((int64_t)blockIdx.x * 2 + ((int)blockIdx.x == wg0)) * kSlot;
            if (n < nrow) {
                const uint32_t off = (((w * 4 + kg) * 16 + n) * ND) * 4;
#pragma unroll
                for (int t2 = 0; t2 < ND; t2 += 4)
                    wt_st128(mine, off + 4 * t2,
                             __builtin_bit_cast(wt_v4i, f32x4{out[t2], out[t2 + 1], out[t2 + 2], out[t2 + 3]}));
                if (w == 0 && kg == 0) {
                    wt_stf(mine, (16 * HD + n) * 4, M);
                    wt_stf(mine, (16 * HD + 16 + n) * 4, Lsum);
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // written through before the arrival is counted
            __syncthreads();
            if (threadIdx.x == 0)
                s_last = __hip_atomic_fetch_add(&cnt[wg0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                         (unsigned)pieces - 1;
            __syncthreads();
            write = s_last;
            if (write) {
                if (threadIdx.x == 0) __hip_atomic_store(&cnt[wg0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                // rows that are not there leave lanes free: lane n takes row n % R of the pieces n / R, n / R + 16 / R, …
                const int R = nrow <= 1 ? 1 : nrow <= 2 ? 2 : nrow <= 4 ? 4 : nrow <= 8 ? 8 : 16;
                const int rn = n % R, step = 16 / R;
                M = kNone;
                Lsum = 0.f;
#pragma unroll
                for (int t2 = 0; t2 < ND; t2++) out[t2] = 0.f;
                const uint32_t off = (((w * 4 + kg) * 16 + rn) * ND) * 4;
                if (rn < nrow) {
                    constexpr int U = 4;   // pieces whose loads are in flight together (one past the end is the last one again)
                    for (int p0 = n / R; p0 < pieces; p0 += U * step) {
                        float pm[U], pl[U], po[U][ND];
#pragma unroll
                        for (int u = 0; u < U; u++) {
                            const int pc = min(p0 + u * step, pieces - 1);
                            const uint32_t so = (uint32_t)((wg0 + pc) * 2 + (pc == 0)) * (kSlot * 4);
                            pm[u] = wt_ldf(part, so + (16 * HD + rn) * 4);
                            pl[u] = wt_ldf(part, so + (16 * HD + 16 + rn) * 4);
#pragma unroll
                            for (int t2 = 0; t2 < ND; t2 += 4) {
                                const float4 f4 = wt_ldf4(part, so + off + 4 * t2);
                                po[u][t2] = f4.x, po[u][t2 + 1] = f4.y, po[u][t2 + 2] = f4.z, po[u][t2 + 3] = f4.w;
                            }
                        }
#pragma unroll
                        for (int u = 0; u < U; u++) {
                            if (p0 + u * step >= pieces) continue;
                            const float mn = fmaxf(M, pm[u]), f0 = __builtin_amdgcn_exp2f(M - mn), f1 = __builtin_amdgcn_exp2f(pm[u] - mn);
                            M = mn;
                            Lsum = Lsum * f0 + pl[u] * f1;
#pragma unroll
                            for (int t2 = 0; t2 < ND; t2++) out[t2] = out[t2] * f0 + po[u][t2] * f1;
                        }
                    }
                }
                for (int s = R; s < 16; s <<= 1) {
                    const float om = __shfl_xor(M, s), ol = __shfl_xor(Lsum, s);
                    const float mn = fmaxf(M, om), f0 = __builtin_amdgcn_exp2f(M - mn), f1 = __builtin_amdgcn_exp2f(om - mn);
                    Lsum = Lsum * f0 + ol * f1;
                    M = mn;
#pragma unroll
                    for (int t2 = 0; t2 < ND; t2++) {
                        const float oo = __shfl_xor(out[t2], s);
                        out[t2] = out[t2] * f0 + oo * f1;
                    }
                }
            }
        }
        if (write && n < nrow) {
            const float inv = Lsum == 0.f ? 0.f : 1.f / Lsum;
#pragma unroll
            for (int t2 = 0; t2 < ND; t2++) out[t2] *= inv;
            int tok, head;
            row_of(anew(n), tok, head);
            const int64_t at_o = (x.row0 + tok) * ldo + (int64_t)head * HD + ND * (4 * kg + w);
#pragma unroll
            for (int t2 = 0; t2 < ND; t2 += 4)
                store_out<QT>(o, a.o_type, at_o + t2, f32x4{out[t2], out[t2 + 1], out[t2 + 2], out[t2 + 3]}, o_vec);
        }
        t += seg;
    }
}


// ------------------------------------------------------------------------------------------------ many rows
// A workgroup takes 128 rows of one sequence and KV head, 32 for each of its 4 waves (v_mfma_f32_32x32x16, the same two
// products: a lane holds 32 of 64 scores of one row), and walks the keys in tiles of 64 that all waves share through two
// LDS buffers: tile t + 1 is on its way (LDS-DMA; 4-bit pages by registers, widened as they are stored) while t is used,
// one barrier a tile.  Vᵀ comes out of LDS by transposing reads.  Rows of 16-byte chunks, chunk c of row r at c ^ swz(r):
//   K  swz = r mod chunks: 8 neighbouring rows' chunks fall in 8 places
//   V  swz = 4 (r mod 4) (head_dim 64: 4 (r / 2 mod 2)): the 4 rows × 64 bytes of a transposing read's half wave fall in
//      the 16 places of 256 bytes
// Work: items (sequence, 128 rows, KV head), a sequence's longest first, KV heads side by side (neighbouring workgroups go to
// different XCDs: with 8 heads an XCD's L2 serves one).  Where the items are too few for the chip, `splits` workgroups
// share one item's keys and the last to arrive joins their parts.
// (Tried and slower: 8 waves in two groups a phase apart, one multiplying while the other takes its softmax; the next tile's
// scores interleaved with the exponentials.)
constexpr int kRowBlock = 128, kPromptKeys = 64;
constexpr int kPromptSlots = 1024;   // parts of all items together where items are split
constexpr int kPromptParts = 32;     // … and of one item

// Parts of an item of so many tiles.  About what takes least: a part walks tiles / parts of 2.6 us and the join reads `parts`
// of about 1 us, one by one, and a few us to be there at all (2 tiles: 14.8 us alone, 16.0 in two parts); and no more than fill
// the chip once (`fill` parts of every item are kPromptSlots), or twice with long parts, which end together
__host__ __device__ inline int prompt_parts(int tiles, int fill, int hd, int most) {
    const int n = max(fill / (hd == 256 ? 3 : 2), min(fill, tiles / 32));
    return tiles < 6 ? 1 : max(1, min(min((int)sqrtf(2.5f * tiles), n), most));
}

template <int HD>
__device__ __forceinline__ int k_swz(int row) { return row & (HD / 8 - 1); }
template <int HD>
__device__ __forceinline__ int v_swz(int row) { return HD == 64 ? (row & 2) << 1 : (row & 3) << 2; }

template <int HD, int CT, int QT>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_paged_prompt(
    KvPages c, AttnArgs a, const void* q, int64_t ldq, const int* __restrict__ q_start,
    const int* __restrict__ kv_len, int rows, void* o, int64_t ldo, float* part, unsigned* cnt, int splits,
    int fill, int q_vec, int o_vec) {
    constexpr int KK = HD / 16, DT = HD / 32, CPR = HD / 8, ROW = HD * 2;
    constexpr bool kAhead = CT == T_MXFP4 || HD == 256;
    constexpr int kSlot = kRowBlock * (HD + 2);   // floats: Oᵀ as [wave][dim tile · 4 + i / 4][lane][4], then m, l per row
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ int s_ok[2][4];
    __shared__ uint64_t s_odd[4];
    __shared__ int s_last;
    constexpr int TILE = kPromptKeys * ROW;
    uint8_t* const ldsK = lds;             // [2][TILE]
    uint8_t* const ldsV = lds + 2 * TILE;  // [2][TILE]
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
    const int G = a.nh / c.nkv;
    const uint32_t codes = (HD / 2) << c.page_shift;
    const float sc = fmaxf(fabsf(a.scale) * 1.44269504088896340736f, 1.17549435e-38f);   // as in k_paged_attn
    const uint32_t q_sign = a.scale < 0.f ? 0x80008000u : 0u;

    // ---- this workgroup's item
    const int split = blockIdx.x % splits, item = blockIdx.x / splits;
    const int kvh = item % c.nkv;
    int blk = item / c.nkv;   // row block, counted over the sequences
    SeqWork x{};
    int seq = -1, edge = first_row(q_start, rows);
    for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
        const SeqWork my = seq_work(c, a, q_start, kv_len, rows, s0, lane, edge);
        const int blocks = (my.nq * G + kRowBlock - 1) / kRowBlock, scan = wave_scan(blocks);
        const int in = __builtin_amdgcn_readlane(scan, 63);
        if (blk < in) {
            const int sl = __popcll(__ballot(scan <= blk));
            seq = s0 + sl;
            x = SeqWork{__builtin_amdgcn_readlane(my.row0, sl), __builtin_amdgcn_readlane(my.nq, sl),
                        __builtin_amdgcn_readlane(my.len, sl), __builtin_amdgcn_readlane(my.lo, sl)};
            blk = __builtin_amdgcn_readlane(scan, sl) - 1 - blk;   // a sequence's last rows see the most keys: first
            break;
        }
        blk -= in;
    }
    if (seq < 0) return;
    const int row_base = blk * kRowBlock, nrow = min(kRowBlock, x.nq * G - row_base);   // rows r = token · G + g
    // the keys that any row of the block sees, in tiles, and this workgroup's part of them
    const int p0 = x.len - x.nq;
    const int b_hi = a.causal ? max(0, min(x.len, p0 + (row_base + nrow - 1) / G + 1)) : x.len;
    const int b_lo = a.window > 0 ? min(b_hi, max(0, p0 + row_base / G - a.window + 1)) : 0;
    // … and those that every row sees
    const int blk_hi = a.causal ? max(0, min(x.len, p0 + row_base / G + 1)) : x.len;
    const int blk_lo = a.window > 0 ? max(0, p0 + (row_base + nrow - 1) / G - a.window + 1) : 0;
    const int tile0 = b_lo / kPromptKeys, tiles = max(0, (b_hi + kPromptKeys - 1) / kPromptKeys - tile0);
    const int parts = prompt_parts(tiles, fill, HD, splits);
    if (split >= parts) return;
    const int t_begin = tile0 + (int)((int64_t)tiles * split / parts), t_end = tile0 + (int)((int64_t)tiles * (split + 1) / parts);

    // ---- this lane's row
    const int wr0 = row_base + 32 * w, wrows = max(0, min(32, row_base + nrow - wr0));   // the wave's rows
    const int r = wr0 + min(n, max(wrows - 1, 0)), tok = min(r / G, x.nq - 1), head = kvh * G + r % G;
    const int at = p0 + tok;
    const int hi = a.causal ? min(x.len, at + 1) : x.len, lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
    const int all_hi = a.causal ? max(0, min(x.len, p0 + wr0 / G + 1)) : x.len;
    const int all_lo = a.window > 0 ? max(0, p0 + (wr0 + max(wrows, 1) - 1) / G - a.window + 1) : 0;
    const int any_hi = a.causal ? max(0, min(x.len, p0 + (wr0 + max(wrows, 1) - 1) / G + 1)) : x.len;
    const int any_lo = a.window > 0 ? max(0, p0 + wr0 / G - a.window + 1) : 0;
    u32x4 qf[KK];
    {
        const uint16_t* qp = (const uint16_t*)q + (x.row0 + tok) * ldq + (int64_t)head * HD + 8 * h;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            if (q_vec) qf[kk] = *(const u32x4*)(qp + 16 * kk);
            else
#pragma unroll
                for (int i = 0; i < 4; i++) qf[kk][i] = qp[16 * kk + 2 * i] | (uint32_t)qp[16 * kk + 2 * i + 1] << 16;
#pragma unroll
            for (int i = 0; i < 4; i++) qf[kk][i] ^= q_sign;
        }
    }

    // ---- staging: wave w brings the tile's keys 16 w .. 16 w + 15; page ids of 64 tiles at a time, one a lane
    const int* tab = c.table + (int64_t)seq * c.max_pages;
    int id = -1;
    auto ids = [&](int t) {
        const int64_t key = ((int64_t)t + lane) * kPromptKeys + 16 * w;
        id = key < x.len ? tab[key >> c.page_shift] : -1;
    };
    Slice<HD, CT> st;   // 4-bit pages: the next tile's codes
    bool st_ok = false;
    auto fetch = [&](int t, int buf) {
        if (((t - t_begin) & 63) == 0) ids(t);
        const int d = __builtin_amdgcn_readlane(id, (t - t_begin) & 63);
        st_ok = (unsigned)d < (unsigned)c.n_pages;
        if (lane == 0) s_ok[buf][w] = st_ok;
        if (!st_ok) return;
        const int64_t b = ((int64_t)d * c.nkv + kvh) * c.block_bytes;
        const int t0 = (t * kPromptKeys + 16 * w) & ((1 << c.page_shift) - 1);
        if constexpr (CT == T_MXFP4) {
            load_k<HD, CT>(st, 0, block_rsrc(c.k + b, c.block_bytes), t0, codes, lane & 15, lane >> 4);
            load_v<HD, CT>(st, 0, block_rsrc(c.v + b, c.block_bytes), t0, codes, lane & 15, lane >> 4);
        } else {
            constexpr int RPI = 64 / CPR > 0 ? 64 / CPR : 1;   // rows of one 1 KB transfer
#pragma unroll
            for (int i = 0; i < 16 / RPI; i++) {
                const int row = 16 * w + i * RPI + lane / CPR, pos = lane % CPR;
                const uint32_t src = (t0 + i * RPI + lane / CPR) * ROW;
                const uint32_t dst = buf * TILE + (16 * w + i * RPI) * ROW;
                dma_lds16(c.k + b + src + 16 * (pos ^ k_swz<HD>(row)), (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ldsK + dst);
                dma_lds16(c.v + b + src + 16 * (pos ^ v_swz<HD>(row)), (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ldsV + dst);
            }
        }
    };
    auto store = [&](int buf) {   // 4-bit pages: widened into the image that the 16-bit ones have
        if constexpr (CT == T_MXFP4) {
            if (!st_ok) return;
            constexpr int ND = HD / 16;
            const int m = lane & 15, kg = lane >> 4;
            const uint32_t nan_k = nan_scale(st.ks[0][0]) | (HD == 256 ? nan_scale(st.ks[0][HD == 256 ? 1 : 0]) : 0u);
#pragma unroll
            for (int kk = 0; kk < HD / 32; kk++) {
                const float f = __uint_as_float(((st.ks[0][kk / 4] >> (8 * (kk % 4))) & 255) << 23);
                const uint32_t wd = st.k[0][kk];
                u32x4 kf = {fp4_pair<QT>(wd, f, 0), fp4_pair<QT>(wd, f, 1), fp4_pair<QT>(wd, f, 2), fp4_pair<QT>(wd, f, 3)};
                if (nan_k) kf = u32x4{0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};   // its scores are no numbers
                const int row = 16 * w + m, ch = kk * 4 + kg;
                *(u32x4*)(ldsK + buf * TILE + row * ROW + 16 * (ch ^ k_swz<HD>(row))) = kf;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t sb = (st.vs[0] >> (8 * j)) & 255;
                const float f = __uint_as_float(sb << 23);
                const int row = 16 * w + 4 * kg + j;
                uint32_t d[ND / 2];
#pragma unroll
                for (int b = 0; b < ND / 2; b++) {
                    const int i = j * (ND / 2) + b;
                    d[b] = fp4_pair<QT>(st.v[0][i / 4], f, i % 4);
                    if (sb == 255) d[b] = 0x7fff7fffu;
                }
                uint8_t* dst = ldsV + buf * TILE + row * ROW;
                if constexpr (ND == 4) {
                    *(u32x2*)(dst + 16 * ((m / 2) ^ v_swz<HD>(row)) + 8 * (m & 1)) = u32x2{d[0], d[1]};
                } else {
#pragma unroll
                    for (int p = 0; p < ND / 8; p++)
                        *(u32x4*)(dst + 16 * ((m * (ND / 8) + p) ^ v_swz<HD>(row))) =
                            u32x4{d[4 * p], d[4 * p + 1], d[4 * p + 2], d[4 * p + 3]};
                }
            }
        }
    };

    f32x16 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) acc[i][j] = 0.f;
    float m = kNone, l = 0.f;
    bool big = false;   // some row's m is

    // Vᵀ operand: dims 32 dt + n, key slots (h, j) = keys 32 u + 16 s + 8 (j / 4) + 4 h + j % 4
    auto read_v = [&](int buf, int u, int s, int dt) {
        const int g16 = (n >> 4), qr = (n & 15) >> 2, pp = n & 3;
        s16x4 rr[2];
#pragma unroll
        for (int jj = 0; jj < 2; jj++) {
            const int row = 32 * u + 16 * s + 8 * jj + 4 * h + qr, ch = 4 * dt + 2 * g16 + (pp >> 1);
            rr[jj] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(__attribute__((address_space(3))) uint8_t*)(
                    ldsV + buf * TILE + row * ROW + 16 * (ch ^ v_swz<HD>(row)) + 8 * (pp & 1)));
        }
        const u32x2 a0 = __builtin_bit_cast(u32x2, rr[0]), a1 = __builtin_bit_cast(u32x2, rr[1]);
        return __builtin_shufflevector(a0, a1, 0, 1, 2, 3);
    };

    if (t_begin < t_end) fetch(t_begin, 0);
    if constexpr (CT == T_MXFP4)
        if (t_begin < t_end) store(0);
    for (int t = t_begin; t < t_end; t++) {
        const int buf = (t - t_begin) & 1;
        if constexpr (CT != T_MXFP4) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();   // tile t is there, and nobody reads the other buffer any more
        if (t + 1 < t_end) fetch(t + 1, buf ^ 1);
        const int key = t * kPromptKeys;
        int have = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) have |= (s_ok[buf][i] ? 1 : 0) << i;
        have = uniform(have);
        // 0 · V is no zero where V is no number.  In tiles that not every row of the workgroup sees whole: V that no row may
        // use (behind the last key, no page) becomes zero, and keys of whose V any is no number (`odd`) are added apart
        uint64_t odd = 0;
        const int zrow = threadIdx.x >> 2;   // a quarter of a row of V for each thread
        u32x4* const zp = (u32x4*)(ldsV + buf * TILE + zrow * ROW + (threadIdx.x & 3) * (ROW / 4));
        if (have != 15 || key < blk_lo || key + kPromptKeys > blk_hi) {   // the same for the whole workgroup
            const bool real = (have >> (zrow >> 4) & 1) && key + zrow < x.len;
            constexpr uint32_t e = QT == T_F16 ? 0x7c007c00u : 0x7f807f80u;
            u16x2 top = {0, 0};
#pragma unroll
            for (int i = 0; i < ROW / 64; i++) {
                if (!real) zp[i] = u32x4{0, 0, 0, 0};
                else {
                    const u32x4 d = zp[i];
#pragma unroll
                    for (int j = 0; j < 4; j++) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, d[j] & e));
                }
            }
            const uint64_t bad = __ballot(top[0] == (e & 0xffffu) || top[1] == (e & 0xffffu));
            if (lane == 0) s_odd[w] = bad;
            __syncthreads();
            const uint64_t some = s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3];
            if (__builtin_expect(uniform((int)(some | some >> 32)) != 0, 0))
                for (int i = 0; i < 64; i++)
                    if (s_odd[i >> 4] >> (4 * (i & 15)) & 15) odd |= 1ull << i;
        }
        const bool active = wrows > 0 && key < any_hi && key + kPromptKeys > any_lo;
        u32x4 pf[2][2] = {};
        uint32_t see = ~0u;   // bit 16 u + i: score i of half u
        if (active) {
            const bool whole = have == 15 && key >= all_lo && key + kPromptKeys <= all_hi;
            f32x16 sv[2];
            __builtin_amdgcn_s_setprio(1);   // a wave that multiplies goes before one that takes its softmax
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < 16; j++) sv[u][j] = 0.f;
            // 4-bit pages, and one wave a SIMD: the operands of 8 steps are read ahead and each register's next one behind the
            // product that frees it (4-bit pages 3 % faster; 16-bit ones of head_dim 128 4 % slower, two waves hide as much)
            constexpr int AHEAD = kAhead ? (KK < 8 ? KK : 8) : 1, STEPS = 2 * KK;
            auto read_k = [&](int i) {   // step i: half i / KK, dims 16 (i % KK) ..
                const int row = 32 * (i / KK) + n, ch = 2 * (i % KK) + h;
                return *(const u32x4*)(ldsK + buf * TILE + row * ROW + 16 * (ch ^ k_swz<HD>(row)));
            };
            if constexpr (kAhead) {
                u32x4 kf[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; i++) kf[i] = read_k(i);
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    sv[i / KK] = mfma32<QT>(kf[i % AHEAD], qf[i % KK], sv[i / KK]);
                    if (i + AHEAD < STEPS) kf[i % AHEAD] = read_k(i + AHEAD);
                }
                __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    if (i + AHEAD < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < STEPS; i++) sv[i / KK] = mfma32<QT>(read_k(i), qf[i % KK], sv[i / KK]);
            }
            __builtin_amdgcn_s_setprio(0);
            if (!whole) {
                const int k4 = key + 4 * anew(h);
                see = 0;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int kj = k4 + 32 * u + 8 * (i / 4) + i % 4;
                        if ((have >> (2 * u + i / 8) & 1) && kj >= lo && kj < hi) see |= 1u << (16 * u + i);
                        else sv[u][i] = -INFINITY;
                    }
            }
            float mx = sv[0][0];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 16; i++) mx = fmaxf(mx, sv[u][i]);
            mx *= sc;
            if (__any(mx > m + kSlack)) {
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= al;
                big = __any(is_big(m));
#pragma unroll
                for (int i = 0; i < DT; i++) acc[i] *= al;
            }
            float c2 = sc, mk = lift<CT>(x.len) - m;
            if (__builtin_expect(big, 0) && is_big(m)) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 16; i++) sv[u][i] = sv[u][i] * sc - m;
                c2 = 1.f;
                mk = lift<CT>(x.len);
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(fmaf(sv[u][i], c2, mk));
                    const float e1 = __builtin_amdgcn_exp2f(fmaf(sv[u][i + 1], c2, mk));
                    pf[u][i / 8][(i % 8) / 2] = pack2<QT>(e0, e1);
                }
        }
        if (__builtin_expect(odd != 0, 0)) {
            for (uint64_t todo = active ? odd : 0; todo; todo &= todo - 1) {
                const int ki = __builtin_ctzll(todo), kk = ki & 31, own = kk >> 2 & 1;   // the lane half that has its weight
                const int idx = (ki >> 5) * 16 + (kk >> 3) * 4 + (kk & 3);
                uint32_t two = 0;
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (idx >> 1 == j) two = pf[j / 8][(j % 8) / 4][j % 4];
                const uint16_t pb = (uint16_t)(idx & 1 ? two >> 16 : two);
                float pw = QT == T_F16 ? (float)__builtin_bit_cast(_Float16, pb) : (float)__builtin_bit_cast(__bf16, pb);
                int sees = see >> idx & 1;
                const float pw2 = __shfl_xor(pw, 32);
                const int sees2 = __shfl_xor(sees, 32);
                if (h != own) pw = pw2, sees = sees2;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const int ch = 4 * dt + g;
                        const uint16_t* vp = (const uint16_t*)(ldsV + buf * TILE + ki * ROW + 16 * (ch ^ v_swz<HD>(ki)) + 8 * h);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float vv = QT == T_F16 ? (float)__builtin_bit_cast(_Float16, vp[i]) : (float)__builtin_bit_cast(__bf16, vp[i]);
                            if (sees) acc[dt][4 * g + i] = fmaf(pw, vv, acc[dt][4 * g + i]);
                        }
                    }
            }
            __syncthreads();
            if (odd >> zrow & 1)
#pragma unroll
                for (int i = 0; i < ROW / 64; i++) zp[i] = u32x4{0, 0, 0, 0};
            __syncthreads();
        }
        __builtin_amdgcn_s_setprio(1);
        if (active) {
            float ls[4] = {};   // the weights' sum goes into the shadow of the products
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int us = 0; us < 4; us++) ls[us] = add2<QT>(pf[us >> 1][us & 1][j], ls[us]);
            l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
            if constexpr (kAhead) {
                u32x4 vf[DT];
#pragma unroll
                for (int dt = 0; dt < DT; dt++) vf[dt] = read_v(buf, 0, 0, dt);
#pragma unroll
                for (int us = 0; us < 4; us++)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        acc[dt] = mfma32<QT>(vf[dt], pf[us >> 1][us & 1], acc[dt]);
                        if (us < 3) vf[dt] = read_v(buf, (us + 1) >> 1, (us + 1) & 1, dt);
                    }
                __builtin_amdgcn_sched_group_barrier(0x100, 2 * DT, 0);
#pragma unroll
                for (int i = 0; i < 4 * DT; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    if (i < 3 * DT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                }
            } else {
#pragma unroll
                for (int us = 0; us < 4; us++)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
                        acc[dt] = mfma32<QT>(read_v(buf, us >> 1, us & 1, dt), pf[us >> 1][us & 1], acc[dt]);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (CT == T_MXFP4)
            if (t + 1 < t_end) store(buf ^ 1);
    }
    l += __shfl_xor(l, 32);

    // ---- out, or joined with the item's other parts
    bool write = true;
    if (parts > 1) {
        const int item_slot = item * splits;
        float* mine = part + (int64_t)(item_slot + split) * kSlot;
        const uint32_t off = ((w * DT * 4) * 64 + lane) * 16;
        if (wrows > 0) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    wt_st128(mine, off + (dt * 4 + g) * 1024,
                             __builtin_bit_cast(wt_v4i, f32x4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]}));
            if (h == 0) {
                wt_stf(mine, (kRowBlock * HD + 32 * w + n) * 4, m);
                wt_stf(mine, (kRowBlock * (HD + 1) + 32 * w + n) * 4, l);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // written through before the arrival is counted
        __syncthreads();
        if (threadIdx.x == 0)
            s_last = __hip_atomic_fetch_add(&cnt[item], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)parts - 1;
        __syncthreads();
        write = s_last;
        if (write) {
            if (threadIdx.x == 0) __hip_atomic_store(&cnt[item], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            float M = kNone;
            for (int pc = 0; pc < parts; pc++)
                M = fmaxf(M, wt_ldf(part + (int64_t)(item_slot + pc) * kSlot, (kRowBlock * HD + 32 * w + n) * 4));
            l = 0.f;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) acc[i][j] = 0.f;
            for (int pc = 0; pc < (wrows > 0 ? parts : 0); pc++) {
                const float* src = part + (int64_t)(item_slot + pc) * kSlot;
                const float f = __builtin_amdgcn_exp2f(wt_ldf(src, (kRowBlock * HD + 32 * w + n) * 4) - M);
                l = fmaf(wt_ldf(src, (kRowBlock * (HD + 1) + 32 * w + n) * 4), f, l);
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const float4 v4 = wt_ldf4(src, off + (dt * 4 + g) * 1024);
                        acc[dt][4 * g] = fmaf(v4.x, f, acc[dt][4 * g]);
                        acc[dt][4 * g + 1] = fmaf(v4.y, f, acc[dt][4 * g + 1]);
                        acc[dt][4 * g + 2] = fmaf(v4.z, f, acc[dt][4 * g + 2]);
                        acc[dt][4 * g + 3] = fmaf(v4.w, f, acc[dt][4 * g + 3]);
                    }
            }
        }
    }
    if (write && n < wrows) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int64_t at_o = (x.row0 + tok) * ldo + (int64_t)head * HD + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                f32x4 v4 = {acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
                v4 *= inv;
                store_out<QT>(o, a.o_type, at_o + 32 * dt + 8 * g, v4, o_vec);
            }
    }
}

}  // namespace

// Which kernel, by the rows (tokens · heads of a KV head) of a sequence.  The few-row one reads the keys anew for every 16
// rows, which L2 bears for a while; the prompt one has whole blocks of 128 rows to fill and more to start.  To 64 rows the
// first (16 / 8 heads of 128, f16, 64 rows of one sequence of 32,768 keys: 53 against 68 us), past 256 the second; between
// them, over 16-bit pages the first while its list gives no workgroup more than 5 tiles (f16, 256 rows: one sequence of 2,000
// keys 21 against 25 us, of 8,192 47 against 39; 4 of 2,000 67 against 32; 16 of 2,000 101 against 45), over 4-bit ones up to
// 16,384 keys (256 rows: 16 x 2,000 keys 44 against 45 us, 16 x 8,192 131 against 126, 4 x 32,768 287 against 203).
// profiles/paged_attention_choice.txt has both at 342 sizes: the rule is off most at 64 rows of several long sequences over
// 16-bit pages (4 x 32,768 keys 287 against 117 us)
enum Rule { kFew, kMid, kMany };
static Rule rule_of(int G, const AttnArgs& a) {
    const int64_t r = (int64_t)a.max_q * G;
    return r <= 64 ? kFew : r <= 256 ? kMid : kMany;
}
static bool is_prompt(const KvPages& c, const AttnArgs& a, int64_t row_tiles) {
    const Rule rule = rule_of(a.nh / c.nkv, a);
    if (rule != kMid) return rule == kMany;
    const int64_t keys = a.window > 0 ? std::min((int64_t)a.max_kv, (int64_t)a.window + a.max_q) : a.max_kv;
    if (c.type == T_MXFP4) return keys > 16384;
    return row_tiles * cdiv64(keys, kTileKeys) > 5 * 256 * wgs_per_cu(c.hd, c.type);
}

size_t paged_attention_ws(const KvPages& c, const AttnArgs& a) {
    const size_t few = (size_t)kSplitWgs * 4 + (size_t)kSplitWgs * 2 * (16 * c.hd + 32) * 4;
    const size_t many = (size_t)kSplitWgs * 4 + (size_t)kPromptSlots * kRowBlock * (c.hd + 2) * 4;
    return rule_of(a.nh / c.nkv, a) == kFew ? few : std::max(few, many);
}

template <int HD, int CT, int QT>
static void launch(const KvPages& c, const AttnArgs& a, const void* q, int64_t ldq, const int* q_start,
                   const int* kv_len, int rows, void* o, int64_t ldo, void* ws, hipStream_t s) {
    const int G = a.nh / c.nkv;
    const int q_vec = ldq % 8 == 0 && ((uintptr_t)q & 15) == 0;
    const int o_vec = ldo % 4 == 0 && ((uintptr_t)o & 15) == 0;
    unsigned* cnt = (unsigned*)ws;
    float* part = (float*)((char*)ws + kSplitWgs * 4);
    const int used = std::min(rows, c.n_seq);   // sequences with rows, at most
    const int64_t row_tiles = ((int64_t)rows * G / 16 + used) * c.nkv;
    // (a list of 2^30 tiles or more, from far more rows than announced, is the prompt kernel's too: unsplit, without scratch)
    const bool prompt = is_prompt(c, a, row_tiles);
    if (prompt || row_tiles * cdiv64(((int64_t)c.max_pages << c.page_shift) + 1, kTileKeys) >= 1 << 30) {
        const int64_t items = ((int64_t)rows * G / kRowBlock + used) * c.nkv;   // at most
        QASR_CHECK(items < 1 << 24, QASR_E_CAPACITY, "paged_attention: too many rows for one call");
        const int fill = (int)std::min<int64_t>(kPromptParts, std::max<int64_t>(1, kPromptSlots / items));
        // the most parts that an item as long as announced is cut into: a workgroup without one holds a place until it has
        // found that out (3 x 308 rows of 5 heads of 256 on up to 5,339 keys: 52 us, with all `fill` launched 116; with a
        // window of 100 keys 22 against 87)
        int64_t keys = std::min<int64_t>(a.max_kv, 1 << 30);
        if (a.window > 0) keys = std::min<int64_t>(keys, (int64_t)a.window + kPromptKeys + (a.causal ? kRowBlock / G : a.max_q));
        const int splits = prompt ? prompt_parts((int)cdiv64(keys, kPromptKeys) + 1, fill, HD, fill) : 1;
        const size_t lds = 4 * kPromptKeys * HD * 2;
        if constexpr (HD == 256)   // (for the current device; past 64 KB)
            QASR_HIP(hipFuncSetAttribute((const void*)k_paged_prompt<HD, CT, QT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        k_paged_prompt<HD, CT, QT><<<(unsigned)(items * splits), 256, lds, s>>>(c, a, q, ldq, q_start, kv_len, rows, o, ldo,
                                                                               part, cnt, splits, fill, q_vec, o_vec);
        return;
    }
    const int64_t tiles = row_tiles * std::max<int64_t>(1, cdiv64(a.max_kv, kTileKeys));
    const int grid = (int)std::min<int64_t>(256 * wgs_per_cu(HD, CT), tiles);
    k_paged_attn<HD, CT, QT><<<grid, 256, 0, s>>>(c, a, q, ldq, q_start, kv_len, rows, o, ldo, part, cnt, q_vec,
                                                  o_vec);
}

void paged_attention(const KvPages& cache, const AttnArgs& a, const void* q, int64_t ldq, const int* q_start,
                     const int* kv_len, int rows, void* o, int64_t ldo, void* ws, hipStream_t s) {
    if (rows <= 0 || cache.n_seq <= 0) return;
    KvPages c = cache;
    if (c.n_pages == 0) c.max_pages = 0;   // no page to read from: no keys
    auto by_types = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (c.type == T_F16) launch<HD, T_F16, T_F16>(c, a, q, ldq, q_start, kv_len, rows, o, ldo, ws, s);
        else if (c.type == T_BF16) launch<HD, T_BF16, T_BF16>(c, a, q, ldq, q_start, kv_len, rows, o, ldo, ws, s);
        else if (a.q_type == T_F16) launch<HD, T_MXFP4, T_F16>(c, a, q, ldq, q_start, kv_len, rows, o, ldo, ws, s);
        else launch<HD, T_MXFP4, T_BF16>(c, a, q, ldq, q_start, kv_len, rows, o, ldo, ws, s);
    };
    if (c.hd == 64) by_types(std::integral_constant<int, 64>{});
    else if (c.hd == 128) by_types(std::integral_constant<int, 128>{});
    else by_types(std::integral_constant<int, 256>{});
}

}  // namespace qasr
