// Attention over a paged K/V cache (include/qasr.h, qasr_op_paged_attention), gfx950.
//
// Query rows of one sequence and KV head are numbered r = token · G + g (G query heads share a KV head), so that every K/V
// byte that is loaded serves all G heads, and taken 16 at a time as the columns of v_mfma_f32_16x16x32:
//   Sᵀ = K·Qᵀ   (16 keys × 16 rows; a lane holds 4 keys of ONE row, so the softmax needs no cross-lane work but a vote)
//   Oᵀ = Vᵀ·Pᵀ  (16 dims × 16 rows; the lane's 8 weights of 32 keys are the B operand as they stand: contraction slot
//                (lane >> 4, j) stands for key 16 (j >> 2) + 4 (lane >> 4) + (j & 3), and V is loaded to match)
// No K/V byte passes LDS: K rows are loaded in the A operand's layout; a lane loads hd/16 dims of its 8 keys of V and
// pairs them key by key in registers (v_perm), which makes MFMA row m of tile t dim (hd/16) m + t.
#include "paged_dev.h"
#include "wt.h"

namespace qasr {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kTileKeys = 128;   // keys of one workgroup step: 32 for each of its 4 waves
constexpr int kSplitWgs = 1024;  // workgroups at most (what the scratch is sized for)
// workgroups that a CU holds by their registers
constexpr int wgs_per_cu(int hd, int ct) { return ct == T_MXFP4 ? (hd == 256 ? 2 : 3) : hd == 256 ? 1 : 2; }
// weights are exp2(s − m + kUp), m at most kSlack below the running maximum: at most 2^15 in f16, and its normal range
// reaches 26 bits further down
constexpr float kSlack = 3.f, kUp = 12.f;
constexpr float kNone = -3.0e38f;   // running maximum before the first key

template <int QT>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (QT == T_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                       0);
}
// two f32 → a packed pair of QT, rounded to nearest even
template <int QT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (QT == T_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
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
// inclusive prefix sum over the wave
__device__ __forceinline__ int wave_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// what one sequence asks for (per lane while scanning, uniform afterwards)
struct SeqWork {
    int row0, nq, len, lo;   // first row of q, rows, keys, first key that any row sees
};
__device__ __forceinline__ SeqWork seq_work(const KvPages& c, const AttnArgs& a, const int* q_start, const int* kv_len,
                                            int rows, int s) {
    SeqWork w;
    w.row0 = max(q_start[s], 0);
    w.nq = max(min(q_start[s + 1], rows) - w.row0, 0);
    w.len = (int)min((int64_t)max(kv_len[s], 0), (int64_t)c.max_pages << c.page_shift);
    // the first row's window starts furthest left; with len < nq its position is negative
    w.lo = a.window > 0 ? max(w.len - w.nq - a.window + 1, 0) : 0;
    return w;
}

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

// ------------------------------------------------------------------------------------------------ few rows
// One launch over every sequence: the work is the list of (sequence, 16-row tile, KV head) items, each ⌈keys / 128⌉ tiles
// long; workgroup w takes tiles [w · per, (w + 1) · per) of the whole list, so lengths that differ a thousandfold load the
// workgroups alike.  A workgroup's part of an item is a segment; a segment that is not its whole item leaves its
// (m, l, Oᵀ) in the scratch, and the last of the item's workgroups to arrive adds them up in their order (the result does
// not depend on who is last).  Slot 0 of a workgroup: the item began in an earlier one; slot 1: it goes on in a later one.
template <int HD, int CT, int QT>
__global__ __launch_bounds__(256, wgs_per_cu(HD, CT)) void k_paged_attn(KvPages c, AttnArgs a, const void* __restrict__ q, int64_t ldq,
                                                       const int* __restrict__ q_start, const int* __restrict__ kv_len,
                                                       int rows, void* __restrict__ o, int64_t ldo, float* part,
                                                       unsigned* cnt, int min_tiles, int q_vec, int o_vec) {
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
    int chunk = 0, before = 0, total = 0;   // first sequence held in the lanes, tiles before it, all tiles
    SeqWork my{};
    int scan = 0;   // tiles up to and with this lane's sequence, from `chunk` on
    auto hold = [&](int s0) {
        chunk = s0;
        my = SeqWork{0, 0, 0, 0};
        if (s0 + lane < c.n_seq) my = seq_work(c, a, q_start, kv_len, rows, s0 + lane);
        scan = wave_scan(my.nq > 0 ? items_of(my) * tiles_of(my) : 0);
    };
    for (int s0 = 0; s0 < c.n_seq; s0 += LANES) {
        hold(s0);
        total += __builtin_amdgcn_readlane(scan, 63);
    }
    const int per = max(min_tiles, (total + (int)gridDim.x - 1) / (int)gridDim.x);
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
        auto clear = [&] {
#pragma unroll
            for (int i = 0; i < ND; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            m = kNone;
            l = 0.f;
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
#pragma unroll
                    for (int t2 = 0; t2 < ND; t2++) acc[t2] *= al;
                }
                u32x4 pf;
                const float mk = kUp - m;
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] = __builtin_amdgcn_exp2f(fmaf(p[j], sc, mk));
#pragma unroll
                for (int j = 0; j < 4; j++) pf[j] = pack2<QT>(p[2 * j], p[2 * j + 1]);
                l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
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
            if (a.o_type == T_F32) {
                float* op = (float*)o + at_o;
#pragma unroll
                for (int t2 = 0; t2 < ND; t2 += 4) {
                    if (o_vec) *(f32x4*)(op + t2) = f32x4{out[t2], out[t2 + 1], out[t2 + 2], out[t2 + 3]};
                    else
#pragma unroll
                        for (int i = 0; i < 4; i++) op[t2 + i] = out[t2 + i];
                }
            } else {
                uint16_t* op = (uint16_t*)o + at_o;
#pragma unroll
                for (int t2 = 0; t2 < ND; t2 += 4) {
                    const u32x2 d = {pack2<QT>(out[t2], out[t2 + 1]), pack2<QT>(out[t2 + 2], out[t2 + 3])};
                    if (o_vec) *(u32x2*)(op + t2) = d;
                    else
#pragma unroll
                        for (int i = 0; i < 4; i++) op[t2 + i] = (uint16_t)(d[i / 2] >> (16 * (i & 1)));
                }
            }
        }
        t += seg;
    }
}

}  // namespace

size_t paged_attention_ws(const KvPages& c, const AttnArgs& a) {
    return (size_t)kSplitWgs * 4 + (size_t)kSplitWgs * 2 * (16 * c.hd + 32) * 4;
}

template <int HD, int CT, int QT>
static void launch(const KvPages& c, const AttnArgs& a, const void* q, int64_t ldq, const int* q_start,
                   const int* kv_len, int rows, void* o, int64_t ldo, void* ws, hipStream_t s) {
    const int G = a.nh / c.nkv, min_tiles = 1;
    const int64_t items = ((int64_t)rows * G / 16 + c.n_seq) * c.nkv;   // at most
    const int64_t tiles = items * std::max<int64_t>(1, cdiv64(a.max_kv, kTileKeys));
    const int grid = (int)std::min<int64_t>(256 * wgs_per_cu(HD, CT), std::max<int64_t>(1, cdiv64(tiles, min_tiles)));
    const int q_vec = ldq % 8 == 0 && ((uintptr_t)q & 15) == 0;
    const int o_vec = ldo % 4 == 0 && ((uintptr_t)o & 15) == 0;
    k_paged_attn<HD, CT, QT><<<grid, 256, 0, s>>>(c, a, q, ldq, q_start, kv_len, rows, o, ldo,
                                                  (float*)((char*)ws + kSplitWgs * 4), (unsigned*)ws, min_tiles, q_vec,
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
