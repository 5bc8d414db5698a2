// Attention over a paged K/V cache (include/qasr.h, qasr_op_paged_attention).
#include "paged_dev.h"

namespace qasr {

template <int CT>
__device__ __forceinline__ float cache_value(const KvPages& c, const uint8_t* blk, bool is_v, int t, int d) {
    if constexpr (CT == T_MXFP4) {
        const uint32_t codes = (c.hd / 2) << c.page_shift;
        const uint32_t b = blk[(is_v ? fp4_v_code : fp4_k_code)(c.hd, t, d)];
        return fp4_value(d & 1 ? b >> 4 : b & 15, blk[codes + (is_v ? fp4_v_scale : fp4_k_scale)(c.hd, t, d)]);
    } else {
        return (float)((const typename Elem<CT>::type*)blk)[t * c.hd + d];
    }
}

// one (row, query head) by one wave: 64 keys at a time, a key per lane for the scores, dims over lanes for P·V
template <int CT, int QT, int OT>
__global__ __launch_bounds__(64) void k_paged_attn_row(KvPages c, AttnArgs a, const void* q, int64_t ldq,
                                                       const int* __restrict__ q_start, const int* __restrict__ kv_len,
                                                       int rows, void* o, int64_t ldo) {
    __shared__ float qs[256], ps[64];
    const int row = blockIdx.x / a.nh, head = blockIdx.x % a.nh, lane = threadIdx.x;
    int seq = -1, n = 0, i = 0;
    for (int s = 0; s < c.n_seq; s++) {
        const int r0 = max(q_start[s], 0), r1 = min(q_start[s + 1], rows);
        if (row >= r0 && row < r1) { seq = s; n = r1 - r0; i = row - r0; break; }
    }
    if (seq < 0) return;
    const auto* qp = (const typename Elem<QT>::type*)q + row * ldq + (int64_t)head * c.hd;
    for (int d = lane; d < c.hd; d += 64) qs[d] = (float)qp[d];
    __syncthreads();
    const int len = (int)min((int64_t)max(kv_len[seq], 0), (int64_t)c.max_pages << c.page_shift);
    const int at = len - n + i, hi = a.causal ? min(len, at + 1) : len;
    const int lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
    const int kvh = head / (a.nh / c.nkv), mask = (1 << c.page_shift) - 1;
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = lo; k0 < hi; k0 += 64) {
        const int key = k0 + lane;
        const int64_t blk = key < hi ? page_block(c, seq, key, kvh) : -1;
        float s = -INFINITY;
        if (blk >= 0) {
            s = 0.f;
            for (int d = 0; d < c.hd; d++) s = fmaf(qs[d], cache_value<CT>(c, c.k + blk, false, key & mask, d), s);
            s *= a.scale;
        }
        float mx = s;
        for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
        const float mn = fmaxf(m, mx);
        const float al = mn == -INFINITY ? 1.f : expf(m - mn), p = blk < 0 || mn == -INFINITY ? 0.f : expf(s - mn);
        float sum = p;
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
        l = l * al + sum;
        m = mn;
        ps[lane] = p;
        __syncthreads();
        for (int j = 0; j < 4; j++) {
            acc[j] *= al;
            const int d = lane + 64 * j;
            if (d >= c.hd) continue;
            for (int kk = 0; kk < 64 && k0 + kk < hi; kk++) {
                const int64_t b = page_block(c, seq, k0 + kk, kvh);
                if (b >= 0) acc[j] = fmaf(ps[kk], cache_value<CT>(c, c.v + b, true, (k0 + kk) & mask, d), acc[j]);
            }
        }
        __syncthreads();
    }
    auto* op = (typename Elem<OT>::type*)o + row * ldo + (int64_t)head * c.hd;
    for (int j = 0; j < 4; j++)
        if (lane + 64 * j < c.hd) op[lane + 64 * j] = (typename Elem<OT>::type)(l == 0.f ? 0.f : acc[j] / l);
}

size_t paged_attention_ws(const KvPages& c, const AttnArgs& a) { return 0; }

template <int CT, int QT>
static void launch_row(const KvPages& c, const AttnArgs& a, const void* q, int64_t ldq, const int* q_start,
                       const int* kv_len, int rows, void* o, int64_t ldo, hipStream_t s) {
    const unsigned grid = (unsigned)rows * a.nh;
    if (a.o_type == T_F32)
        k_paged_attn_row<CT, QT, T_F32><<<grid, 64, 0, s>>>(c, a, q, ldq, q_start, kv_len, rows, o, ldo);
    else
        k_paged_attn_row<CT, QT, QT><<<grid, 64, 0, s>>>(c, a, q, ldq, q_start, kv_len, rows, o, ldo);
}

void paged_attention(const KvPages& c, const AttnArgs& a, const void* q, int64_t ldq, const int* q_start,
                     const int* kv_len, int rows, void* o, int64_t ldo, void* ws, hipStream_t s) {
    if (rows <= 0 || c.n_seq <= 0) return;
    if (c.type == T_F16) launch_row<T_F16, T_F16>(c, a, q, ldq, q_start, kv_len, rows, o, ldo, s);
    else if (c.type == T_BF16) launch_row<T_BF16, T_BF16>(c, a, q, ldq, q_start, kv_len, rows, o, ldo, s);
    else if (a.q_type == T_F16) launch_row<T_MXFP4, T_F16>(c, a, q, ldq, q_start, kv_len, rows, o, ldo, s);
    else launch_row<T_MXFP4, T_BF16>(c, a, q, ldq, q_start, kv_len, rows, o, ldo, s);
}

}  // namespace qasr
