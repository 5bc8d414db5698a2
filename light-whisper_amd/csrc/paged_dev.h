// Device code shared by the paged K/V cache kernels: element types, places in pages, the e2m1 / e8m0 format.
#pragma once
#include "kernels_paged.h"

namespace qasr {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <int T>
struct Elem;
template <>
struct Elem<T_F32> { typedef float type; };
template <>
struct Elem<T_F16> { typedef _Float16 type; };
template <>
struct Elem<T_BF16> { typedef __bf16 type; };

// the block of (seq, pos)'s page and KV head `head`, as a byte offset in either pool; -1: no such place
__device__ __forceinline__ int64_t page_block(const KvPages& c, int seq, int pos, int head) {
    if ((unsigned)seq >= (unsigned)c.n_seq || pos < 0 || (pos >> c.page_shift) >= c.max_pages) return -1;
    const int page = c.table[(int64_t)seq * c.max_pages + (pos >> c.page_shift)];
    if ((unsigned)page >= (unsigned)c.n_pages) return -1;
    return ((int64_t)page * c.nkv + head) * c.block_bytes;
}

// byte offset in an MXFP4 block of the code of (token, dim) (its half: dim & 1), and of its scale
__device__ __forceinline__ uint32_t fp4_k_code(int hd, int t, int d) {
    return t * (hd / 2) + ((d % 32) / 8) * (hd / 8) + (d / 32) * 4 + (d % 8) / 2;
}
__device__ __forceinline__ uint32_t fp4_v_code(int hd, int t, int d) {
    const int nd = hd / 16;
    return (t / 16) * 8 * hd + ((((t % 16) / 4) * 16 + d / nd) * 4 + t % 4) * (nd / 2) + (d % nd) / 2;
}
__device__ __forceinline__ uint32_t fp4_k_scale(int hd, int t, int d) { return t * (hd / 32) + d / 32; }
__device__ __forceinline__ uint32_t fp4_v_scale(int hd, int t, int d) {
    return (t / 16) * (hd / 2) + (d / 32) * 16 + t % 16;
}

// scale byte of a block of 32 with this max |x| (any non-finite input: 255).  x = 1.m · 2^e ≤ 6 · 2^E = 1.5 · 2^(E+2):
// E = e − 2 where 1.m ≤ 1.5, else e − 1; kept in [−23, 13]
__device__ __forceinline__ int fp4_scale(float amax) {
    const uint32_t b = __float_as_uint(amax) & 0x7fffffffu;
    if (b >= 0x7f800000u) return 255;
    const int e = (int)(b >> 23) - 127 - ((b & 0x7fffffu) <= 0x400000u ? 2 : 1);
    return min(max(e, -23), 13) + 127;
}
__device__ __forceinline__ float fp4_value(uint32_t code, uint32_t scale) {
    if (scale == 255) return __uint_as_float(0x7fc00000u);
    const uint32_t m = code & 7;
    // 0, ½, then 1.m · 2^(e−1): m < 2 has no leading one
    const float v = m < 2 ? 0.5f * m : __uint_as_float((126 + (m >> 1)) << 23 | (m & 1) << 22);
    const float r = v * __uint_as_float(scale << 23);
    return code & 8 ? -r : r;
}

}  // namespace qasr
