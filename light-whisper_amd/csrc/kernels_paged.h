// The paged K/V cache operators (include/qasr.h, "paged K/V cache"): validated views of the C descriptions and the launch
// wrappers (kernels_paged.hip, kernels_pattn.hip).  As in kernels.h: device pointers and a stream, no allocation, no
// synchronisation, graph-capturable.
#pragma once
#include "common.h"

namespace qasr {

enum ElemType : int { T_F32 = 0, T_F16 = 1, T_BF16 = 2, T_MXFP4 = 3 };
inline int elem_bytes(int t) { return t == T_F32 ? 4 : 2; }

struct KvPages {
    uint8_t* k;
    uint8_t* v;
    const int* table;
    int n_seq, max_pages, n_pages, page_shift, nkv, hd, type;
    uint32_t block_bytes;   // one (page, KV head)
};
struct RopeArgs {
    const float* cs;
    int n_pos, rot, interleaved;
    const float* norm_w;
    float eps;
};
// x / y: element type, row stride in elements
struct Rows {
    const void* p;
    int type;
    int64_t ld;
};

// what a table's frequencies follow from
struct RopeFreqs {
    int kind, rot;
    double log2_theta, inv_factor, lo, inv_span, mscale;
};
void rope_table_scaled(const RopeFreqs& f, int64_t first, int n_pos, float* cs, hipStream_t s);
void rope_rows(const Rows& x, const int* pos, int rows, int heads, int hd, const RopeArgs& r, const Rows& y,
               hipStream_t s);
void kv_append(const KvPages& c, const Rows& k, const Rows& v, const int* seq, const int* pos, int rows,
               const RopeArgs& r, hipStream_t s);
void kv_gather(const KvPages& c, const int* seq, const int* pos, int rows, const Rows& k, const Rows& v,
               hipStream_t s);

struct AttnArgs {
    int nh, q_type, o_type, causal, window, max_q, max_kv;
    float scale;
};
size_t paged_attention_ws(const KvPages& c, const AttnArgs& a);
void paged_attention(const KvPages& c, const AttnArgs& a, const void* q, int64_t ldq, const int* q_start,
                     const int* kv_len, int rows, void* o, int64_t ldo, void* ws, hipStream_t s);

}  // namespace qasr
