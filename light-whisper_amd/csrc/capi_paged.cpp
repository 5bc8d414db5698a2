// extern "C" entry points of the paged K/V cache operators — see include/qasr.h: checks of arguments, then the launch.
#include <limits.h>
#include <math.h>

#include "../../include/qasr.h"
#include "capi_util.h"
#include "kernels_paged.h"

using namespace qasr;

namespace {

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

hipStream_t stream_of(void* stream) {
    if (stream) {   // a launch on another device's stream would run with this device's kernel image
        hipDevice_t on;
        int cur = 0;
        QASR_HIP(hipStreamGetDevice((hipStream_t)stream, &on));
        QASR_HIP(hipGetDevice(&cur));
        QASR_CHECK((int)on == cur, QASR_E_INVALID, "the stream belongs to another device than the current one");
    }
    return (hipStream_t)stream;
}

KvPages pages_of(const qasr_kv_cache* c, bool pools) {
    QASR_CHECK(c, QASR_E_INVALID, "kv cache: NULL description");
    QASR_CHECK(c->type == QASR_T_F16 || c->type == QASR_T_BF16 || c->type == QASR_T_MXFP4, QASR_E_INVALID,
               "kv cache: type must be f16, bf16 or mxfp4");
    QASR_CHECK(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, QASR_E_INVALID,
               "kv cache: head_dim must be 64, 128 or 256");
    QASR_CHECK(c->n_kv_heads >= 1 && c->n_kv_heads <= 1024, QASR_E_INVALID, "kv cache: n_kv_heads must be 1 .. 1024");
    QASR_CHECK(c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0, QASR_E_INVALID,
               "kv cache: page_size must be a power of two from 16 to 1024");
    QASR_CHECK(c->n_pages >= 0 && c->n_seq >= 0 && c->max_pages >= 0, QASR_E_INVALID, "kv cache: negative count");
    QASR_CHECK((int64_t)c->max_pages * c->page_size <= 1 << 30, QASR_E_INVALID,
               "kv cache: max_pages * page_size must be at most 2^30 positions");
    if (pools) {
        QASR_CHECK(c->n_pages == 0 || (c->k && c->v), QASR_E_INVALID, "kv cache: NULL pool");
        QASR_CHECK(aligned(c->k, 16) && aligned(c->v, 16), QASR_E_INVALID, "kv cache: pools must be 16-byte aligned");
        QASR_CHECK((int64_t)c->n_seq * c->max_pages == 0 || (c->page_table && aligned(c->page_table, 4)), QASR_E_INVALID,
                   "kv cache: NULL or misaligned page table");
    }
    KvPages p{};
    p.k = (uint8_t*)c->k;
    p.v = (uint8_t*)c->v;
    p.table = c->page_table;
    p.n_seq = c->n_seq;
    p.max_pages = c->max_pages;
    p.n_pages = c->n_pages;
    p.page_shift = __builtin_ctz((unsigned)c->page_size);
    p.nkv = c->n_kv_heads;
    p.hd = c->head_dim;
    p.type = c->type;
    const uint32_t n = (uint32_t)c->page_size * c->head_dim;
    p.block_bytes = c->type == QASR_T_MXFP4 ? n / 32 * 17 : n * 2;
    return p;
}

RopeArgs rope_of(const qasr_rope* r, int head_dim) {
    RopeArgs a{};
    if (!r) return a;
    if (r->cs) {
        QASR_CHECK(aligned(r->cs, 8), QASR_E_INVALID, "rope: the table must be 8-byte aligned");
        QASR_CHECK(r->rot_dim >= 0 && r->rot_dim <= head_dim && r->rot_dim % 2 == 0, QASR_E_INVALID,
                   "rope: rot_dim must be even and at most head_dim");
        QASR_CHECK(r->n_pos >= 0, QASR_E_INVALID, "rope: negative n_pos");
        a.cs = r->cs;
        a.n_pos = r->n_pos;
        a.rot = r->rot_dim;
        a.interleaved = r->interleaved != 0;
    }
    if (r->norm_w) {
        QASR_CHECK(aligned(r->norm_w, 4) && r->eps >= 0.f && isfinite(r->eps), QASR_E_INVALID,
                   "rope: norm weight alignment, eps >= 0");
        a.norm_w = r->norm_w;
        a.eps = r->eps;
    }
    return a;
}

Rows rows_of(const void* p, int type, int64_t ld, int64_t width, int64_t rows, const char* what) {
    QASR_CHECK(type == QASR_T_F32 || type == QASR_T_F16 || type == QASR_T_BF16, QASR_E_INVALID,
               std::string(what) + ": type must be f32, f16 or bf16");
    QASR_CHECK(ld >= width && ld <= INT64_MAX / 16 / (rows > 0 ? rows : 1), QASR_E_INVALID,
               std::string(what) + ": row stride below the row's width");
    QASR_CHECK(aligned(p, (size_t)elem_bytes(type)), QASR_E_INVALID, std::string(what) + ": misaligned pointer");
    return Rows{p, type, ld};
}

AttnArgs attn_of(const KvPages& c, const qasr_paged_attn* a) {
    QASR_CHECK(a, QASR_E_INVALID, "paged_attention: NULL description");
    QASR_CHECK(a->n_heads >= 1 && a->n_heads % c.nkv == 0 && a->n_heads <= 65536, QASR_E_INVALID,
               "paged_attention: n_heads must be a multiple of n_kv_heads");
    QASR_CHECK((a->q_type == QASR_T_F16 || a->q_type == QASR_T_BF16) && (c.type == QASR_T_MXFP4 || a->q_type == c.type),
               QASR_E_INVALID, "paged_attention: q must be f16 or bf16, the cache's own type where that has 16 bits");
    QASR_CHECK(a->o_type == a->q_type || a->o_type == QASR_T_F32, QASR_E_INVALID,
               "paged_attention: o must be of q's type or f32");
    QASR_CHECK(isfinite(a->scale * (float)M_LOG2E), QASR_E_INVALID, "paged_attention: scale must be finite, times log2 e too");
    QASR_CHECK(a->window >= 0 && a->max_q >= 0 && a->max_kv >= 0, QASR_E_INVALID, "paged_attention: negative size");
    // no position lies further than 2^30 from another
    return AttnArgs{a->n_heads, a->q_type, a->o_type, a->causal != 0, a->window < 1 << 30 ? a->window : 1 << 30, a->max_q, a->max_kv, a->scale};
}

}  // namespace

extern "C" {

QASR_API int qasr_kv_pool_bytes(const qasr_kv_cache* c, size_t* bytes) {
    return guard([&] {
        const KvPages p = pages_of(c, false);
        QASR_CHECK(bytes, QASR_E_INVALID, "kv_pool_bytes: NULL result");
        *bytes = (size_t)p.n_pages * p.nkv * p.block_bytes;
    });
}

QASR_API int qasr_op_rope_table_scaled(const qasr_rope_scaling* r, int64_t first, int32_t n_pos, float* cs,
                                       void* stream) {
    return guard([&] {
        QASR_CHECK(r, QASR_E_INVALID, "rope table: NULL description");
        QASR_CHECK(r->kind >= QASR_ROPE_PLAIN && r->kind <= QASR_ROPE_YARN, QASR_E_INVALID, "rope table: unknown kind");
        QASR_CHECK(r->rot_dim % 2 == 0 && r->rot_dim >= (r->kind == QASR_ROPE_NTK ? 4 : 2) && r->rot_dim <= 4096,
                   QASR_E_INVALID, "rope table: rot_dim must be even and positive (NTK: at least 4)");
        QASR_CHECK(r->theta > 0 && isfinite(r->theta), QASR_E_INVALID, "rope table: theta must be positive");
        QASR_CHECK(r->kind == QASR_ROPE_PLAIN || (r->factor >= 1 && isfinite(r->factor)), QASR_E_INVALID,
                   "rope table: factor must be at least 1");
        QASR_CHECK(n_pos >= 0 && first >= 0 && first <= (int64_t)1 << 40, QASR_E_INVALID, "rope table: bad positions");
        QASR_CHECK(n_pos == 0 || (cs && aligned(cs, 8)), QASR_E_INVALID, "rope table: NULL or misaligned table");
        RopeFreqs f{r->kind, r->rot_dim, log2(r->theta), 1.0, 0.0, 0.0, 1.0};
        const double rot = r->rot_dim;
        if (r->kind != QASR_ROPE_PLAIN) f.inv_factor = 1.0 / r->factor;
        if (r->kind == QASR_ROPE_NTK) f.log2_theta += log2(r->factor) * rot / (rot - 2.0);
        if (r->kind == QASR_ROPE_YARN) {
            QASR_CHECK(r->theta > 1 && r->orig_ctx > 0 && isfinite(r->orig_ctx) && r->beta_slow > 0 &&
                           r->beta_fast >= r->beta_slow && isfinite(r->beta_fast),
                       QASR_E_INVALID, "rope table: YaRN needs theta > 1, orig_ctx > 0, beta_fast >= beta_slow > 0");
            const double ln = log(r->theta);
            auto dim = [&](double beta) { return rot * log(r->orig_ctx / (beta * 2 * M_PI)) / (2 * ln); };
            const double lo = fmax(floor(dim(r->beta_fast)), 0.0), hi = fmin(ceil(dim(r->beta_slow)), rot - 1);
            f.lo = lo;
            f.inv_span = 1.0 / fmax(hi - lo, 1e-3);
            f.mscale = 0.1 * log(r->factor) + 1.0;
        }
        rope_table_scaled(f, first, n_pos, cs, stream_of(stream));
        QASR_HIP(hipGetLastError());
    });
}

QASR_API int qasr_op_rope(const void* x, int32_t x_type, int64_t ldx, const int32_t* pos, int32_t rows, int32_t heads,
                          int32_t head_dim, const qasr_rope* rope, void* y, int32_t y_type, int64_t ldy, void* stream) {
    return guard([&] {
        QASR_CHECK(rows >= 0 && heads >= 1 && heads <= 65536 && head_dim >= 2 && head_dim <= 1024 && head_dim % 2 == 0,
                   QASR_E_INVALID, "rope: rows >= 0, heads >= 1, head_dim even and at most 1024");
        QASR_CHECK(rope, QASR_E_INVALID, "rope: NULL description");
        QASR_CHECK((int64_t)rows * heads <= INT_MAX, QASR_E_INVALID, "rope: rows * heads must stay below 2^31");
        const int64_t w = (int64_t)heads * head_dim;
        const Rows xr = rows_of(x, x_type, ldx, w, rows, "rope: x"), yr = rows_of(y, y_type, ldy, w, rows, "rope: y");
        const RopeArgs r = rope_of(rope, head_dim);
        if (rows == 0) return;
        QASR_CHECK(x && y && (!r.cs || (pos && aligned(pos, 4))), QASR_E_INVALID, "rope: NULL argument");
        QASR_CHECK(x != y || (x_type == y_type && ldx == ldy), QASR_E_INVALID,
                   "rope: in place needs one type and stride");
        rope_rows(xr, pos, rows, heads, head_dim, r, yr, stream_of(stream));
        QASR_HIP(hipGetLastError());
    });
}

QASR_API int qasr_op_kv_append(const qasr_kv_cache* c, const void* k, const void* v, int32_t x_type, int64_t ldk,
                               int64_t ldv, const int32_t* seq, const int32_t* pos, int32_t rows, const qasr_rope* rope,
                               void* stream) {
    return guard([&] {
        const KvPages p = pages_of(c, true);
        QASR_CHECK(rows >= 0 && (int64_t)rows * p.nkv <= INT_MAX, QASR_E_INVALID, "kv_append: bad row count");
        const int64_t w = (int64_t)p.nkv * p.hd;
        const Rows kr = rows_of(k, x_type, ldk, w, rows, "kv_append: k"), vr = rows_of(v, x_type, ldv, w, rows, "kv_append: v");
        const RopeArgs r = rope_of(rope, p.hd);
        if (rows == 0 || p.n_seq == 0 || p.max_pages == 0 || p.n_pages == 0) return;
        QASR_CHECK(k && v && seq && pos && aligned(seq, 4) && aligned(pos, 4), QASR_E_INVALID, "kv_append: NULL argument");
        kv_append(p, kr, vr, seq, pos, rows, r, stream_of(stream));
        QASR_HIP(hipGetLastError());
    });
}

QASR_API int qasr_op_kv_gather(const qasr_kv_cache* c, const int32_t* seq, const int32_t* pos, int32_t rows, void* k,
                               void* v, int32_t y_type, int64_t ldk, int64_t ldv, void* stream) {
    return guard([&] {
        const KvPages p = pages_of(c, true);
        QASR_CHECK(rows >= 0 && (int64_t)rows * p.nkv <= INT_MAX, QASR_E_INVALID, "kv_gather: bad row count");
        const int64_t w = (int64_t)p.nkv * p.hd;
        const Rows kr = rows_of(k, y_type, k ? ldk : w, w, rows, "kv_gather: k"),
                   vr = rows_of(v, y_type, v ? ldv : w, w, rows, "kv_gather: v");
        if (rows == 0 || p.n_seq == 0 || p.max_pages == 0 || p.n_pages == 0 || (!k && !v)) return;
        QASR_CHECK(seq && pos && aligned(seq, 4) && aligned(pos, 4), QASR_E_INVALID, "kv_gather: NULL argument");
        kv_gather(p, seq, pos, rows, kr, vr, stream_of(stream));
        QASR_HIP(hipGetLastError());
    });
}

QASR_API int qasr_paged_attention_workspace(const qasr_kv_cache* c, const qasr_paged_attn* a, size_t* bytes) {
    return guard([&] {
        const KvPages p = pages_of(c, false);
        const AttnArgs at = attn_of(p, a);
        QASR_CHECK(bytes, QASR_E_INVALID, "paged_attention_workspace: NULL result");
        *bytes = paged_attention_ws(p, at);
    });
}

QASR_API int qasr_op_paged_attention(const qasr_kv_cache* c, const qasr_paged_attn* a, const void* q, int64_t ldq,
                                     const int32_t* q_start, const int32_t* kv_len, int32_t rows, void* o, int64_t ldo,
                                     void* ws, size_t ws_bytes, void* stream) {
    return guard([&] {
        const KvPages p = pages_of(c, true);
        const AttnArgs at = attn_of(p, a);
        QASR_CHECK(rows >= 0 && (int64_t)rows * at.nh <= 1 << 30, QASR_E_INVALID,
                   "paged_attention: rows * n_heads must be at most 2^30");
        const int64_t w = (int64_t)at.nh * p.hd;
        rows_of(q, at.q_type, ldq, w, rows, "paged_attention: q");
        rows_of(o, at.o_type, ldo, w, rows, "paged_attention: o");
        if (rows == 0 || p.n_seq == 0) return;
        QASR_CHECK(q && o && q_start && kv_len && aligned(q_start, 4) && aligned(kv_len, 4), QASR_E_INVALID,
                   "paged_attention: NULL argument");
        QASR_CHECK(q != o || (at.q_type == at.o_type && ldq == ldo), QASR_E_INVALID,
                   "paged_attention: in place needs one type and stride");
        const size_t need = paged_attention_ws(p, at);
        QASR_CHECK(need == 0 || (ws && aligned(ws, 128) && ws_bytes >= need), QASR_E_CAPACITY,
                   "paged_attention: the workspace is smaller than qasr_paged_attention_workspace says, or misaligned");
        paged_attention(p, at, q, ldq, q_start, kv_len, rows, o, ldo, ws, stream_of(stream));
        QASR_HIP(hipGetLastError());
    });
}

}  // extern "C"
