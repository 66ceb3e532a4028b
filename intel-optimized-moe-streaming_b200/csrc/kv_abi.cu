// kv_abi.cu -- the extern "C" entry points of the paged key/value cache and
// its attention (include/moe_b200.h): argument checks, then the launches.
#include "attend.h"
#include "launch.h"

namespace moeb200 {

namespace {

bool any_type(int t) { return t == KV_F32 || t == KV_F16 || t == KV_BF16; }

int type_bytes(int t) { return t == KV_F32 ? 4 : 2; }

int check_cache(const moe_b200_kv_cache* c, KvCache* out) {
    if (!c || !c->k || !c->v) return ST_ARG;
    if (c->num_pages < 1 || c->kv_heads < 1 || c->kv_heads > 1024) return ST_ARG;
    if (c->type != KV_F16 && c->type != KV_BF16 && c->type != Q8_0) return ST_TYPE;
    if (c->head_dim < 32 || c->head_dim > 256 || c->head_dim % 32) return ST_TYPE;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return ST_ARG;
    if ((int64_t)c->num_pages * c->kv_heads > 0x7fffffffll) return ST_ARG;
    const bool scaled = c->type == Q8_0;
    if (scaled != (c->k_scales != nullptr) || scaled != (c->v_scales != nullptr)) return ST_ARG;
    if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & 15u)
        return ST_ALIGN;
    if (out) {
        int shift = 4;
        while ((1 << shift) < c->page_size) ++shift;
        *out = KvCache{c->k, c->v, static_cast<__half*>(c->k_scales),
                       static_cast<__half*>(c->v_scales), c->type, c->num_pages, c->page_size,
                       shift, c->kv_heads, c->head_dim};
    }
    return ST_OK;
}

int check_batch(const moe_b200_kv_batch* b, KvBatch* out) {
    if (!b || b->sequences < 0 || b->tokens < 0 || b->max_pages < 0) return ST_ARG;
    if (b->sequences > 0 && (!b->q_start || !b->kv_lens)) return ST_ARG;
    if (b->sequences > 0 && b->max_pages > 0 && !b->page_table) return ST_ARG;
    if (b->table_stride < b->max_pages) return ST_ARG;
    if (((uintptr_t)b->q_start | (uintptr_t)b->kv_lens | (uintptr_t)b->page_table) & 3u)
        return ST_ALIGN;
    *out = KvBatch{b->q_start, b->kv_lens, b->page_table, b->table_stride,
                   b->sequences, b->tokens, b->max_pages};
    return ST_OK;
}

bool rows_aligned(const void* p, int64_t ts, int64_t hs, int bytes) {
    return !(((uintptr_t)p | (uintptr_t)(ts * bytes) | (uintptr_t)(hs * bytes)) & 15u);
}

int clear_status(int32_t* status, cudaStream_t s) {
    if (!status) return ST_OK;
    const cudaError_t e = cudaMemsetAsync(status, 0, 4, s);
    return e == cudaSuccess ? ST_OK : cuda_fail(e);
}

int kv_rows(bool write, const moe_b200_kv_cache* cache, const moe_b200_kv_batch* batch, int type,
            void* k, int64_t k_ts, int64_t k_hs, void* v, int64_t v_ts, int64_t v_hs,
            int32_t* status, void* stream) {
    KvCache c;
    KvBatch b;
    int st = check_cache(cache, &c);
    if (st == ST_OK) st = check_batch(batch, &b);
    if (st != ST_OK) return st;
    if (!any_type(type)) return ST_TYPE;
    if (b.T > 0 && (!k || !v)) return ST_ARG;
    const int w = type_bytes(type);
    if (!rows_aligned(k, k_ts, k_hs, w) || !rows_aligned(v, v_ts, v_hs, w) ||
        ((uintptr_t)status & 3u))
        return ST_ALIGN;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    st = clear_status(status, s);
    if (st != ST_OK || b.T == 0 || b.B == 0) return st;
    const cudaError_t e = launch_kv_rows(write, b, c, type, k, k_ts, k_hs, v, v_ts, v_hs,
                                         reinterpret_cast<unsigned*>(status), s);
    return e == cudaSuccess ? ST_OK : cuda_fail(e);
}

}  // namespace

}  // namespace moeb200

using namespace moeb200;

extern "C" {

int moe_b200_kv_write(const moe_b200_kv_cache* cache, const moe_b200_kv_batch* batch, int32_t type,
                      const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                      int64_t v_token_stride, int64_t v_head_stride, int32_t* status,
                      void* stream) {
    try {
        return kv_rows(true, cache, batch, type, const_cast<void*>(k), k_token_stride, k_head_stride,
                       const_cast<void*>(v), v_token_stride, v_head_stride, status, stream);
    } catch (...) {
        return ST_INTERNAL;
    }
}

int moe_b200_kv_read(const moe_b200_kv_cache* cache, const moe_b200_kv_batch* batch, int32_t type,
                     void* k, int64_t k_token_stride, int64_t k_head_stride, void* v,
                     int64_t v_token_stride, int64_t v_head_stride, int32_t* status,
                     void* stream) {
    try {
        return kv_rows(false, cache, batch, type, k, k_token_stride, k_head_stride, v, v_token_stride,
                       v_head_stride, status, stream);
    } catch (...) {
        return ST_INTERNAL;
    }
}

int moe_b200_attend_workspace(const moe_b200_kv_cache* cache, const moe_b200_kv_batch* batch,
                              int32_t q_heads, size_t* bytes) {
    try {
        KvCache c;
        KvBatch b;
        int st = check_cache(cache, &c);
        if (st == ST_OK) st = check_batch(batch, &b);
        if (st != ST_OK) return st;
        if (!bytes || q_heads < 1 || q_heads % c.heads) return ST_ARG;
        *bytes = attend_workspace_bytes(b, c, q_heads);
        return ST_OK;
    } catch (...) {
        return ST_INTERNAL;
    }
}

int moe_b200_attend(const moe_b200_kv_cache* cache, const moe_b200_kv_batch* batch, int32_t type,
                    const void* q, int64_t q_token_stride, int64_t q_head_stride, int32_t q_heads,
                    void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse,
                    float scale, int32_t causal, int32_t window, void* workspace,
                    size_t workspace_bytes, int32_t* status, void* stream) {
    try {
        AttendArgs a{};
        int st = check_cache(cache, &a.c);
        if (st == ST_OK) st = check_batch(batch, &a.b);
        if (st != ST_OK) return st;
        if (type != KV_F16 && type != KV_BF16) return ST_TYPE;
        if (a.c.type != Q8_0 && a.c.type != type) return ST_TYPE;
        if (q_heads < 1 || q_heads > 65536 || q_heads % a.c.heads) return ST_ARG;
        if ((causal != 0 && causal != 1) || window < 0 || (window > 0 && !causal)) return ST_ARG;
        if (!(scale >= -3.402823466e38f && scale <= 3.402823466e38f)) return ST_ARG;
        // a head group's rows are counted up to whole tiles of 256 in 32 bits
        if ((int64_t)a.b.T * q_heads > 0x7fffff00ll) return ST_ARG;
        if (a.b.T > 0 && (!q || !out || !workspace)) return ST_ARG;
        if (!rows_aligned(q, q_token_stride, q_head_stride, 2) ||
            !rows_aligned(out, out_token_stride, out_head_stride, 2) || ((uintptr_t)lse & 3u) ||
            ((uintptr_t)status & 3u) || ((uintptr_t)workspace & 255u))
            return ST_ALIGN;
        if (a.b.T > 0 && workspace_bytes < attend_workspace_bytes(a.b, a.c, q_heads))
            return ST_WORKSPACE;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        st = clear_status(status, s);
        if (st != ST_OK || a.b.T == 0 || a.b.B == 0) return st;
        a.q = q;
        a.out = out;
        a.lse = lse;
        a.q_ts = q_token_stride;
        a.q_hs = q_head_stride;
        a.o_ts = out_token_stride;
        a.o_hs = out_head_stride;
        a.type = type;
        a.q_heads = q_heads;
        a.group = q_heads / a.c.heads;
        a.by_group = FastDiv(a.group);
        a.scale = scale;
        a.causal = causal;
        a.window = window;
        a.status = reinterpret_cast<unsigned*>(status);
        const cudaError_t e = launch_attend(a, workspace, s);
        return e == cudaSuccess ? ST_OK : cuda_fail(e);
    } catch (...) {
        return ST_INTERNAL;
    }
}

}  // extern "C"
