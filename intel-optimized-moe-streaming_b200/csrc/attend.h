// attend.h -- arguments of the attention over a paged cache.
#pragma once

#include "kv.cuh"

namespace moeb200 {

struct AttendArgs {
    KvBatch b;
    KvCache c;
    const void* q;    // [T][q_heads][dim], strides in elements
    void* out;
    float* lse;       // [T][q_heads] or null
    int64_t q_ts, q_hs, o_ts, o_hs;
    int type;         // of q and out
    int q_heads, group;
    float scale;
    int causal, window;
    unsigned* status;
};

cudaError_t launch_kv_rows(bool write, const KvBatch& b, const KvCache& c, int type, void* k,
                           int64_t k_ts, int64_t k_hs, void* v, int64_t v_ts, int64_t v_hs,
                           unsigned* status, cudaStream_t s);

size_t attend_workspace_bytes(const KvBatch& b, const KvCache& c, int q_heads);
cudaError_t launch_attend(const AttendArgs& a, void* ws, cudaStream_t s);

// Keys [lo, hi) that the row at position pos attends.
__host__ __device__ __forceinline__ void attend_range(int pos, int kv_len, int causal, int window,
                                                      int& lo, int& hi) {
    hi = causal ? (pos + 1 < kv_len ? pos + 1 : kv_len) : kv_len;
    lo = window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0;
    if (hi < lo) hi = lo;
}

}  // namespace moeb200
