// attend.cu -- attention of new token rows over a paged key/value cache:
//   o = sum_j softmax_j(scale * q . k_j) v_j  over the keys the row attends,
// one pass over the keys with a running maximum m and sum l of the softmax
// (o and l are multiplied by exp(m_old - m_new) when the maximum grows).
// One warp per (row, query head), a lane holds every 32nd value of the head.
#include "attend.h"
#include "launch.h"

namespace moeb200 {

namespace {

template <typename TC>
__device__ __forceinline__ float cache_value(const void* p, const __half* s, int64_t row, int dim,
                                             int d) {
    if constexpr (sizeof(TC) == 1)
        return round16(__half2float(s[row * (dim >> 5) + (d >> 5)]) *
                       (float)static_cast<const int8_t*>(p)[row * dim + d]);
    else
        return kv_to_f<TC>(static_cast<const TC*>(p)[row * dim + d]);
}

template <typename TQ, typename TC>
__global__ void __launch_bounds__(128) k_attend_rows(AttendArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= (int64_t)a.b.T * a.q_heads) return;
    const int t = (int)(w / a.q_heads), h = (int)(w % a.q_heads), kvh = h / a.group;
    const int s = kv_find_seq(a.b, t);
    if (s < 0) return;
    const int len = a.b.kv_lens[s];
    const int pos = len - a.b.q_start[s + 1] + t;
    int lo, hi;
    attend_range(pos, kv_length(a.b, a.c, s, a.status), a.causal, a.window, lo, hi);
    const int nd = a.c.dim >> 5;
    float q[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        o[i] = 0.f;
        q[i] = i < nd ? kv_to_f<TQ>(static_cast<const TQ*>(a.q)[t * a.q_ts + h * a.q_hs + 32 * i + lane])
                      : 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = lo; j < hi; ++j) {
        const int page = kv_page(a.b, a.c, s, j >> a.c.page_shift, lane == 0 ? a.status : nullptr);
        if (page < 0) continue;
        const int64_t row = (((int64_t)page * a.c.heads + kvh) << a.c.page_shift) +
                            (j & (a.c.page_size - 1));
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < nd)
                dot = fmaf(q[i], cache_value<TC>(a.c.k, a.c.ks, row, a.c.dim, 32 * i + lane), dot);
        const float sc = warp_sum(dot) * a.scale;
        const float mn = fmaxf(m, sc);
        const float keep = mn == -INFINITY ? 1.f : expf(m - mn);
        const float p = expf(sc - mn);
        m = mn;
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < nd)
                o[i] = o[i] * keep + p * cache_value<TC>(a.c.v, a.c.vs, row, a.c.dim, 32 * i + lane);
    }
    const bool empty = lo >= hi;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < nd)
            static_cast<TQ*>(a.out)[t * a.o_ts + h * a.o_hs + 32 * i + lane] =
                kv_from_f<TQ>(empty ? 0.f : o[i] / l);
    if (a.lse && lane == 0)
        a.lse[(int64_t)t * a.q_heads + h] = empty ? -INFINITY : m + logf(l);
}

}  // namespace

size_t attend_workspace_bytes(const KvBatch&, const KvCache&, int) { return 256; }

cudaError_t launch_attend(const AttendArgs& a, void*, cudaStream_t s) {
    const int64_t warps = (int64_t)a.b.T * a.q_heads;
    const unsigned grid = (unsigned)((warps + 3) / 4);
    if (a.c.type == KV_F16)
        k_attend_rows<__half, __half><<<grid, 128, 0, s>>>(a);
    else if (a.c.type == KV_BF16)
        k_attend_rows<__nv_bfloat16, __nv_bfloat16><<<grid, 128, 0, s>>>(a);
    else if (a.type == KV_F16)
        k_attend_rows<__half, int8_t><<<grid, 128, 0, s>>>(a);
    else
        k_attend_rows<__nv_bfloat16, int8_t><<<grid, 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace moeb200
