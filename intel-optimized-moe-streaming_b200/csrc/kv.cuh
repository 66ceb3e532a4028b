// kv.cuh -- the paged key/value cache as the kernels see it: page lookup,
// the sequence of a token row, and the Q8_0 block arithmetic of the cache.
//
// Layout: k and v are [page][kv head][row in page][head_dim], so the rows of
// one head in one page are contiguous and a tile of keys is one copy.  A
// Q8_0 cache keeps int8 codes in that layout and the binary16 scales (one
// per 32 values) in a plane of their own, [page][kv head][row][head_dim/32]:
// the 34-byte blocks of a GGUF row would leave no tile 16-byte aligned.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace moeb200 {

// ggml type ids of the plain types (F32, F16, BF16); Q8_0 is common.cuh's.
enum : int { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 30 };

// Bits of the status word.
enum : unsigned { KV_BAD_PAGE = 1, KV_BAD_LENGTH = 2, KV_TIMEOUT = 4 };

// Largest scale a written block gets: 127 * 515.5 = 65468.5, below binary16's
// largest value, so code * scale never overflows binary16.
constexpr float kKvScaleMax = 515.5f;
constexpr int kKvBlock = 32;

struct KvBatch {
    const int32_t* q_start;   // [B + 1] first row of each sequence
    const int32_t* kv_lens;   // [B] cached tokens, the new ones included
    const int32_t* table;     // [B][max_pages], row stride table_stride; null: page p of
                              // sequence b is b * max_pages + p
    int64_t table_stride;
    int B, T, max_pages;
};

struct KvCache {
    void* k;
    void* v;
    __half* ks;   // Q8_0 scales, else null
    __half* vs;
    int type, pages, page_size, page_shift, heads, dim;
};

__device__ __forceinline__ void kv_flag(unsigned* status, unsigned bit) {
    if (status) atomicOr(status, bit);
}

// Sequence that holds row t: the last b with q_start[b] <= t, or -1 when t
// lies before the first or behind the last sequence.  All 32 lanes take part
// (each step narrows the range 32 times); any content of q_start keeps every
// access inside its B + 1 words.
__device__ __forceinline__ int kv_find_seq(const KvBatch& b, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = b.B;
    while (n > 1) {
        const int step = (n + 31) >> 5;
        const int at = lane * step;
        const bool le = at < n && __ldg(b.q_start + lo + at) <= t;
        const unsigned m = __ballot_sync(0xffffffffu, le);
        if (!m) return -1;
        const int top = (31 - __clz(m)) * step;
        lo += top;
        n = n - top < step ? n - top : step;
    }
    return (__ldg(b.q_start + lo) <= t && t < __ldg(b.q_start + lo + 1)) ? lo : -1;
}

// Page id of a logical page of a sequence, or -1 (and a status bit) when it
// lies outside the table or the cache.
__device__ __forceinline__ int kv_page(const KvBatch& b, const KvCache& c, int seq, int page,
                                       unsigned* status) {
    if (page >= b.max_pages) {
        kv_flag(status, KV_BAD_LENGTH);
        return -1;
    }
    const int id = b.table ? __ldg(b.table + (int64_t)seq * b.table_stride + page)
                           : seq * b.max_pages + page;
    if (id < 0 || id >= c.pages) {
        kv_flag(status, KV_BAD_PAGE);
        return -1;
    }
    return id;
}

// Two multiply-adds, two additions in one issue slot, for loops that have no
// other to spare (the softmax warps of a chunk: 3% of its time; quantising).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
          "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}

template <typename T> __device__ __forceinline__ float kv_to_f(T v);
template <> __device__ __forceinline__ float kv_to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float kv_to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float kv_to_f<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <typename T> __device__ __forceinline__ T kv_from_f(float v);
template <> __device__ __forceinline__ float kv_from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half kv_from_f<__half>(float v) {
    return __float2half_rn(v);
}
template <> __device__ __forceinline__ __nv_bfloat16 kv_from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

}  // namespace moeb200
