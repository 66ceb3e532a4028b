// kv_cache.cu -- writing new keys and values into the pages of a key/value
// cache (16-bit, or quantised to Q8_0 on the way) and reading rows back.
//
// Row i of sequence b stands at position p = kv_len - q_len + i, in row
// p % page_size of page table[b][p / page_size].  Q8_0, per 32 values:
//   d = max|x| / 127 rounded up to binary16 (at most 515.5), code = rint(x / d)
// so |x - d * code| <= d / 2: a scale rounded to nearest could fall below
// max|x| / 127 and push the largest value past code 127.  A block that holds
// a NaN or an infinity gets a NaN scale and reads back as NaN.
//
// Both kernels move each value once: bound by HBM.  A thread owns 16 values
// of a head (two 16-byte loads of a 16-bit row, one 16-byte store of codes),
// two threads own a Q8_0 block.  A CTA looks up the slots of its up to 32
// tokens, one lane per token, then all its threads walk the units of those
// tokens, keys and values in the same iteration so that both loads are in
// flight.  Measured, 105k tokens x 8 heads x 128: write as Q8_0 127 us (5.2
// TB/s), read back as bfloat16 121 us (5.5 TB/s).  Issue slots are the next
// bound: with a division per unit, single fp32 operations and conversions of
// the codes, 138 us and 125 us; with stores that pass the caches, 129 us and
// 123 us.
#include <type_traits>

#include "kv.cuh"
#include "launch.h"

namespace moeb200 {

namespace {

constexpr int kKvThreads = 256;
constexpr int kKvMaxTokens = 32;   // tokens per CTA at most: one per lane

struct KvRows {
    void* k;
    void* v;
    int64_t k_ts, k_hs, v_ts, v_hs;   // strides in elements
};

template <typename T> struct alignas(16) Vec16 {
    T v[16];
};

template <typename T>
__device__ __forceinline__ void load16(Vec16<T>& d, const T* p) {
    const uint4* s = reinterpret_cast<const uint4*>(p);
    uint4* r = reinterpret_cast<uint4*>(d.v);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) r[i] = __ldcs(s + i);
}

template <typename T>
__device__ __forceinline__ void store16(T* p, const Vec16<T>& d) {
    uint4* s = reinterpret_cast<uint4*>(p);
    const uint4* r = reinterpret_cast<const uint4*>(d.v);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) s[i] = r[i];
}

// Bits of the largest magnitude of 16 values, as an fp32 pattern: patterns of
// magnitudes order like integers, infinities and NaN above all others.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Vec16<T>& x) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(x.v);
    if constexpr (sizeof(T) == 4) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, w[i] & 0x7fffffffu);
        return top;
    } else {
        uint32_t pair = w[0] & 0x7fff7fffu;
#pragma unroll
        for (int i = 1; i < 8; ++i) pair = __vmaxu2(pair, w[i] & 0x7fff7fffu);
        const unsigned short h = (unsigned short)max(pair & 0xffffu, pair >> 16);
        if constexpr (std::is_same<T, __half>::value)
            return __float_as_uint(__half2float(__ushort_as_half(h))) & 0x7fffffffu;
        return (uint32_t)h << 16;
    }
}

// One thread's half of a Q8_0 block: codes of its 16 values and the block's
// scale (the other half sits in the neighbouring lane; the whole warp must call).
template <typename T>
__device__ __forceinline__ __half quantise16(const Vec16<T>& x, Vec16<int8_t>& q) {
    uint32_t top = top_bits(x);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    if (top >= 0x7f800000u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) q.v[i] = 0;
        return __ushort_as_half(0x7fff);
    }
    const float want = __half2float(__float2half_ru(__fdiv_rn(__uint_as_float(top), 127.f)));
    const float step = fminf(want, kKvScaleMax);
    const float inv = step > 0.f ? __frcp_rn(step) : 0.f;
    const float2 inv2 = make_float2(inv, inv), minus = make_float2(-step, -step);
    const float2 whole = make_float2(12582912.f, 12582912.f), none = make_float2(0.f, 0.f);
    uint32_t* out = reinterpret_cast<uint32_t*>(q.v);
    auto codes = [&](auto clamp) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t n[4];
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                // x / step: x times the reciprocal, and one step of Newton's
                // correction, whose remainder the fused multiply-add gives
                // exactly: off by 2^-46 before its rounding, so ties stay ties
                const float2 f = make_float2(kv_to_f<T>(x.v[4 * w + i]),
                                             kv_to_f<T>(x.v[4 * w + i + 1]));
                const float2 y = fma2(f, inv2, none);
                float2 c = fma2(fma2(y, minus, f), inv2, y);
                if constexpr (decltype(clamp)::value) {
                    c.x = fminf(fmaxf(c.x, -127.f), 127.f);
                    c.y = fminf(fmaxf(c.y, -127.f), 127.f);
                }
                // nearest integer, ties to even: 1.5 * 2^23 leaves no fraction bits
                c = add2(c, whole);
                n[i] = __float_as_uint(c.x);
                n[i + 1] = __float_as_uint(c.y);
            }
            out[w] = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040),
                                 0x5410);
        }
    };
    if (want > kKvScaleMax) codes(std::true_type{});   // |x / step| <= 127 otherwise
    else codes(std::false_type{});
    return __float2half_rn(step);
}

// A thread's units of 16 values among a CTA's tokens, kKvThreads apart: token i,
// head h, values from d on; stepped by carries, without a division.
struct KvUnit {
    int i, h, d;           // d in units of 16
    int di, dh, dd;
    __device__ __forceinline__ KvUnit(int u, int per_head, int heads) {
        const int per_token = per_head * heads;
        auto split = [&](int n, int& a, int& b, int& c) {
            a = n / per_token;
            b = (n - a * per_token) / per_head;
            c = n - a * per_token - b * per_head;
        };
        split(u, i, h, d);
        split(kKvThreads, di, dh, dd);
    }
    __device__ __forceinline__ void next(int per_head, int heads) {
        d += dd;
        const int up = d >= per_head;
        d -= up ? per_head : 0;
        h += dh + up;
        const int over = h >= heads;
        h -= over ? heads : 0;
        i += di + over;
    }
};

// Slot (page * heads * page_size + row, in rows of one head; -1: none, -2:
// behind the last sequence) of the CTA's tokens: the first warp searches the
// first token's sequence, and each lane goes on from there for its own token.
// The other threads wait at the caller's barrier.
__device__ __forceinline__ void cta_slots(const KvBatch& b, const KvCache& c, int t0, int n,
                                          int64_t* slots, unsigned* status) {
    const int lane = threadIdx.x & 31;
    if (threadIdx.x >= 32) return;
    int s = kv_find_seq(b, t0);
    const int t = t0 + lane;
    if (lane >= n) return;
    // s = -1: before the first sequence (a malformed q_start), or behind the last
    int lo = s < 0 ? 0 : s, hi = b.B;
    if (s < 0 || t >= __ldg(b.q_start + s + 1)) {   // the last b with q_start[b] <= t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(b.q_start + mid) <= t) lo = mid; else hi = mid;
        }
        s = lo;
    }
    const int q0 = __ldg(b.q_start + s), q1 = __ldg(b.q_start + s + 1);
    int64_t slot = -2;
    if (q0 <= t && t < q1) {
        slot = -1;
        const int pos = max(__ldg(b.kv_lens + s), 0) - q1 + t;
        if (pos >= 0) {
            const int page = kv_page(b, c, s, pos >> c.page_shift, status);
            if (page >= 0)
                slot = ((int64_t)page * c.heads << c.page_shift) + (pos & (c.page_size - 1));
        }
    }
    slots[lane] = slot;
}

// TI: type of the rows, TC: type of the cache (int8_t: Q8_0).
template <typename TI, typename TC>
__global__ void __launch_bounds__(kKvThreads, sizeof(TI) == 4 ? 2 : 4)
k_kv_write(KvBatch b, KvCache c, KvRows in, int tokens, unsigned* status) {
    __shared__ int64_t slots[kKvMaxTokens];
    const int t0 = blockIdx.x * tokens;
    const int n = b.T - t0 < tokens ? b.T - t0 : tokens;
    const int per_head = c.dim >> 4;
    const int units = n * per_head * c.heads;
    // a unit's rows are loaded while the one before it is stored, the first
    // while the slots are looked up
    Vec16<TI> x[2] = {};
    KvUnit at(threadIdx.x, per_head, c.heads);
    auto load = [&] {
        const int h = at.h, d = at.d << 4;
        load16(x[0], static_cast<const TI*>(in.k) + (t0 + at.i) * in.k_ts + h * in.k_hs + d);
        load16(x[1], static_cast<const TI*>(in.v) + (t0 + at.i) * in.v_ts + h * in.v_hs + d);
    };
    int u = threadIdx.x;
    if (u < units) load();
    cta_slots(b, c, t0, n, slots, status);
    __syncthreads();
    for (; (u & ~31) < units; u += kKvThreads) {   // whole warps: two lanes share a block
        const int64_t slot = u < units ? slots[at.i] : -1;
        const int64_t row = slot + ((int64_t)at.h << c.page_shift);
        const int d = at.d << 4;
        const Vec16<TI> y0 = x[0], y1 = x[1];
        at.next(per_head, c.heads);
        if (u + kKvThreads < units) load();
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const Vec16<TI>& v = w ? y1 : y0;
            Vec16<TC> y;
            if constexpr (sizeof(TC) == 1) {
                const __half s = quantise16(v, y);
                if (slot >= 0 && !(d & 16)) (w ? c.vs : c.ks)[row * (c.dim >> 5) + (d >> 5)] = s;
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) y.v[j] = kv_from_f<TC>(kv_to_f<TI>(v.v[j]));
            }
            if (slot >= 0) store16(static_cast<TC*>(w ? c.v : c.k) + row * c.dim + d, y);
        }
    }
}

// Rows whose position is negative, or whose page is refused, read as zeros.
template <typename TO, typename TC>
__global__ void __launch_bounds__(kKvThreads)
k_kv_read(KvBatch b, KvCache c, KvRows out, int tokens, unsigned* status) {
    __shared__ int64_t slots[kKvMaxTokens];
    const int t0 = blockIdx.x * tokens;
    const int n = b.T - t0 < tokens ? b.T - t0 : tokens;
    cta_slots(b, c, t0, n, slots, status);
    __syncthreads();
    const int per_head = c.dim >> 4;
    const int units = n * per_head * c.heads;
    KvUnit at(threadIdx.x, per_head, c.heads);
#pragma unroll 2
    for (int u = threadIdx.x; u < units; u += kKvThreads, at.next(per_head, c.heads)) {
        const int i = at.i, h = at.h, d = at.d << 4;
        const int64_t slot = slots[i];
        if (slot == -2) continue;   // behind the last sequence: left as it is
        const int64_t row = slot + ((int64_t)h << c.page_shift);
        Vec16<TC> x[2];
        float s[2] = {0.f, 0.f};
        if (slot >= 0) {
            load16(x[0], static_cast<const TC*>(c.k) + row * c.dim + d);
            load16(x[1], static_cast<const TC*>(c.v) + row * c.dim + d);
            if constexpr (sizeof(TC) == 1) {
                s[0] = __half2float(c.ks[row * (c.dim >> 5) + (d >> 5)]);
                s[1] = __half2float(c.vs[row * (c.dim >> 5) + (d >> 5)]);
            }
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            Vec16<TO> y{};
            if (slot >= 0) {
                if constexpr (sizeof(TC) == 1) {
                    // a code as fp32: 2^23 + 128 + code by a byte permute, less
                    // 2^23 + 128 (a conversion runs at a quarter of their rate)
                    const uint32_t* q = reinterpret_cast<const uint32_t*>(x[w].v);
                    const float2 off = make_float2(-8388736.f, -8388736.f);
                    const float2 s2 = make_float2(s[w], s[w]), none = make_float2(0.f, 0.f);
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const uint32_t p = q[j / 4] ^ 0x80808080u;
                        float2 f;
                        f.x = __uint_as_float(__byte_perm(p, 0x4b000000u, 0x7440 + j % 4));
                        f.y = __uint_as_float(__byte_perm(p, 0x4b000000u, 0x7441 + j % 4));
                        f = fma2(add2(f, off), s2, none);
                        y.v[j] = kv_from_f<TO>(f.x);
                        y.v[j + 1] = kv_from_f<TO>(f.y);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) y.v[j] = kv_from_f<TO>(kv_to_f<TC>(x[w].v[j]));
                }
            }
            TO* p = w ? static_cast<TO*>(out.v) + (t0 + i) * out.v_ts + h * out.v_hs + d
                      : static_cast<TO*>(out.k) + (t0 + i) * out.k_ts + h * out.k_hs + d;
            store16(p, y);
        }
    }
}

// Tokens per CTA: as many as leave four CTAs per SM, so that small calls
// spread over the GPU and large ones look several slots up at once.
int tokens_per_cta(int T) {
    int n = T / (4 * sm_count());
    return n < 1 ? 1 : n > kKvMaxTokens ? kKvMaxTokens : n;
}

template <bool WRITE, typename A, typename B>
cudaError_t launch_rows(const KvBatch& b, const KvCache& c, const KvRows& r, unsigned* status,
                        cudaStream_t s) {
    const int n = tokens_per_cta(b.T);
    const int grid = (b.T - 1) / n + 1;   // up to 2^31 - 1 rows
    if constexpr (WRITE)
        k_kv_write<A, B><<<grid, kKvThreads, 0, s>>>(b, c, r, n, status);
    else
        k_kv_read<A, B><<<grid, kKvThreads, 0, s>>>(b, c, r, n, status);
    return cudaGetLastError();
}

template <bool WRITE, typename A>
cudaError_t launch_cache(const KvBatch& b, const KvCache& c, const KvRows& r, unsigned* status,
                         cudaStream_t s) {
    if (c.type == KV_F16) return launch_rows<WRITE, A, __half>(b, c, r, status, s);
    if (c.type == KV_BF16) return launch_rows<WRITE, A, __nv_bfloat16>(b, c, r, status, s);
    return launch_rows<WRITE, A, int8_t>(b, c, r, status, s);
}

}  // namespace

cudaError_t launch_kv_rows(bool write, const KvBatch& b, const KvCache& c, int type, void* k,
                           int64_t k_ts, int64_t k_hs, void* v, int64_t v_ts, int64_t v_hs,
                           unsigned* status, cudaStream_t s) {
    const KvRows r{k, v, k_ts, k_hs, v_ts, v_hs};
    if (write) {
        if (type == KV_F32) return launch_cache<true, float>(b, c, r, status, s);
        if (type == KV_F16) return launch_cache<true, __half>(b, c, r, status, s);
        return launch_cache<true, __nv_bfloat16>(b, c, r, status, s);
    }
    if (type == KV_F32) return launch_cache<false, float>(b, c, r, status, s);
    if (type == KV_F16) return launch_cache<false, __half>(b, c, r, status, s);
    return launch_cache<false, __nv_bfloat16>(b, c, r, status, s);
}

}  // namespace moeb200
