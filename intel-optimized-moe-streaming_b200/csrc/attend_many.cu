// attend_many.cu -- attention of chunks of new rows over a paged cache on
// tcgen05.
//
// 4 D operations per (row, key, head) against 2 D values read per key of a
// whole tile: bound by the tensor cores, and next to them by the exponentials
// (128 x 128 scores take 1043 cycles of an SM's special function units, the
// two products of a 128-value head 1024 cycles of its tensor core).
//
// A CTA (one per SM) holds the query tile of a group's rows -- two of 128 rows
// for head dimensions up to 128, one above -- and walks units of 128 keys.
// Tensor memory has the two score tiles S (128 columns each) and the output
// sums O (2 x DP columns, or 256); the probabilities overwrite their scores as
// 16-bit values, 64 keys at a time, and are the value product's A operand from
// there.
//   warps 0-7   softmax: a thread owns a row (one of two tiles; or, with one
//               tile, half the columns of a row, the two halves agreeing on
//               the maximum through shared memory).  The maximum in use is
//               only replaced when it grows by more than 2^8, so O is rarely
//               rescaled; the same threads do that, load the queries, and
//               divide and store the rows at a tile's end.
//   warp 8      copies: a ring of NST stages of up to 32 KB (keys x 64-value
//               slabs, 128-byte swizzle) filled by tensor copies, one lane per
//               page piece and slab
//   warp 9      issues all products: with two tiles S_t(j + 1) follows the
//               value product of tile t, so that a tile's softmax runs under
//               the other tile's products; with one tile there are two score
//               buffers and S(j + 1) comes before the value product of j
//   warps 10-11 look through the values of units that not all rows attend
//   warps 12-15 (Q8_0) instead of the copies: codes are loaded a stage ahead
//               into registers, become binary16 and go to the ring
// Measured (1965 MHz at the start, power-capped below it later): 2048 rows
// over 8k keys, 32/8 heads x 128, 230 us = 1047 TFLOP/s, 3550 cycles a unit of
// two tiles: 470 maximum, 1690 exponentials (1400 alone: the tiles' phases
// meet), 200 hand-over, 1190 until the next scores, which wait for the last
// half of the value product because P stands on S.  4096 rows over 16k keys,
// 16/2 heads x 256, 920 us = 1046 TFLOP/s, 3300 cycles a unit: 128 KB of keys
// and values through the ring per unit and SM, 8.4 TB/s out of L2 in all.
#include "attend_mma.cuh"
#include "launch.h"

namespace moeb200 {

namespace {

constexpr int kManyKeys = 128;               // keys of a unit
constexpr int kManyCost = 2;                 // starting and ending a tile, in units
constexpr uint32_t kManyPolls = 1u << 21;
constexpr float kManyGrow = 8.f;             // log 2 of the growth that replaces the maximum

template <int DP, int KIND>
struct Many {
    static constexpr bool Q8 = KIND == KIND_Q8;
    static constexpr int NQ = DP > 128 ? 1 : 2;          // query tiles of 128 rows
    static constexpr int M = 128 * NQ;
    static constexpr int SLABS = DP / 64;
    static constexpr int KPARTS = DP > 128 ? 2 : 1;      // stages of a unit's keys, and values
    static constexpr int KSLABS = SLABS / KPARTS;        // slabs of a stage of keys (by dimension)
    static constexpr int VKEYS = kManyKeys / KPARTS;     // keys of a stage of values
    static constexpr int STAGEB = KSLABS * kManyKeys * 128;
    static constexpr int QB = NQ * SLABS * 128 * 128;
    static constexpr int NST = DP == 64 ? 8 : 5;
    static constexpr int OC = NQ == 2 ? DP : DP / 2;     // output columns of a thread
    static constexpr int THREADS = Q8 ? 512 : 384;
    // binary16 probabilities: 2^7 of the maximum in use, at most 2^15.  The
    // maximum and what is taken off the scores are rounded up, so that this holds
    // for large scores too, whose neighbours in fp32 lie far apart (at 2^25, 4).
    static constexpr float SHIFT = KIND == KIND_BF16 ? 0.f : 7.f;
    static constexpr int o_stage = QB;
    static constexpr int o_bar = QB + NST * STAGEB;
    static constexpr int o_fac = o_bar + 512;            // row factors
    static constexpr int o_max = o_fac + M * 4;          // maxima and sums of half rows
    static constexpr int smem = o_max + (NQ == 1 ? 2048 : 0);
    static_assert(smem <= 232448, "shared memory of a CTA");
    static constexpr uint32_t IDESC_S = umma_idesc_f16(128, kManyKeys) |
                                        (KIND == KIND_BF16 ? (1u << 7) | (1u << 10) : 0u);
    static constexpr uint32_t IDESC_O = umma_idesc_f16(128, DP) | (1u << 16) |   // B: N-major
                                        (KIND == KIND_BF16 ? (1u << 7) | (1u << 10) : 0u);
};

struct ManyBars {
    uint64_t full[8], empty[8], s_full[2], p_full[2][2], pv_done[2], q_full[2];
    uint32_t tmem, lost;
    uint32_t products;     // units whose value products have been issued
    uint32_t checked[2];   // partly attended units that each checking warp is done with
    uint32_t odd[8][4];    // such units in turn: keys whose values are not all finite
};
static_assert(sizeof(ManyBars) <= 512, "");

// D (+)= A . B with A in tensor memory.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                            uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 1, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc)
        : "memory");
}

// Descriptor of an N-major SWIZZLE_128B operand (values: 64 dimensions of a
// key are 128 contiguous bytes): 8-key atoms 1024 bytes apart along K, slabs
// of 64 dimensions `slab` bytes apart along N.
__device__ __forceinline__ uint64_t umma_desc_nmajor(uint32_t saddr, uint32_t slab) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(slab >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void shfl_swap(uint4& keep, uint4& give, int mask, bool upper) {
    // the lane with the bit clear gives `give` and takes the partner's `keep`
    uint32_t* k = reinterpret_cast<uint32_t*>(&keep);
    uint32_t* g = reinterpret_cast<uint32_t*>(&give);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t out = upper ? k[e] : g[e];
        const uint32_t in = __shfl_xor_sync(0xffffffffu, out, mask);
        if (upper) k[e] = in; else g[e] = in;
    }
}

// y[i] of lane q of a quad becomes y[q] of lane i.
__device__ __forceinline__ void quad_transpose(uint4 (&y)[4], int lane) {
    shfl_swap(y[0], y[2], 2, lane & 2);
    shfl_swap(y[1], y[3], 2, lane & 2);
    shfl_swap(y[0], y[1], 1, lane & 1);
    shfl_swap(y[2], y[3], 1, lane & 1);
}

template <int ID, int N>
__device__ __forceinline__ void bar_sync() {
    asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
}

template <int N>
__device__ __forceinline__ void bar_sync(int id) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(valid ? 16 : 0)
                 : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(e));
    return e != 0;
}

// A value that all lanes hold, marked as such for the compiler.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

// One role's walk over the segments (stretch of one tile) of its CTA.
template <int DP, int KIND>
struct Walk {
    AttendCursor cur;
    AttendSeq s;
    int u0, take;
    int64_t used;
    bool begins, ends;
    __device__ bool open(const AttendArgs& a) {   // the current segment's units
        if (cur.left <= 0) return false;
        const AttendPart p = attend_part<Many<DP, KIND>::M, kManyKeys, kManyCost>(a, cur, s);
        u0 = p.u0;
        take = p.take;
        used = p.used;
        begins = p.begins;
        ends = p.ends;
        return take > 0;   // 0: the stretch ends before the tile's first unit
    }
    __device__ void next(const AttendArgs& a) {
        cur.left -= used;
        if (cur.left > 0) attend_next<Many<DP, KIND>::M>(a, cur, s);
    }
};

// Stage of the ring, counted over the segment: two tiles take keys and values
// in turn; one tile takes the keys of j + 1 before the values of j.
template <int NQ>
__device__ __forceinline__ int stage_k(int j) {
    return NQ == 2 ? 2 * j : j == 0 ? 0 : 4 * j - 2;
}
template <int NQ>
__device__ __forceinline__ int stage_v(int j, int take) {
    return NQ == 2 ? 2 * j + 1 : j + 1 < take ? 4 * j + 4 : 4 * j + 2;
}

// Queries of this warp's rows of a tile into the swizzled operand layout.
// TQ values are copied as they are (cp.async); or, for bfloat16 over Q8_0 values and
// for negative scales, through registers: scaled to binary16, sign flipped.
template <int DP, int KIND, typename TQ>
struct QueryRows {
    using F = Many<DP, KIND>;
    static constexpr bool CONVERT = KIND != KIND_BF16 && std::is_same<TQ, __nv_bfloat16>::value;
    static constexpr int LPR = DP / 8;        // lanes of a row, 16 bytes each
    static constexpr int RPI = 32 / LPR;      // rows of an iteration
    static constexpr int BATCH = 4;

    // rows [0, n) relative to row0 of the tile; the warp takes 32 / split rows
    __device__ static void load(const AttendArgs& a, const Walk<DP, KIND>& w, int row0, int n_rows,
                                unsigned char* tile, float* fac, int valid) {
        const int lane = threadIdx.x & 31;
        const int ch = lane % LPR, sub = lane / LPR;
        const bool in_dim = ch * 8 < a.c.dim;
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
        const bool copy = !CONVERT && flip == 0;
        // lane i: where row row0 + i of the tile starts
        const int mine = w.cur.tile * F::M + row0 + lane;
        const int tok = a.by_group.div(mine);
        const int64_t start = (int64_t)(w.s.q0 + tok) * a.q_ts +
                              (int64_t)(w.cur.kvh * a.group + mine - tok * a.group) * a.q_hs;
        for (int i0 = 0; i0 < n_rows; i0 += RPI * BATCH) {
            uint4 x[BATCH];
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int i = i0 + b * RPI + sub, r = row0 + i;
                const bool ok = in_dim && r < valid;
                const int64_t at = __shfl_sync(0xffffffffu, start, i);
                const TQ* q = static_cast<const TQ*>(a.q) + (ok ? at + ch * 8 : 0);
                if (copy) {
                    const int t = r & 127;
                    cp_async16(smem_u32(tile + (r >> 7) * (F::SLABS * 16384) + (ch >> 3) * 16384) +
                                   sw128_offset(t, ch & 7), q, ok);
                } else {
                    x[b] = make_uint4(0, 0, 0, 0);
                    if (ok) x[b] = __ldg(reinterpret_cast<const uint4*>(q));
                }
            }
            if (copy) continue;
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int r = row0 + i0 + b * RPI + sub, t = r & 127;
                uint32_t* w32 = reinterpret_cast<uint32_t*>(&x[b]);
                if constexpr (CONVERT) {
                    float v[8], top = 0.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[2 * i] = __uint_as_float(w32[i] << 16);
                        v[2 * i + 1] = __uint_as_float(w32[i] & 0xffff0000u);
                        top = fmaxf(top, fmaxf(fabsf(v[2 * i]), fabsf(v[2 * i + 1])));
                    }
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1)
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const float f = row_factor(top);
                    if (ch == 0) fac[r] = f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) w32[i] = pack16<KIND_F16>(v[2 * i] * f, v[2 * i + 1] * f);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) w32[i] ^= flip;
                *reinterpret_cast<uint4*>(tile + (r >> 7) * (F::SLABS * 16384) + (ch >> 3) * 16384 +
                                          sw128_offset(t, ch & 7)) = x[b];
            }
        }
    }
};

template <int DP, int KIND, typename TQ>
__global__ void __launch_bounds__(Many<DP, KIND>::THREADS, 1)
k_attend_many(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
              const __grid_constant__ AttendArgs a, void* wsp) {
    using F = Many<DP, KIND>;
    extern __shared__ __align__(1024) unsigned char smem_many[];
    unsigned char* sm = smem_many;
    ManyBars* bars = reinterpret_cast<ManyBars*>(sm + F::o_bar);
    float* fac = reinterpret_cast<float*>(sm + F::o_fac);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < F::NST; ++i) {
            mbar_init(&bars->full[i], F::Q8 ? 4 : 1);
            mbar_init(&bars->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars->s_full[i], 1);
            for (int h = 0; h < 2; ++h) mbar_init(&bars->p_full[i][h], 4);
            mbar_init(&bars->pv_done[i], 1);
            mbar_init(&bars->q_full[i], F::NQ == 2 ? 4 : 8);
        }
        bars->lost = 0;
        bars->products = bars->checked[0] = bars->checked[1] = 0;
        for (int i = 0; i < 32; ++i) bars->odd[i / 4][i % 4] = 0;
        mbar_fence_init();
    }
    if (warp == 9) tmem_alloc(&bars->tmem, 512);
    const int ctas = gridDim.x;
    AttendWs ws(wsp, ctas);
    Walk<DP, KIND> w;
    w.cur = attend_place<F::M, kManyKeys, kManyCost, kManyCost + 1, F::THREADS>(
        a, *reinterpret_cast<AttendScratch*>(sm), blockIdx.x, ctas, a.status);
    fence_async_smem();   // the scratch lies where the queries go
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars->tmem);
    if (w.cur.left > 0) w.s = attend_seq(a, w.cur.seq, nullptr);

    bool lost = false;
    auto await = [&](uint64_t* bar, uint32_t parity) {
        if (!mbar_wait(bar, parity & 1u, lost ? 64u : kManyPolls)) {
            lost = true;
            *reinterpret_cast<volatile uint32_t*>(&bars->lost) = 1;
        }
    };

    // waits until a counter in shared memory reaches `upto`
    auto spin = [&](const uint32_t* word, uint32_t upto) {
        for (uint32_t i = 0; (int)(*reinterpret_cast<const volatile uint32_t*>(word) - upto) < 0; ++i)
            if (i >= (lost ? 64u : kManyPolls * 8)) {
                lost = true;
                *reinterpret_cast<volatile uint32_t*>(&bars->lost) = 1;
                break;
            }
        __threadfence_block();
    };

    if (warp < 8) {
        // ------------------------------------------------------------ softmax
        const int wg = warp >> 2, quarter = warp & 3;
        const int row = quarter * 32 + lane;                       // of the 128-row tile
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;     // TMEM lane offset
        const int trow = F::NQ == 2 ? wg * 128 + row : row;        // of the CTA's rows
        const uint32_t t_o = tmem + lanes + 256 + (F::NQ == 2 ? wg * DP : wg * 128);
        const int q0 = F::NQ == 2 ? wg * 128 + quarter * 32 : quarter * 32 + wg * 16;
        constexpr int QN = F::NQ == 2 ? 32 : 16;                   // query rows the warp loads
        const int tw = F::NQ == 2 ? wg : 0;                        // query tile
        float* xmax = reinterpret_cast<float*>(sm + F::o_max);     // [2][2][128]
        AttendRecord rec{};
        uint32_t it = 0;       // units done by the CTA
        uint32_t partial = 0;  // of them, those that not all rows attend
        int stage0 = 0;        // ring stages before this segment

        auto load_queries = [&](int n_valid) {
            QueryRows<DP, KIND, TQ>::load(a, w, q0, QN, sm, fac, n_valid);
        };
        auto hand_queries = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->q_full[F::NQ == 2 ? wg : 0]);
        };
        // The unit's odd values: all eight warps meet here.
        auto poisoned = [&](volatile uint32_t* odd, int j, uint32_t t_s, int key0, int lo, int hi) {
            unsigned char* st[F::KPARTS];
#pragma unroll
            for (int h = 0; h < F::KPARTS; ++h) {
                const int n = stage0 + stage_v<F::NQ>(j, w.take) + h;
                st[h] = sm + F::o_stage + (n % F::NST) * F::STAGEB;
                await(&bars->full[n % F::NST], (uint32_t)(n / F::NST));
            }
            tc_fence_before();
            bar_sync<2, 256>();   // with one tile, O takes both halves' probabilities
            tc_fence_after();
            if (j > 0) {
                await(&bars->pv_done[tw], it - 1);
                tc_fence_after();
            }
#pragma unroll 1
            for (int k = 0; k < kManyKeys; ++k) {
                if (!((odd[k >> 5] >> (k & 31)) & 1)) continue;
                const uint32_t pw = tmem_ld1(t_s + (k >> 6) * 64 + (k & 63) / 2);
                tmem_wait_ld();
                const uint16_t p16 = (uint16_t)(k & 1 ? pw >> 16 : pw);
                const float p = KIND == KIND_BF16 ? __bfloat162float(__ushort_as_bfloat16(p16))
                                                  : __half2float(__ushort_as_half(p16));
                const bool at = key0 + k >= lo && key0 + k < hi;
                const unsigned char* vt = st[k / F::VKEYS];
                const int kr = k % F::VKEYS;
#pragma unroll 1
                for (int c = 0; c < F::OC / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16(t_o + c * 16, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int d = (F::NQ == 1 ? wg * 128 : 0) + c * 16 + e;
                        const uint16_t v16 = *reinterpret_cast<const uint16_t*>(
                            vt + (d >> 6) * (F::VKEYS * 128) + sw128_offset(kr, (d >> 3) & 7) +
                            (d & 7) * 2);
                        if (at && odd16<KIND>(v16))
                            o[e] = __float_as_uint(
                                __uint_as_float(o[e]) +
                                p * (KIND == KIND_BF16 ? __bfloat162float(__ushort_as_bfloat16(v16))
                                                       : __half2float(__ushort_as_half(v16))));
                    }
                    __syncwarp();
                    tmem_st16(t_o + c * 16, o);
                }
                tmem_wait_st();
            }
            tc_fence_before();
            bar_sync<2, 256>();
#pragma unroll
            for (int h = 0; h < F::KPARTS; ++h)
                for (int i = tid; i < F::STAGEB / 2; i += 256) {
                    uint16_t* v = reinterpret_cast<uint16_t*>(st[h]) + i;
                    if (odd16<KIND>(*v)) *v = 0;
                }
            if (tid < 4) odd[tid] = 0;
            fence_async_smem();
            bar_sync<2, 256>();
        };
        bool more = w.open(a);
        if (more) {
            load_queries(w.s.n * a.group - w.cur.tile * F::M);
            hand_queries();
        }
        while (more) {
            const AttendSeq s = w.s;
            const AttendCursor cur = w.cur;
            const int u0 = w.u0, take = w.take;
            const bool begins = w.begins, ends = w.ends;
            const int rows = s.n * a.group - cur.tile * F::M;   // valid rows: the first `rows`
            // keys that all rows of the CTA attend, all rows of this warp, and this row
            const AttendTile tile = attend_tile(a, s, cur.tile * F::M, F::M);
            int lo = 0, hi = 0;
            if (trow < rows)
                attend_range(s.first + a.by_group.div(cur.tile * F::M + trow), s.len, a.causal,
                             a.window, lo, hi);
            int warp_lo = trow < rows ? lo : 0, warp_hi = trow < rows ? hi : 0x7fffffff;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                warp_lo = max(warp_lo, __shfl_xor_sync(0xffffffffu, warp_lo, o));
                warp_hi = min(warp_hi, __shfl_xor_sync(0xffffffffu, warp_hi, o));
            }
            float m = -INFINITY, l = 0.f;   // what is taken off the scores (the
                                            // maximum in use less SHIFT); their sum
            float mul = 0.f;
            {   // O starts from zeros
                uint32_t z[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) z[i] = 0;
#pragma unroll
                for (int c = 0; c < F::OC / 32; ++c) tmem_st32(t_o + c * 32, z);
                tmem_wait_st();
                tc_fence_before();   // with one tile, the maximum's barrier follows
            }
#pragma unroll 1
            for (int j = 0; j < take; ++j, ++it) {
                const int buf = F::NQ == 2 ? wg : (int)(it & 1);
                const uint32_t ph = F::NQ == 2 ? it : it >> 1;
                const uint32_t t_s = tmem + lanes + buf * 128;
                await(&bars->s_full[buf], ph);
                tc_fence_after();
                if (j == 0) {
                    float f = 1.f;
                    if constexpr (QueryRows<DP, KIND, TQ>::CONVERT) f = fac[trow];
                    mul = score_factor(a.scale, f);
                }
                const int key0 = (u0 + j) * kManyKeys;
                const bool whole = key0 >= tile.all_lo && key0 + kManyKeys <= tile.all_hi;
                const bool masked = key0 < warp_lo || key0 + kManyKeys > warp_hi;
                // 32 score columns; those the row does not attend to -infinity
                auto mask = [&](uint32_t* v, int col) {
                    const int f = min(max(lo - key0 - col, 0), 32);
                    const int t = min(max(hi - key0 - col, 0), 32);
                    const uint32_t keep = (uint32_t)(((1ull << t) - 1) & ~((1ull << f) - 1));
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!(keep >> i & 1)) v[i] = 0xff800000u;
                };
                float t0 = -INFINITY, t1 = t0, t2 = t0, t3 = t0;
                auto highest = [&](const uint32_t* v) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        t0 = fmaxf(fmaxf(t0, __uint_as_float(v[i])), __uint_as_float(v[i + 1]));
                        t1 = fmaxf(fmaxf(t1, __uint_as_float(v[i + 2])), __uint_as_float(v[i + 3]));
                        t2 = fmaxf(fmaxf(t2, __uint_as_float(v[i + 4])), __uint_as_float(v[i + 5]));
                        t3 = fmaxf(fmaxf(t3, __uint_as_float(v[i + 6])), __uint_as_float(v[i + 7]));
                    }
                };
                // A thread of the two-tile form reads its 128 scores in two
                // halves of 64 and, having the maximum, takes the second half
                // from registers and the first one from tensor memory again.
                uint32_t va[32], vb[32];
                if constexpr (F::NQ == 2) {
                    tmem_ld32(t_s, va);
                    tmem_ld32(t_s + 32, vb);
                    tmem_wait_ld();
                    if (masked) {
                        mask(va, 0);
                        mask(vb, 32);
                    }
                    highest(va);
                    highest(vb);
                }
                const int last = F::NQ == 2 ? 64 : wg * 64;
                tmem_ld32(t_s + last, va);
                tmem_ld32(t_s + last + 32, vb);
                tmem_wait_ld();
                if (masked) {
                    mask(va, last);
                    mask(vb, last + 32);
                }
                highest(va);
                highest(vb);
                float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
                top = __fadd_ru(__fmul_ru(top, mul), -F::SHIFT);
                if constexpr (F::NQ == 1) {
                    float* xm = xmax + (it & 1) * 256;
                    xm[wg * 128 + row] = top;
                    bar_sync<1, 256>();
                    top = fmaxf(top, xm[(wg ^ 1) * 128 + row]);
                }
                const bool grow = top > __fadd_rd(m, kManyGrow) || (m == -INFINITY && top > m);
                if (__any_sync(0xffffffffu, grow && j > 0)) {
                    const float f = grow ? ex2(m - top) : 1.f;
                    l *= f;
                    await(&bars->pv_done[tw], it - 1);
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < F::OC / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld16(t_o + c * 16, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st16(t_o + c * 16, o);
                    }
                    tmem_wait_st();
                    // With one tile the value product of the first 64 keys goes
                    // to both halves of O and starts when warps 0-3 hand over:
                    // each of them meets the warp that rescales the other half
                    // of its rows.  Both come here together: the maximum in use
                    // and the new one are the same in both.
                    if constexpr (F::NQ == 1) {
                        tc_fence_before();
                        bar_sync<64>(3 + quarter);
                        tc_fence_after();
                    }
                }
                if (grow) m = top;
                const float base = m == -INFINITY ? 0.f : m;
                const float2 scale2 = make_float2(mul, mul), base2 = make_float2(-base, -base);
                float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
                // 32 scores to probabilities, in 16 columns at `at`
                auto weigh = [&](const uint32_t* v, uint32_t at) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 x = fma2(make_float2(__uint_as_float(v[2 * i]),
                                                    __uint_as_float(v[2 * i + 1])), scale2, base2);
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        if (i & 1) sum1 = add2(sum1, x); else sum0 = add2(sum0, x);
                        pk[i] = pack16<KIND>(x.x, x.y);
                    }
                    tmem_st16(at, pk);
                };
                auto hand_over = [&](int half) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars->p_full[buf][half]);
                };
                weigh(va, t_s + last);
                if constexpr (F::NQ == 2) tmem_ld32(t_s, va);
                weigh(vb, t_s + last + 16);
                if constexpr (F::NQ == 2) tmem_ld32(t_s + 32, vb);
                tmem_wait_st();
                if constexpr (F::NQ == 2) {
                    if (whole) hand_over(1);
                    tmem_wait_ld();
                    if (masked) {
                        mask(va, 0);
                        mask(vb, 32);
                    }
                    weigh(va, t_s);
                    weigh(vb, t_s + 16);
                    tmem_wait_st();
                }
                sum0 = add2(sum0, sum1);
                l += sum0.x + sum0.y;
                if (!whole) {
                    // A key that only some rows attend, or none: 0 * NaN would
                    // reach the others.  Two warps look through the values of
                    // such a unit and clear those that no row attends; if any
                    // that are left are not finite, they are added to the rows
                    // that attend them one by one and leave the stage.
                    ++partial;
                    spin(&bars->checked[0], partial);
                    spin(&bars->checked[1], partial);
                    volatile uint32_t* odd = bars->odd[partial & 7];
                    if (odd[0] | odd[1] | odd[2] | odd[3]) poisoned(odd, j, t_s, key0, lo, hi);
                    if (F::NQ == 2) hand_over(1);
                }
                // One tile: the end waits for the last value product by its
                // phase's parity.  S(j) only tells that product j - 2 is done:
                // were j - 1 still running then, its phase would be taken for
                // that of the last.
                if (F::NQ == 1 && j > 0 && j == take - 1) await(&bars->pv_done[0], it - 1);
                hand_over(F::NQ == 2 ? 0 : wg);
            }
            // the next segment's queries are on their way while this one ends
            w.next(a);
            more = w.open(a);
            if (more) load_queries(w.s.n * a.group - w.cur.tile * F::M);
            await(&bars->pv_done[tw], it - 1);
            tc_fence_after();
            if constexpr (F::NQ == 1) {   // both halves' sums
                float* xl = xmax + (it & 1) * 256;
                xl[wg * 128 + row] = l;
                bar_sync<1, 256>();
                l = xl[row] + xl[128 + row];
                bar_sync<1, 256>();
            }
            const bool full = begins && ends;
            const int which = begins;   // 1: tail slot, 0: head slot
            if (!full) {
                if (which) {
                    rec.tail = 1;
                    rec.seq = cur.seq;
                    rec.tile = cur.tile;
                    rec.kvh = cur.kvh;
                } else {
                    rec.head = ends ? 2 : 1;
                }
            }
            const bool valid = trow < rows;
            const bool none = lo >= hi;
            const float inv = none ? 0.f : 1.f / l;
            const int rr = cur.tile * F::M + (valid ? trow : 0);
            const int tk = a.by_group.div(rr);
            const int tok = s.q0 + tk, h = cur.kvh * a.group + rr - tk * a.group;
            float* slot = ws.slot(blockIdx.x, which, F::M, DP);
            TQ* orow = static_cast<TQ*>(a.out) + (int64_t)tok * a.o_ts + (int64_t)h * a.o_hs;
            const int d0 = F::NQ == 1 ? wg * 128 : 0;
            // rows of the lanes of this quad (lane q of four stores 16 bytes of each)
            TQ* qrow[4];
            bool qvalid[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int from = (lane & ~3) + i;
                qrow[i] = reinterpret_cast<TQ*>(
                    __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(orow), from));
                qvalid[i] = __shfl_sync(0xffffffffu, (int)valid, from);
            }
#pragma unroll 2
            for (int c = 0; c < F::OC / 32; ++c) {
                uint32_t o[32];
                __syncwarp();
                tmem_ld32(t_o + c * 32, o);
                tmem_wait_ld();
                const int d = d0 + c * 32;
                if (!full) {
                    if (valid) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4*>(slot + ((size_t)(d / 4 + i) * F::M + trow) * 4) =
                                make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                } else {
                    constexpr int OK = std::is_same<TQ, __nv_bfloat16>::value ? KIND_BF16 : KIND_F16;
                    uint4 y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t* yw = reinterpret_cast<uint32_t*>(&y[i]);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            yw[e] = none ? 0u
                                         : pack16<OK>(__uint_as_float(o[8 * i + 2 * e]) * inv,
                                                      __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
                    }
                    // 4 x 4 transposition within the quad, so that a store
                    // covers 64 bytes of a row: swap across lane bit 1, then 0
                    quad_transpose(y, lane);
                    if (d + (lane & 3) * 8 < a.c.dim) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (qvalid[i])
                                *reinterpret_cast<uint4*>(qrow[i] + d + (lane & 3) * 8) = y[i];
                    }
                }
            }
            if (valid && d0 == 0) {
                if (!full) {
                    slot[(size_t)F::M * DP + 2 * trow] = m;
                    slot[(size_t)F::M * DP + 2 * trow + 1] = l;
                } else if (a.lse) {
                    a.lse[(int64_t)tok * a.q_heads + h] =
                        none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
                }
            }
            __syncwarp();
            tc_fence_before();
            if (more) hand_queries();
            stage0 += 2 * F::KPARTS * take;
        }
        if (tid == 0) ws.rec[blockIdx.x] = rec;
    } else if (warp < 12) {
        if (warp == 9) {
            // ------------------------------------------------------- products
            // The whole warp walks along and one elected lane issues: the
            // products' operands are then known to be uniform and stay in
            // uniform registers.  Issued by a lane that branched off alone,
            // each took about 120 cycles, twice what a 128 x 128 x 16 product
            // needs.
            uint32_t it = 0, seg = 0;
            int stage0 = 0;
            auto wait_stage = [&](int n) {
                await(&bars->full[n % F::NST], (uint32_t)(n / F::NST));
            };
            // A descriptor's address field counts 16 bytes and no operand ends
            // beyond it, so the steps are additions to its low word.
            const uint32_t t_mem = uniform(tmem);
            const uint64_t q_desc = umma_desc_sw128(smem_u32(sm));
            const uint64_t k_desc = umma_desc_sw128(smem_u32(sm + F::o_stage));
            const uint64_t v_desc = umma_desc_nmajor(smem_u32(sm + F::o_stage), F::VKEYS * 128);
            auto slot_of = [&](int n) { return uniform((n % F::NST) * (F::STAGEB >> 4)); };
            auto free_at = [&](int n) { return &bars->empty[uniform(n % F::NST)]; };
            // S = Q K^T of one query tile with a unit's keys, from their stages
            // (parts by head dimension), into score buffer b
            auto score = [&](int tile, int j, uint32_t b) {
                const uint32_t d = t_mem + uniform(b * 128);
#pragma unroll
                for (int h = 0; h < F::KPARTS; ++h) {
                    const int n = stage0 + stage_k<F::NQ>(j) + h;
                    if (tile == 0) wait_stage(n);
                    const uint64_t q = q_desc + uniform((tile * F::SLABS + h * F::KSLABS) * 1024);
                    const uint64_t k0 = k_desc + slot_of(n);
                    uint64_t* empty = free_at(n);
                    uint64_t* ready = &bars->s_full[uniform(b)];
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int sl = 0; sl < F::KSLABS; ++sl)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                umma_f16(d, q + (sl * 1024 + k * 2), k0 + (sl * 1024 + k * 2),
                                         F::IDESC_S, h > 0 || sl > 0 || k > 0);
                        if (tile == F::NQ - 1) umma_commit(empty);
                        if (h == F::KPARTS - 1) umma_commit(ready);
                    }
                    __syncwarp();
                }
            };
            // O += P V, half a unit's keys at a time as their probabilities come
            // (two tiles: the second half first)
            auto value = [&](int tile, int j, uint32_t b) {
                const uint32_t p = t_mem + uniform(b * 128);
                const uint32_t d = t_mem + 256 + uniform(tile * DP);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int h = F::NQ == 2 ? 1 - i : i;
                    const int n = stage0 + stage_v<F::NQ>(j, w.take) + (F::NQ == 2 ? 0 : h);
                    if (F::NQ == 1 || (tile == 0 && i == 0)) wait_stage(n);
                    const uint64_t v0 = v_desc + slot_of(n) + (F::NQ == 2 ? h * 512 : 0);
                    uint64_t* empty = free_at(n);
                    uint64_t* done = &bars->pv_done[uniform(tile)];
                    await(&bars->p_full[b][h], F::NQ == 2 ? it : it >> 1);
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f16_ts(d, p + h * 64 + k * 8, v0 + k * 128, F::IDESC_O);
                        if (F::NQ == 1 || (tile == 1 && i == 1)) umma_commit(empty);
                        if (i == 1) umma_commit(done);
                    }
                    __syncwarp();
                }
            };
            while (w.open(a)) {
                const int take = w.take;
                await(&bars->q_full[0], seg);
                if constexpr (F::NQ == 2) {
                    score(0, 0, 0);
                    await(&bars->q_full[1], seg);
                    score(1, 0, 1);
                } else {
                    score(0, 0, it & 1);
                }
                for (int j = 0; j < take; ++j) {
                    if constexpr (F::NQ == 2) {
                        for (int t = 0; t < 2; ++t) {
                            value(t, j, t);
                            if (j + 1 < take) score(t, j + 1, t);
                        }
                    } else {
                        if (j + 1 < take) score(0, j + 1, (it + 1) & 1);
                        value(0, j, it & 1);
                    }
                    ++it;
                    if (lane == 0) *reinterpret_cast<volatile uint32_t*>(&bars->products) = it;
                }
                stage0 += 2 * F::KPARTS * take;
                ++seg;
                w.next(a);
            }
            // every product has been waited for by the softmax warps
        } else if (warp >= 10) {
            // --------------------------- values of partly attended units
            // Units are skipped, so a stage's barrier may be phases behind: a unit
            // is looked at once the value products were issued that come behind
            // the previous use of its stage (which was full, then), and its own
            // cannot be issued before it has been.
            int stage0 = 0;
            uint32_t partial = 0, it = 0;
            while (w.open(a)) {
                const AttendTile tile = attend_tile(a, w.s, w.cur.tile * F::M, F::M);
                for (int j = 0; j < w.take; ++j, ++it) {
                    const int key0 = (w.u0 + j) * kManyKeys;
                    if (key0 >= tile.all_lo && key0 + kManyKeys <= tile.all_hi) continue;
                    ++partial;
                    // two tiles: the stage's last use was as keys two units ago
                    if (F::NQ == 1)
                        spin(&bars->products, it);
                    else if (it > 0)
                        spin(&bars->products, it - 1);
                    uint32_t* odd = bars->odd[partial & 7];
                    for (int h = 0; h < F::KPARTS; ++h) {
                        const int n = stage0 + stage_v<F::NQ>(j, w.take) + h;
                        uint4* st = reinterpret_cast<uint4*>(sm + F::o_stage +
                                                             (n % F::NST) * F::STAGEB);
                        await(&bars->full[n % F::NST], (uint32_t)(n / F::NST));
                        // keys that every row attends are left alone: what
                        // they hold belongs to all rows
                        const int k0 = h * F::VKEYS;
                        const int cut0 = min(max(tile.all_lo - key0 - k0, 0), F::VKEYS);
                        const int cut1 = min(max(tile.all_hi - key0 - k0, cut0), F::VKEYS);
                        const int n_keys = cut0 + F::VKEYS - cut1;
                        constexpr int CPK = DP / 8;   // 16-byte chunks of a key
#pragma unroll 8
                        for (int i = tid - 320; i < n_keys * CPK; i += 64) {
                            const int q = i / CPK, c = i % CPK;
                            const int k = q < cut0 ? q : q - cut0 + cut1;
                            uint4* at = st + (c >> 3) * (F::VKEYS * 8) + k * 8 + (c & 7);
                            const int key = key0 + k0 + k;
                            const uint4 v = *at;
                            if (key < tile.t_lo || key >= tile.t_hi)
                                *at = make_uint4(0, 0, 0, 0);
                            else if (odd16x8<KIND>(v))
                                atomicOr(&odd[(k0 + k) >> 5], 1u << ((k0 + k) & 31));
                        }
                    }
                    fence_async_smem();
                    __threadfence_block();
                    __syncwarp();
                    if (lane == 0) *reinterpret_cast<volatile uint32_t*>(&bars->checked[warp - 10]) = partial;
                }
                stage0 += 2 * F::KPARTS * w.take;
                w.next(a);
            }
        } else if (!F::Q8 && warp == 8) {
            // --------------------------------------------------------- copies
            int stage0 = 0;
            const int piece = a.c.page_size < kManyKeys ? a.c.page_size : kManyKeys;
            const int vpiece = piece < F::VKEYS ? piece : F::VKEYS;
            const int pieces = kManyKeys / piece;
            while (w.open(a)) {
                const int take = w.take;
                const AttendTile tile = attend_tile(a, w.s, w.cur.tile * F::M, F::M);
                // lane i: page of the unit's i-th piece, if some row attends a
                // key of it (the table need not name pages that none does)
                auto page_at = [&](int j) {
                    const int key = (w.u0 + j) * kManyKeys + lane * piece;
                    if (j >= take || lane >= pieces || key >= w.s.len || key >= tile.t_hi ||
                        key + piece <= tile.t_lo)
                        return -1;
                    return kv_page(a.b, a.c, w.cur.seq, key >> a.c.page_shift, a.status);
                };
                auto fill = [&](int n, const CUtensorMap* map, int page_id, int key0, int keys,
                                int step, int x0, int slabs) {
                    const int slot = n % F::NST;
                    if (n >= F::NST) await(&bars->empty[slot], (uint32_t)(n / F::NST) + 1);
                    const int boxes = keys / step;
                    const int b = lane % boxes, sl = lane / boxes;
                    const int key = key0 + b * step;
                    const int page = __shfl_sync(0xffffffffu, page_id,
                                                 (key & (kManyKeys - 1)) / piece);
                    const bool go = sl < slabs && page >= 0;
                    const int n_go = __popc(__ballot_sync(0xffffffffu, go));
                    if (lane == 0) mbar_arrive_expect_tx(&bars->full[slot], n_go * step * 128);
                    __syncwarp();
                    if (go)
                        tma_load_3d(sm + F::o_stage + slot * F::STAGEB + sl * keys * 128 + b * step * 128,
                                    map, x0 + sl * 64, key & (a.c.page_size - 1),
                                    page * a.c.heads + w.cur.kvh, &bars->full[slot]);
                };
                int page = page_at(0);
                auto keys_of = [&](int j, int pg) {
                    for (int h = 0; h < F::KPARTS; ++h)
                        fill(stage0 + stage_k<F::NQ>(j) + h, &kmap, pg, (w.u0 + j) * kManyKeys,
                             kManyKeys, piece, h * 128, F::KSLABS);
                };
                keys_of(0, page);
                for (int j = 0; j < take; ++j) {
                    const int ahead = page_at(j + 1);
                    if (F::NQ == 1 && j + 1 < take) keys_of(j + 1, ahead);
                    for (int h = 0; h < F::KPARTS; ++h)
                        fill(stage0 + stage_v<F::NQ>(j, take) + h, &vmap, page,
                             (w.u0 + j) * kManyKeys + h * F::VKEYS, F::VKEYS, vpiece, 0, F::SLABS);
                    if (F::NQ == 2 && j + 1 < take) keys_of(j + 1, ahead);
                    page = ahead;
                }
                stage0 += 2 * F::KPARTS * take;
                w.next(a);
            }
        }
    } else if constexpr (F::Q8) {
        // ------------------------------------------------------ Q8_0 decoding
        const int t = tid - 384, nb = a.c.dim >> 5;
        constexpr int CH = F::STAGEB / 32 / 128;   // 16-code chunks of a thread and stage
        constexpr int KC = F::KSLABS * 4;          // chunks of a row in a stage of keys
        constexpr int VC = F::SLABS * 4;           // chunks of a row in a stage of values
        int stage0 = 0;
        while (w.open(a)) {
            const int take = w.take;
            const int total = 2 * F::KPARTS * take;
            // page ids of a unit's pieces, one per lane; one unit's (with two
            // stages per unit two units') are kept
            const int piece_shift = a.c.page_shift < 7 ? a.c.page_shift : 7;
            const AttendTile tile = attend_tile(a, w.s, w.cur.tile * F::M, F::M);
            auto page_ids = [&](int j) {
                const int key = (w.u0 + j) * kManyKeys + (lane << piece_shift);
                if (j >= take || lane >= (kManyKeys >> piece_shift) || key >= w.s.len ||
                    key >= tile.t_hi || key + (1 << piece_shift) <= tile.t_lo)
                    return -1;
                return kv_page(a.b, a.c, w.cur.seq, key >> a.c.page_shift, a.status);
            };
            int ids[F::KPARTS];
#pragma unroll
            for (int h = 0; h < F::KPARTS; ++h) ids[h] = page_ids(h);
            // the segment's n-th stage: unit j, part h, keys or values
            struct Stage {
                int j, h;
                bool v;
            };
            auto stage_of = [&](int n) {
                if (F::NQ == 2) return Stage{n >> 1, 0, (n & 1) != 0};
                const int g = n >> 1;   // K0 | K1 V0 | K2 V1 | ... | V(take-1)
                const bool last = g == 2 * take - 1;
                const bool v = last || (g > 0 && !(g & 1));
                return Stage{last ? take - 1 : v ? g / 2 - 1 : (g + 1) / 2, n & 1, v};
            };
            uint4 code[CH];
            uint32_t scl[CH];
            auto load = [&](const Stage& g, int pid, int c) {
                const int per = KC == VC ? KC : g.v ? VC : KC;
                const int key = (w.u0 + g.j) * kManyKeys + (g.v ? g.h * F::VKEYS : 0) + (c * 128 + t) / per;
                const int d = (g.v ? 0 : g.h * 128) + t % per * 16;
                const int page = __shfl_sync(0xffffffffu, pid, (key & (kManyKeys - 1)) >> piece_shift);
                const bool ok = page >= 0 && key < w.s.len && d < a.c.dim;
                const int64_t r = (((int64_t)page * a.c.heads + w.cur.kvh) << a.c.page_shift) +
                                  (key & (a.c.page_size - 1));
                code[c] = make_uint4(0, 0, 0, 0);
                scl[c] = 0;
                if (ok) {
                    code[c] = __ldg(reinterpret_cast<const uint4*>(
                        static_cast<const int8_t*>(g.v ? a.c.v : a.c.k) + r * a.c.dim + d));
                    scl[c] = __ldg(reinterpret_cast<const unsigned short*>(g.v ? a.c.vs : a.c.ks) +
                                   r * nb + (d >> 5));
                }
            };
            auto ids_of = [&](const Stage& g) {
                return F::KPARTS == 2 && (g.j & 1) ? ids[F::KPARTS - 1] : ids[0];
            };
            {
                const Stage g = stage_of(0);
                const int pid = ids_of(g);
#pragma unroll
                for (int c = 0; c < CH; ++c) load(g, pid, c);
            }
            for (int n = 0; n < total; ++n) {
                const Stage g = stage_of(n);
                if (g.v && g.h == F::KPARTS - 1) {   // this unit's page ids have been used
                    const int next = page_ids(g.j + F::KPARTS);
                    if (F::KPARTS == 2 && (g.j & 1)) ids[F::KPARTS - 1] = next; else ids[0] = next;
                }
                const Stage gn = stage_of(n + 1 < total ? n + 1 : n);
                const int pid = ids_of(gn);
                const int slot = (stage0 + n) % F::NST;
                if (stage0 + n >= F::NST) await(&bars->empty[slot], (uint32_t)((stage0 + n) / F::NST) + 1);
                const int per = KC == VC ? KC : g.v ? VC : KC, keys = g.v ? F::VKEYS : kManyKeys;
                const int q = t % per, c0 = (q & 3) * 2;
                // lanes of the odd slabs store their second half first, so
                // that eight lanes cover eight different 16-byte columns
                const int first = (q >> 2) & 1;
                unsigned char* slab = sm + F::o_stage + slot * F::STAGEB + (q >> 2) * keys * 128;
                unsigned char* at0 = slab + sw128_offset(t / per, c0 + first);
                unsigned char* at1 = slab + sw128_offset(t / per, c0 + 1 - first);
#pragma unroll
                for (int c = 0; c < CH; ++c) {   // 128 / per rows on: whole 8-row atoms
                    const __half2 d = __half2half2(__ushort_as_half((unsigned short)scl[c]));
                    uint32_t x[8];
                    const uint32_t* cw = reinterpret_cast<const uint32_t*>(&code[c]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) codes4(cw[i], d, x[2 * i], x[2 * i + 1]);
                    const uint4 lo4 = make_uint4(x[0], x[1], x[2], x[3]);
                    const uint4 hi4 = make_uint4(x[4], x[5], x[6], x[7]);
                    const int step = c * (128 / per) * 128;
                    *reinterpret_cast<uint4*>(at0 + step) = first ? hi4 : lo4;
                    *reinterpret_cast<uint4*>(at1 + step) = first ? lo4 : hi4;
                    if (n + 1 < total) load(gn, pid, c);   // this chunk of the next stage
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->full[slot]);
            }
            stage0 += total;
            w.next(a);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (tid == 0 && *reinterpret_cast<volatile uint32_t*>(&bars->lost)) kv_flag(a.status, KV_TIMEOUT);
    if (warp == 9) tmem_dealloc(tmem, 512);
}

template <int DP, int KIND, typename TQ>
cudaError_t launch_many(const AttendArgs& a, void* ws, cudaStream_t s) {
    using F = Many<DP, KIND>;
    CUtensorMap kmap{}, vmap{};
    if (!F::Q8) {
        const int piece = a.c.page_size < kManyKeys ? a.c.page_size : kManyKeys;
        if (!attend_map(&kmap, a.c, a.c.k, 64, piece) ||
            !attend_map(&vmap, a.c, a.c.v, 64, piece < F::VKEYS ? piece : F::VKEYS))
            return cudaErrorInvalidValue;
    }
    static bool raised[64] = {};   // shared memory limit, per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 64 || !raised[dev])) {
        e = cudaFuncSetAttribute(k_attend_many<DP, KIND, TQ>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 F::smem);
        if (e == cudaSuccess && dev >= 0 && dev < 64) raised[dev] = true;
    }
    if (e != cudaSuccess) return e;
    k_attend_many<DP, KIND, TQ><<<sm_count(), F::THREADS, F::smem, s>>>(kmap, vmap, a, ws);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_attend_join(a, ws, sm_count(), F::M, DP, s);
}

template <int DP>
cudaError_t launch_dim(const AttendArgs& a, void* ws, cudaStream_t s) {
    if (a.c.type == KV_F16)   // bfloat16 queries: over the expanded form of a Q8_0 cache
        return a.type == KV_F16 ? launch_many<DP, KIND_F16, __half>(a, ws, s)
                                : launch_many<DP, KIND_F16, __nv_bfloat16>(a, ws, s);
    if (a.c.type == KV_BF16) return launch_many<DP, KIND_BF16, __nv_bfloat16>(a, ws, s);
    if (a.type == KV_F16) return launch_many<DP, KIND_Q8, __half>(a, ws, s);
    return launch_many<DP, KIND_Q8, __nv_bfloat16>(a, ws, s);
}

}  // namespace

cudaError_t launch_attend_many(const AttendArgs& a, void* ws, cudaStream_t s) {
    const int dp = attend_dim(a.c.dim);
    if (dp == 64) return launch_dim<64>(a, ws, s);
    if (dp == 128) return launch_dim<128>(a, ws, s);
    return launch_dim<256>(a, ws, s);
}

}  // namespace moeb200
