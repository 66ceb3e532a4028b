// attend_few.cu -- attention over a paged cache for calls of few rows per
// sequence: single decoded tokens, drafted tokens, short chunks.
//
// Such a call reads every key and value once and does little with them, so
// it is bound by HBM.  A tile of 8 rows (the query heads of a group, times
// tokens; 16 where sequences have more) is the N of mma.sync: scores come as
// keys x rows, outputs as dimensions x rows, and no product is spent on rows
// that are not there.  The CUDA cores would need all of their rate for 8 heads
// to a group; tcgen05's smallest M is 64, and its operands go through shared
// and tensor memory, which so few rows do not repay.
//
// A warp walks subtiles of 16 to 64 keys (8 KB) on its own: a ring of NS
// shared-memory entries per warp (a subtile's keys, then its values) filled by
// tensor copies with a 128-byte swizzle, no block barrier in the loop.  A
// subtile is one chain of products, maximum, exponentials and products, about
// 1900 cycles long however few keys it has, so it has as many as fit.
// The running maximum, sum and DP x 8 outputs stay in the warp's registers
// until the tile ends; then the four warps' sums are added through shared
// memory.  Probabilities change places between the products by movmatrix.  Two
// CTAs per SM, so that one loads while the other starts or ends a tile.
//
// Q8_0: codes become binary16 by a byte permute (1024 + 128 + code, exact) and
// one subtraction, times the block's scale, rounded once: the value of
// scale * code in binary16.  The order of head dimensions within the key
// product, and of output rows, is permuted so that a thread takes its codes
// as 16 consecutive bytes and no transposing load is needed.
// Measured: 64 contexts of 3.5k tokens, 32/8 heads x 128, bf16: 151 us, 6.03
// TB/s (HBM); 33 x 5 drafted rows over 5 to 3000 tokens, 16/8 x 64, binary16:
// 32 us, 3.35 TB/s; 24 contexts of 18k tokens, 16/2 heads x 256, Q8_0: 109 us,
// 4.36 TB/s (some 1400 instructions a warp and 32 keys, most of them decoding;
// issue slots 45% used: two warps a scheduler wait on their own chains); one
// context of 1000 tokens: 14 us (the start of two kernels, 16 pieces a head).
#include "attend_mma.cuh"
#include "launch.h"

namespace moeb200 {

namespace {

constexpr int kFewWarps = 4;
constexpr int kFewThreads = kFewWarps * 32;
// Starting a tile (its queries, the ring's first copies) and ending it (the join
// of the warps) take about as long as two units: with 0, 1, 2, 3, 4 the 33 x 5
// drafted rows took 52, 41, 40, 40, 42 us, the 64 ragged contexts 181, 176, 173,
// 175, 173, the 24 contexts in Q8_0 122, 115, 114, 116, 116 (single calls after
// a flush of L2).
constexpr int kFewCost = 2;
constexpr uint32_t kFewPolls = 1u << 21;

// Codes that a thread takes of a Q8_0 value row.
template <int DP> constexpr int kFewCodes = DP >= 128 ? 16 : 8;

// NT: row tiles of 8.
template <int DP, int KIND, int NT>
struct Few {
    static constexpr int M = 8 * NT;
    static constexpr bool Q8 = KIND == KIND_Q8;
    static constexpr int EB = Q8 ? 1 : 2;
    static constexpr int ROWB = DP * EB;                       // bytes of a cached row
    static constexpr int SLABB = ROWB < 128 ? ROWB : 128;      // bytes of a row in one copy
    static constexpr int SLABS = ROWB / SLABB;
    // G groups of 16 keys at a time, as many as make an entry of 8 KB (at most 4)
    static constexpr int G = 8192 / (16 * ROWB) > 4 ? 4 : 8192 / (16 * ROWB);
    static constexpr int KEYS = 16 * G;                        // keys of a subtile
    static constexpr int UNIT = KEYS * kFewWarps;              // keys of a unit
    static constexpr int TILEB = KEYS * ROWB;
    static constexpr int SLAB = KEYS * SLABB;
    static constexpr int SCALEB = Q8 ? KEYS * DP / 16 : 0;     // KEYS rows of DP / 32 scales
    // ring entries: at most 102 KB per CTA (two CTAs share an SM), and 8
    static constexpr int FIT = 104448 / (kFewWarps * (TILEB + SCALEB));
    static constexpr int NS = FIT > 8 ? 8 : FIT;
    static constexpr int TILES = DP / 16;                      // output tiles of 16 dimensions
    static constexpr bool QSM = NT * DP > 256;                 // queries in shared memory
    // binary16 probabilities are taken 2^15 times as large (the largest is
    // 2^15, below 65504), so that those down to 2^-29 keep all their bits.  The
    // maximum and what is taken off the scores are rounded up, so that this holds
    // for large scores too, whose neighbours in fp32 lie far apart (at 2^25, 4).
    static constexpr float SHIFT = KIND == KIND_BF16 ? 0.f : 15.f;
    static constexpr int PD = DP < 128 ? DP : 128;             // columns joined per pass
    static constexpr int o_scale = kFewWarps * NS * TILEB;
    static constexpr int o_q = o_scale + kFewWarps * NS * SCALEB;
    static constexpr int o_bar = o_q + (QSM ? DP / 16 * NT * 32 * 8 : 0);
    static constexpr int o_m = o_bar + kFewWarps * NS * 8;
    static constexpr int o_l = o_m + kFewWarps * 16 * 4;
    static constexpr int smem = o_l + kFewWarps * 16 * 4 + 1024;   // 1024: base alignment
    static_assert(NS >= 3, "");
    static_assert(2 * (smem + 1024) <= 233472, "two CTAs per SM");
    static_assert(kFewWarps * M * (PD + 4) * 4 <= o_q, "join buffer inside the ring");
};

template <int KIND>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    if constexpr (KIND == KIND_BF16)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool TRANS>
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
}

// A NaN, an infinity, or a scale that takes code -128 out of binary16 (512 and
// above): where nothing was copied, scales and codes are any bits.
__device__ __forceinline__ bool odd_scale(__half s) {
    return (__half_as_ushort(s) & 0x7fffu) >= 0x6000u;
}

// Key of row n of an 8-key score tile.  Q8_0 swaps odd keys n and n ^ 4: the
// 16-byte chunks that a quarter warp reads of the keys (rows 2 q and 2 q + 1)
// and of the values (those of the even, or the odd, rows) then lie in
// different banks of the swizzled rows.
template <int KIND>
__device__ __forceinline__ int row_key(int n) {
    return KIND == KIND_Q8 ? n ^ ((n & 1) << 2) : n;
}

// Head dimension of output tile i, row n (h: n + 8).
template <int DP, int KIND>
__device__ __forceinline__ int out_dim(int i, int n, int h) {
    using F = Few<DP, KIND, 1>;
    constexpr int C = kFewCodes<DP>;
    if constexpr (F::Q8) return (i / (C / 2)) * (C * 8) + n * C + i % (C / 2) * 2 + h;
    return i * 16 + n + 8 * h;
}

// A pair of 16-bit values, in its place among the copies.
__device__ __forceinline__ uint32_t ldg_first(const void* p) {
    uint32_t v;
    asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// Transposes an 8 x 8 matrix of 16-bit values held as accumulator pairs.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t t;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
    return t;
}

// TQ: type of q and out.
template <int DP, int KIND, int NT, typename TQ>
__global__ void __launch_bounds__(kFewThreads, 2)
k_attend_few(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
             const __grid_constant__ AttendArgs a, void* wsp) {
    using F = Few<DP, KIND, NT>;
    constexpr int M = F::M, R = 2 * NT;   // rows of the tile; rows of a thread
    constexpr bool CONVERT = F::Q8 && std::is_same<TQ, __nv_bfloat16>::value;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint2* qf = reinterpret_cast<uint2*>(sm + F::o_q);
    float* sm_m = reinterpret_cast<float*>(sm + F::o_m);
    float* sm_l = reinterpret_cast<float*>(sm + F::o_l);
    float* joinb = reinterpret_cast<float*>(sm);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n8 = lane >> 2, c4 = lane & 3;
    unsigned char* ring = sm + warp * F::NS * F::TILEB;
    unsigned char* sring = sm + F::o_scale + warp * F::NS * F::SCALEB;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + F::o_bar) + warp * F::NS;
    const int nb = a.c.dim >> 5;   // scale blocks of a row

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (lane == 0)
        for (int i = 0; i < F::NS; ++i) mbar_init(&bars[i], 1);
    mbar_fence_init();

    const int ctas = gridDim.x;
    AttendWs ws(wsp, ctas);
    AttendCursor cur = attend_place<M, F::UNIT, kFewCost, 1, kFewThreads>(
        a, *reinterpret_cast<AttendScratch*>(sm), blockIdx.x, ctas, a.status);
    fence_async_smem();   // the scratch lies in the ring
    AttendRecord rec{};
    int in_slot = 0, out_slot = 0;        // ring positions to fill and to read next
    uint32_t out_phase = 0;
    bool lost = false;
    AttendSeq s{};
    if (cur.left > 0) s = attend_seq(a, cur.seq, nullptr);

    while (cur.left > 0) {
        const AttendPart part = attend_part<M, F::UNIT, kFewCost>(a, cur, s);
        if (part.take <= 0) break;   // the stretch ends before the tile's first unit
        const int u0 = part.u0, take = part.take;
        const int rows = s.n * a.group - cur.tile * M;   // valid rows: the first `rows`
        const AttendTile tile = attend_tile(a, s, cur.tile * M, M);
        const int t_lo = tile.t_lo, t_hi = tile.t_hi, all_lo = tile.all_lo, all_hi = tile.all_hi;
        // A subtile is fetched in boxes of whole pages or parts of one; the
        // page ids of 32 boxes at a time are held one per lane (-1: nothing
        // there).
        const int box = a.c.page_size < F::KEYS ? a.c.page_size : F::KEYS;
        const int boxes = F::KEYS / box;
        int page_of = -1, win = 0;
        uint32_t there = 0;   // bit j % 32: a part of subtile j was fetched
        auto look_up = [&](int b0) {
            win = b0;
            page_of = -1;
            const int j = (b0 + lane) / boxes;
            const int key = ((u0 + j) * kFewWarps + warp) * F::KEYS + (b0 + lane) % boxes * box;
            if (j < take && key < t_hi && key + box > t_lo)
                page_of = kv_page(a.b, a.c, cur.seq, key >> a.c.page_shift, a.status);
        };
        // entry e: the keys (even) or values (odd) of subtile e / 2
        auto fetch = [&](int e) {
            const int j = e >> 1, w = e & 1;
            if (j >= take) return;
            if (j * boxes - win >= 32) look_up(j * boxes);
            const int page = __shfl_sync(0xffffffffu, page_of, (j * boxes - win + lane % boxes) & 31);
            const bool go = lane < boxes && page >= 0;
            const int n = __popc(__ballot_sync(0xffffffffu, go));
            if (!w) there = (there & ~(1u << (j & 31))) | ((n ? 1u : 0u) << (j & 31));
            if (!n) return;
            uint64_t* bar = &bars[in_slot];
            if (lane == 0)
                mbar_arrive_expect_tx(bar, (uint32_t)(n * box * (F::ROWB + (F::Q8 ? nb * 2 : 0))));
            __syncwarp();
            if (go) {
                const int key = ((u0 + j) * kFewWarps + warp) * F::KEYS + lane * box;
                const int row = key & (a.c.page_size - 1);
                const int z = page * a.c.heads + cur.kvh;
                unsigned char* dst = ring + in_slot * F::TILEB + lane * box * F::SLABB;
#pragma unroll
                for (int sl = 0; sl < F::SLABS; ++sl)
                    tma_load_3d(dst + sl * F::SLAB, w ? &vmap : &kmap, sl * (F::SLABB / F::EB), row,
                                z, bar);
                if constexpr (F::Q8)
                    bulk_g2s(sring + in_slot * F::SCALEB + lane * box * nb * 2,
                             (w ? a.c.vs : a.c.ks) + (((int64_t)z << a.c.page_shift) + row) * nb,
                             (uint32_t)(box * nb * 2), bar);
            }
            in_slot = in_slot + 1 == F::NS ? 0 : in_slot + 1;
        };
        auto await = [&]() {
            if (!mbar_wait(&bars[out_slot], out_phase, lost ? 64u : kFewPolls)) lost = true;
        };
        auto release = [&]() {
            out_slot = out_slot + 1 == F::NS ? 0 : out_slot + 1;
            out_phase ^= out_slot == 0;
        };
        // Queries as B operands: this thread's are of row n8 of each row tile;
        // bf16 ones over a Q8_0 cache become binary16 after an exact scaling of
        // the row to a maximum in [1, 2).  The four warps hold the same ones.
        // They are asked for before the ring's first copies, which would keep
        // them waiting until all of those have come (5 us over 33 sequences).
        uint2 qraw[NT][DP / 16];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = t * 8 + n8;
            const int rr = cur.tile * M + (r < rows ? r : 0);
            const int tok = a.by_group.div(rr);
            const TQ* q = static_cast<const TQ*>(a.q) + (int64_t)(s.q0 + tok) * a.q_ts +
                          (int64_t)(cur.kvh * a.group + rr - tok * a.group) * a.q_hs;
#pragma unroll
            for (int st = 0; st < DP / 16; ++st) {   // the two registers of 16 dimensions
                const int d = F::Q8 ? (st >> 2) * 64 + c4 * 16 + (st & 3) * 4 : st * 16 + c4 * 2;
                const int d2 = d + (F::Q8 ? 2 : 8);
                qraw[t][st].x = r < rows && d < a.c.dim ? ldg_first(q + d) : 0u;
                qraw[t][st].y = r < rows && d2 < a.c.dim ? ldg_first(q + d2) : 0u;
            }
        }
        look_up(0);
#pragma unroll 1
        for (int e = 0; e < F::NS; ++e) fetch(e);

        uint2 qreg[F::QSM ? 1 : DP / 16][NT];
        float factor[NT];
        {
            const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                factor[t] = 1.f;
                if constexpr (CONVERT) {
                    float top = 0.f;
#pragma unroll
                    for (int st = 0; st < DP / 16; ++st) {
                        const uint2 w = qraw[t][st];
                        top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w.x << 16)),
                                               fabsf(__uint_as_float(w.x & 0xffff0000u))));
                        top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w.y << 16)),
                                               fabsf(__uint_as_float(w.y & 0xffff0000u))));
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    factor[t] = row_factor(top);
                }
                auto convert = [&](uint32_t w) {
                    if constexpr (CONVERT)
                        w = pack16<KIND_F16>(__uint_as_float(w << 16) * factor[t],
                                             __uint_as_float(w & 0xffff0000u) * factor[t]);
                    return w ^ flip;
                };
#pragma unroll
                for (int st = 0; st < DP / 16; ++st) {
                    const uint2 x = make_uint2(convert(qraw[t][st].x), convert(qraw[t][st].y));
                    if constexpr (F::QSM) {
                        if ((st & 3) == warp) qf[(st * NT + t) * 32 + lane] = x;
                    } else {
                        qreg[st][t] = x;
                    }
                }
            }
            if constexpr (F::QSM) __syncthreads();
        }
        auto q_at = [&](int st, int t) {
            if constexpr (F::QSM) return qf[(st * NT + t) * 32 + lane];
            else return qreg[st][t];
        };
        // this thread's rows t * 8 + 2 c4 + e: the keys they attend, the factor
        // that takes a score to units of log 2
        int lo[R], hi[R];
        float mul[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = i / 2 * 8 + c4 * 2 + (i & 1);
            lo[i] = hi[i] = 0;
            if (r < rows)
                attend_range(s.first + a.by_group.div(cur.tile * M + r), s.len, a.causal, a.window,
                             lo[i], hi[i]);
            float f = 1.f;
            if constexpr (CONVERT)
                f = __shfl_sync(0xffffffffu, factor[i / 2], (c4 * 2 + (i & 1)) * 4);
            mul[i] = score_factor(a.scale, f);
        }
        float o[F::TILES][NT][4];
#pragma unroll
        for (int i = 0; i < F::TILES; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][t][e] = 0.f;
        float m[R], l[R];   // the maximum less SHIFT; the sum, which belongs to it
#pragma unroll
        for (int i = 0; i < R; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
        }

#pragma unroll 1
        for (int j = 0; j < take; ++j) {
            if (!((there >> (j & 31)) & 1)) {
                fetch(2 * j + F::NS);
                fetch(2 * j + 1 + F::NS);
                continue;
            }
            const int key0 = ((u0 + j) * kFewWarps + warp) * F::KEYS;
            // ---- scores: 16 keys x 8 rows; element e: key (e >> 1) * 8 + n8,
            // row 2 c4 + (e & 1)
            float p[F::G][NT][4] = {};
            await();
            {
                const unsigned char* kt = ring + out_slot * F::TILEB;
                if constexpr (!F::Q8) {
                    const uint32_t kaddr = smem_u32(kt);
                    const int key = lane & 15, half = lane >> 4;
#pragma unroll
                    for (int st = 0; st < DP / 16; ++st) {
                        uint32_t ka[F::G][4];
                        const int ch = (st & 3) * 2 + half;
#pragma unroll
                        for (int g = 0; g < F::G; ++g)
                            ldsm4<false>(ka[g], kaddr + (st >> 2) * F::SLAB + (g * 16 + key) * 128 +
                                                    ((ch ^ (key & 7)) << 4));
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const uint2 q = q_at(st, t);
#pragma unroll
                            for (int g = 0; g < F::G; ++g) mma16816<KIND>(p[g][t], ka[g], q.x, q.y);
                        }
                    }
                } else {
                    const __half* ks = reinterpret_cast<const __half*>(sring + out_slot * F::SCALEB);
#pragma unroll
                    for (int sp = 0; sp < DP / 64; ++sp) {
                        const int blk = sp * 2 + (c4 >> 1);
#pragma unroll
                        for (int g = 0; g < F::G; ++g) {
                            uint32_t w[2][4];
                            __half2 d[2];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int key = g * 16 + h * 8 + row_key<KIND>(n8);
                                const int at = F::SLABB == 128
                                                   ? (sp >> 1) * F::SLAB + key * 128 +
                                                         ((((sp & 1) * 4 + c4) ^ (key & 7)) << 4)
                                                   : key * 64 + c4 * 16;
                                *reinterpret_cast<uint4*>(w[h]) =
                                    *reinterpret_cast<const uint4*>(kt + at);
                                d[h] = __half2half2(blk < nb ? ks[key * nb + blk]
                                                             : __ushort_as_half(0));
                            }
#pragma unroll
                            for (int st = 0; st < 4; ++st) {
                                uint32_t ka[4];
                                codes4(w[0][st], d[0], ka[0], ka[2]);
                                codes4(w[1][st], d[1], ka[1], ka[3]);
#pragma unroll
                                for (int t = 0; t < NT; ++t) {
                                    const uint2 q = q_at(sp * 4 + st, t);
                                    mma16816<KIND>(p[g][t], ka, q.x, q.y);
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();
            release();
            fetch(2 * j + F::NS);
            // ---- softmax of this subtile
            const bool whole = key0 >= all_lo && key0 + F::KEYS <= all_hi;
            if (!whole) {
#pragma unroll
                for (int g = 0; g < F::G; ++g)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + g * 16 + (e >> 1) * 8 + row_key<KIND>(n8);
                            const int i = 2 * t + (e & 1);
                            if (key < lo[i] || key >= hi[i]) p[g][t][e] = -INFINITY;
                        }
            }
            bool grew = false;
            float keep[R], base[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                float top = -INFINITY;
#pragma unroll
                for (int g = 0; g < F::G; ++g)
                    top = fmaxf(fmaxf(top, p[g][i / 2][i & 1]), p[g][i / 2][2 + (i & 1)]);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                const float mn = fmaxf(m[i], __fadd_ru(__fmul_ru(top, mul[i]), -F::SHIFT));
                base[i] = mn == -INFINITY ? 0.f : mn;
                keep[i] = ex2(m[i] - base[i]);
                grew = grew || mn > m[i];
                m[i] = mn;
            }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int i = 0; i < R; ++i) l[i] *= keep[i];
#pragma unroll
                for (int i = 0; i < F::TILES; ++i)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][t][e] *= keep[2 * t + (e & 1)];
            }
            uint32_t pb[F::G][NT][2];   // probabilities as B operands: keys x rows
#pragma unroll
            for (int g = 0; g < F::G; ++g)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 2 * t + (e & 1);
                        p[g][t][e] = ex2(fmaf(p[g][t][e], mul[i], -base[i]));
                        l[i] += p[g][t][e];
                    }
                    pb[g][t][0] = transpose8(pack16<KIND>(p[g][t][0], p[g][t][1]));
                    pb[g][t][1] = transpose8(pack16<KIND>(p[g][t][2], p[g][t][3]));
                }
            // ---- values
            await();
            unsigned char* vt = ring + out_slot * F::TILEB;
            __half* vs = reinterpret_cast<__half*>(sring + out_slot * F::SCALEB);
            if (!whole) {
                // A key that only some rows attend, or none: 0 * NaN would
                // reach the others.  Keys that no row attends (they may lie
                // behind the sequence, or not have been copied) become zeros.
                // Of the others, values that are not finite are added to the
                // rows that attend them one by one and leave the tile.
                const int r_lo = t_lo - key0, r_hi = t_hi - key0;
                bool odd = false;
                if constexpr (F::Q8) {
                    for (int i = lane; i < F::KEYS; i += 32)
                        for (int b = 0; b < nb; ++b) {
                            if (i < r_lo || i >= r_hi)
                                vs[i * nb + b] = __ushort_as_half(0);
                            else
                                odd = odd || odd_scale(vs[i * nb + b]);
                        }
                } else {
                    uint4* v4 = reinterpret_cast<uint4*>(vt);
#pragma unroll 4
                    for (int i = lane; i < F::TILEB / 16; i += 32) {
                        const int r = (i >> 3) % F::KEYS;
                        if (r < r_lo || r >= r_hi) {
                            v4[i] = make_uint4(0, 0, 0, 0);
                        } else {
                            const uint4 w = v4[i];
                            odd = odd || odd16x8<KIND>(w);
                        }
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (__any_sync(0xffffffffu, odd)) {
                    // value of key k, dimension d when it is not finite, else 0
                    auto odd_value = [&](int k, int d) {
                        if constexpr (F::Q8) {
                            if (d >= a.c.dim) return 0.f;
                            const __half s = vs[k * nb + (d >> 5)];
                            if (!odd_scale(s)) return 0.f;
                            const int at = F::SLABB == 128
                                               ? (d >> 7) * F::SLAB + k * 128 +
                                                     ((((d >> 4) & 7) ^ (k & 7)) << 4) + (d & 15)
                                               : k * 64 + d;
                            return __half2float(s) * (float)reinterpret_cast<const int8_t*>(vt)[at];
                        } else {
                            const int at = (d >> 6) * F::SLAB + k * 128 +
                                           ((((d >> 3) & 7) ^ (k & 7)) << 4) + (d & 7) * 2;
                            const uint16_t w = *reinterpret_cast<const uint16_t*>(vt + at);
                            if (!odd16<KIND>(w)) return 0.f;
                            return KIND == KIND_BF16 ? __bfloat162float(__ushort_as_bfloat16(w))
                                                     : __half2float(__ushort_as_half(w));
                        }
                    };
#pragma unroll
                    for (int gh = 0; gh < 2 * F::G; ++gh) {   // 8 keys at a time
#pragma unroll 1
                        for (int k8 = 0; k8 < 8; ++k8) {
                            const int k = gh * 8 + k8;
                            const int from = row_key<KIND>(k8) * 4 + c4;   // row_key undoes itself
                            float pk[R];
                            bool at[R];
#pragma unroll
                            for (int i = 0; i < R; ++i) {
                                pk[i] = __shfl_sync(0xffffffffu,
                                                    p[gh / 2][i / 2][(gh & 1) * 2 + (i & 1)], from);
                                at[i] = key0 + k >= lo[i] && key0 + k < hi[i];
                            }
#pragma unroll
                            for (int x = 0; x < F::TILES; ++x)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const float v = odd_value(k, out_dim<DP, KIND>(x, n8, h));
                                    if (v != 0.f) {   // NaN or infinite
#pragma unroll
                                        for (int i = 0; i < R; ++i)
                                            if (at[i]) o[x][i / 2][2 * h + (i & 1)] += pk[i] * v;
                                    }
                                }
                        }
                    }
                    __syncwarp();
                    if constexpr (F::Q8) {
                        for (int i = lane; i < F::KEYS * nb; i += 32)
                            if (odd_scale(vs[i])) vs[i] = __ushort_as_half(0);
                    } else {
                        uint16_t* v2 = reinterpret_cast<uint16_t*>(vt);
                        for (int i = lane; i < F::TILEB / 2; i += 32)
                            if (odd16<KIND>(v2[i])) v2[i] = 0;
                    }
                    fence_async_smem();
                    __syncwarp();
                }
            }
            if constexpr (!F::Q8) {
                const uint32_t vaddr = smem_u32(vt);
                const int key = (lane >> 4) * 8 + (lane & 7), half = (lane >> 3) & 1;
#pragma unroll
                for (int x = 0; x < DP / 16; ++x) {
                    const int ch = (x & 3) * 2 + half;
#pragma unroll
                    for (int g = 0; g < F::G; ++g) {
                        uint32_t va[4];
                        ldsm4<true>(va, vaddr + (x >> 2) * F::SLAB + (g * 16 + key) * 128 +
                                            ((ch ^ (key & 7)) << 4));
#pragma unroll
                        for (int t = 0; t < NT; ++t)
                            mma16816<KIND>(o[x][t], va, pb[g][t][0], pb[g][t][1]);
                    }
                }
            } else {
                constexpr int W = kFewCodes<DP> / 4;   // 32-bit words of codes per key
#pragma unroll
                for (int sl = 0; sl < DP / (kFewCodes<DP> * 8); ++sl) {
                    const int blk = (sl * kFewCodes<DP> * 8 + n8 * kFewCodes<DP>) >> 5;
#pragma unroll
                    for (int g = 0; g < F::G; ++g) {
                        uint32_t w[4][W];
                        __half2 d[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = g * 16 + row_key<KIND>(c4 * 2 + (i & 1)) + (i >> 1) * 8;
                            d[i] = __half2half2(blk < nb ? vs[key * nb + blk] : __ushort_as_half(0));
                            if constexpr (kFewCodes<DP> == 16)
                                *reinterpret_cast<uint4*>(w[i]) = *reinterpret_cast<const uint4*>(
                                    vt + sl * F::SLAB + key * 128 + ((n8 ^ (key & 7)) << 4));
                            else
                                *reinterpret_cast<uint2*>(w[i]) =
                                    *reinterpret_cast<const uint2*>(vt + key * 64 + n8 * 8);
                        }
#pragma unroll
                        for (int q = 0; q < W; ++q) {
                            uint32_t x[4][2];
#pragma unroll
                            for (int i = 0; i < 4; ++i) codes4(w[i][q], d[i], x[i][0], x[i][1]);
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t va[4] = {__byte_perm(x[0][e], x[1][e], 0x5410),
                                                        __byte_perm(x[0][e], x[1][e], 0x7632),
                                                        __byte_perm(x[2][e], x[3][e], 0x5410),
                                                        __byte_perm(x[2][e], x[3][e], 0x7632)};
#pragma unroll
                                for (int t = 0; t < NT; ++t)
                                    mma16816<KIND>(o[sl * (kFewCodes<DP> / 2) + q * 2 + e][t], va,
                                                   pb[g][t][0], pb[g][t][1]);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            release();
            fetch(2 * j + 1 + F::NS);
        }

        // ---- the warps' sums of the tile, or of this piece of it
#pragma unroll
        for (int i = 0; i < R; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
            if (n8 == 0) {
                sm_m[warp * 16 + i / 2 * 8 + c4 * 2 + (i & 1)] = m[i];
                sm_l[warp * 16 + i / 2 * 8 + c4 * 2 + (i & 1)] = l[i];
            }
        }
        __syncthreads();
        float keep[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w)
                mm = fmaxf(mm, sm_m[w * 16 + i / 2 * 8 + c4 * 2 + (i & 1)]);
            keep[i] = m[i] == -INFINITY ? 0.f : ex2(m[i] - mm);
        }
        const bool full = part.begins && part.ends;
        const int which = part.begins;   // 1: tail slot, 0: head slot
        float* slot = ws.slot(blockIdx.x, which, M, DP);
        if (!full) {
            if (which) {
                rec.tail = 1;
                rec.seq = cur.seq;
                rec.tile = cur.tile;
                rec.kvh = cur.kvh;
            } else {
                rec.head = part.ends ? 2 : 1;
            }
        }
        // row of this thread's quads in the second half, and what its sums need
        const int qr = tid % M;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, sm_m[w * 16 + qr]);
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float x = sm_m[w * 16 + qr];
            sum += sm_l[w * 16 + qr] * (x == -INFINITY ? 0.f : ex2(x - top));
        }
        const int orow = cur.tile * M + (qr < rows ? qr : 0);
        const int otok = a.by_group.div(orow);
        const int oh = cur.kvh * a.group + orow - otok * a.group;
        int l0, h0;
        attend_range(s.first + otok, s.len, a.causal, a.window, l0, h0);
        const bool none = l0 >= h0;
        const float inv = none ? 0.f : 1.f / sum;
        TQ* out = static_cast<TQ*>(a.out) + (int64_t)(s.q0 + otok) * a.o_ts + (int64_t)oh * a.o_hs;
#pragma unroll
        for (int pass = 0; pass < DP / F::PD; ++pass) {
#pragma unroll
            for (int x = 0; x < F::TILES; ++x)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = out_dim<DP, KIND>(x, n8, h);
                    if (d / F::PD == pass) {
#pragma unroll
                        for (int i = 0; i < R; ++i)
                            joinb[(warp * M + i / 2 * 8 + c4 * 2 + (i & 1)) * (F::PD + 4) + d % F::PD] =
                                o[x][i / 2][2 * h + (i & 1)] * keep[i];
                    }
                }
            __syncthreads();
            // quads of columns, rows inside: a warp's partial sums fill lines
            for (int i = tid; i < M * F::PD / 4; i += kFewThreads) {
                const int x = i / M * 4;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w) {
                    const float4 t = *reinterpret_cast<const float4*>(
                        joinb + (w * M + qr) * (F::PD + 4) + x);
                    v.x += t.x;
                    v.y += t.y;
                    v.z += t.z;
                    v.w += t.w;
                }
                const int d = pass * F::PD + x;
                if (!full) {
                    *reinterpret_cast<float4*>(slot + (d / 4 * M + qr) * 4) = v;
                } else if (qr < rows && d < a.c.dim) {
                    TQ y[4] = {kv_from_f<TQ>(v.x * inv), kv_from_f<TQ>(v.y * inv),
                               kv_from_f<TQ>(v.z * inv), kv_from_f<TQ>(v.w * inv)};
                    *reinterpret_cast<uint2*>(out + d) =
                        none ? make_uint2(0, 0) : *reinterpret_cast<uint2*>(y);
                }
            }
            fence_async_smem();   // the ring's next copies come after these writes
            __syncthreads();
        }
        if (tid < M) {
            if (!full) {
                slot[M * DP + 2 * qr] = top;
                slot[M * DP + 2 * qr + 1] = sum;
            } else if (a.lse && qr < rows) {
                a.lse[(int64_t)(s.q0 + otok) * a.q_heads + oh] =
                    none ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
            }
        }
        cur.left -= part.used;
        if (cur.left > 0) attend_next<M>(a, cur, s);
    }
    if (lost) kv_flag(a.status, KV_TIMEOUT);
    if (tid == 0) ws.rec[blockIdx.x] = rec;
}

template <int DP, int KIND, int NT, typename TQ>
cudaError_t launch_few(const AttendArgs& a, void* ws, cudaStream_t s) {
    using F = Few<DP, KIND, NT>;
    CUtensorMap kmap, vmap;
    const int box = a.c.page_size < F::KEYS ? a.c.page_size : F::KEYS;
    if (!attend_map(&kmap, a.c, a.c.k, F::SLABB / F::EB, box) ||
        !attend_map(&vmap, a.c, a.c.v, F::SLABB / F::EB, box))
        return cudaErrorInvalidValue;
    static bool raised[64] = {};   // shared memory limit, per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 64 || !raised[dev])) {
        e = cudaFuncSetAttribute(k_attend_few<DP, KIND, NT, TQ>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, F::smem);
        if (e == cudaSuccess && dev >= 0 && dev < 64) raised[dev] = true;
    }
    if (e != cudaSuccess) return e;
    k_attend_few<DP, KIND, NT, TQ>
        <<<attend_few_ctas(), kFewThreads, F::smem, s>>>(kmap, vmap, a, ws);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_attend_join(a, ws, attend_few_ctas(), F::M, DP, s);
}

template <int DP, int NT>
cudaError_t launch_kind(const AttendArgs& a, void* ws, cudaStream_t s) {
    // 16 rows of more than 128 values: attend_many.cu, unless Q8_0
    if constexpr (NT == 1 || DP <= 128) {
        if (a.c.type == KV_F16) return launch_few<DP, KIND_F16, NT, __half>(a, ws, s);
        if (a.c.type == KV_BF16) return launch_few<DP, KIND_BF16, NT, __nv_bfloat16>(a, ws, s);
    }
    if (a.c.type != Q8_0) return cudaErrorInvalidValue;
    if (a.type == KV_F16) return launch_few<DP, KIND_Q8, NT, __half>(a, ws, s);
    return launch_few<DP, KIND_Q8, NT, __nv_bfloat16>(a, ws, s);
}

template <int NT>
cudaError_t launch_dim(const AttendArgs& a, void* ws, cudaStream_t s) {
    const int dp = attend_dim(a.c.dim);
    if (dp == 64) return launch_kind<64, NT>(a, ws, s);
    if (dp == 128) return launch_kind<128, NT>(a, ws, s);
    return launch_kind<256, NT>(a, ws, s);
}

}  // namespace

int attend_few_ctas() { return 2 * sm_count(); }

cudaError_t launch_attend_few(const AttendArgs& a, int rows, void* ws, cudaStream_t s) {
    return rows == 8 ? launch_dim<1>(a, ws, s) : launch_dim<2>(a, ws, s);
}

}  // namespace moeb200
