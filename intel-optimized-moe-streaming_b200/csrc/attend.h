// attend.h -- arguments of the attention over a paged cache, and how its work
// is cut into pieces for the GPU.
//
// The rows of a sequence (token, query head of one key/value head's group) are
// cut into tiles of M rows that share a key/value head; a tile walks the keys
// its rows attend in units of KT keys.  The units of all tiles form one line,
// and each CTA takes an equal stretch of it, so a CTA holds at most one tile
// that began in an earlier CTA (its head) and one that ends in a later CTA
// (its tail); such pieces leave their unnormalised sums in the workspace and
// k_attend_join adds them up in CTA order.  The cut balances units whatever the
// lengths, costs at most two partial tiles per CTA, and needs no length on the
// host.  (It does not choose the kernel: that is one for the call, attend.cu.)
//
// Held in 16 bits, because the matrix instructions take no wider operands of
// these types: the probabilities (the softmax sum adds them unrounded; a second
// operand for what is cut off would double the value products), Q8_0 values
// (scale * code) and bfloat16 queries over them.  Error of the outputs against 64
// bits, in units of what rounding the output alone gives: 1.1 to 1.4; Q8_0 into
// binary16, where the rounded keys weigh most, 1.5 to 2.5.  Everything else is
// fp32.
#pragma once

#include "kv.cuh"

namespace moeb200 {

// Quotients by a divisor d set on the host: with s = ceil(log2 d) and
// m = floor(2^32 (2^s - d) / d) + 1, n / d = (mulhi(n, m) + n) >> s for
// 0 <= n < 2^31.
struct FastDiv {
    uint32_t d, m, s;
    FastDiv() = default;
    explicit FastDiv(int by) : d((uint32_t)by), m(0), s(0) {
        while ((1ull << s) < d) ++s;
        m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ int div(int n) const {
        return (int)((__umulhi((uint32_t)n, m) + (uint32_t)n) >> s);
    }
#endif
};

struct AttendArgs {
    KvBatch b;
    KvCache c;
    const void* q;    // [T][q_heads][dim], strides in elements
    void* out;
    float* lse;       // [T][q_heads] or null
    int64_t q_ts, q_hs, o_ts, o_hs;
    int type;         // of q and out
    int q_heads, group;
    FastDiv by_group;
    float scale;
    int causal, window;
    unsigned* status;
};

// Pieces a CTA left in the workspace.
struct AttendRecord {
    int head;          // 0 none, 1 a middle piece of a tile, 2 its last piece
    int tail;          // 1: the first piece of the tile (seq, tile, kvh)
    int seq, tile, kvh;
    int pad[3];
};

// Workspace: one record per CTA, then two slots per CTA (head, tail) of M rows
// of DP sums with each row's maximum (in units of log 2) and softmax sum.  Sum
// d of a row is at (d / 4 * M + row) * 4 + d % 4: threads that own a row each
// write whole lines.
struct AttendWs {
    AttendRecord* rec;
    float* slots;
    __host__ __device__ static size_t slot_floats(int M, int DP) { return (size_t)M * (DP + 2); }
    __host__ __device__ static size_t bytes(int ctas, int M, int DP) {
        return ((ctas * sizeof(AttendRecord) + 255) & ~(size_t)255) +
               2 * (size_t)ctas * slot_floats(M, DP) * 4;
    }
    __host__ __device__ AttendWs(void* p, int ctas)
        : rec(static_cast<AttendRecord*>(p)),
          slots(reinterpret_cast<float*>(static_cast<char*>(p) +
                                         ((ctas * sizeof(AttendRecord) + 255) & ~(size_t)255))) {}
    __device__ float* slot(int cta, int which, int M, int DP) const {
        return slots + (2 * (size_t)cta + which) * slot_floats(M, DP);
    }
};

cudaError_t launch_kv_rows(bool write, const KvBatch& b, const KvCache& c, int type, void* k,
                           int64_t k_ts, int64_t k_hs, void* v, int64_t v_ts, int64_t v_hs,
                           unsigned* status, cudaStream_t s);

size_t attend_workspace_bytes(const KvBatch& b, const KvCache& c, int q_heads);
cudaError_t launch_attend(const AttendArgs& a, void* ws, cudaStream_t s);

// Head dimension that the kernels are built for: the next of 64, 128, 256
// (the values beyond head_dim are zeros).
inline int attend_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Tiles of 8 or 16 rows (attend_few.cu): decoding and other calls of few rows.
int attend_few_ctas();
cudaError_t launch_attend_few(const AttendArgs& a, int rows, void* ws, cudaStream_t s);

// Tiles of 256 rows (128 for a head dimension above 128) on tcgen05
// (attend_many.cu): chunks of prompts.
inline int many_rows(int dp) { return dp > 128 ? 128 : 256; }
cudaError_t launch_attend_many(const AttendArgs& a, void* ws, cudaStream_t s);

// Tensor map over a cache plane [pages * heads][page_size][dim]: boxes of
// `cols` values x `rows` rows, 128-byte swizzle when a box row has 128 bytes.
bool attend_map(void* map, const KvCache& c, const void* base, int cols, int rows);

// Whether a call may need k_attend_join after tiles of M rows and units of
// KT keys on `ctas` CTAs, and its launch.
cudaError_t launch_attend_join(const AttendArgs& a, void* ws, int ctas, int M, int DP,
                               cudaStream_t s);

// Keys [lo, hi) that the row at position pos attends (len: cached tokens).
__host__ __device__ __forceinline__ void attend_range(int pos, int len, int causal, int window,
                                                      int& lo, int& hi) {
    hi = causal && pos + 1 < len ? pos + 1 : len;
    lo = window > 0 && pos >= window ? pos - window + 1 : 0;
    if (hi < lo) hi = lo;
}

#ifdef __CUDACC__

// Longest sequence: a key's number, rounded up to the units that a kernel looks
// ahead to, stays below 2^31.
constexpr int64_t kAttendKeys = 0x7fff0000;

struct AttendSeq {
    int q0, n;        // first row of the batch, number of rows
    int len, first;   // cached tokens; position of the first row
};

__device__ __forceinline__ AttendSeq attend_seq(const AttendArgs& a, int b, unsigned* status) {
    AttendSeq s;
    int q0 = __ldg(a.b.q_start + b);
    const int end = __ldg(a.b.q_start + b + 1);   // may lie behind the given rows
    int raw = __ldg(a.b.kv_lens + b);
    raw = raw > 0 ? raw : 0;
    q0 = q0 > 0 ? q0 : 0;
    const int q1 = end < a.b.T ? end : a.b.T;
    s.q0 = q0;
    s.n = q1 > q0 ? q1 - q0 : 0;
    s.first = s.n > 0 ? raw - (end - q0) : raw;
    int64_t cap = (int64_t)a.b.max_pages << a.c.page_shift;
    cap = cap < kAttendKeys ? cap : kAttendKeys;
    s.len = raw;
    if (raw > cap) {
        kv_flag(status, KV_BAD_LENGTH);
        s.len = (int)cap;
    }
    return s;
}

// First and last row of a tile of rows r0 .. r0 + M - 1 attend keys from t_lo
// and up to t_hi; every row attends [all_lo, all_hi).
struct AttendTile {
    int t_lo, t_hi, all_lo, all_hi;
};

__device__ __forceinline__ AttendTile attend_tile(const AttendArgs& a, const AttendSeq& s, int r0,
                                                  int M) {
    const int last = s.n * a.group - 1;
    const int r1 = r0 + M - 1 < last ? r0 + M - 1 : last;
    AttendTile t;
    attend_range(s.first + a.by_group.div(r0), s.len, a.causal, a.window, t.t_lo, t.all_hi);
    attend_range(s.first + a.by_group.div(r1), s.len, a.causal, a.window, t.all_lo, t.t_hi);
    return t;
}

// Units [lo, hi) of KT keys of a tile; one whose rows attend nothing still has
// a unit, in which its zeros are written.
template <int M, int KT>
__device__ __forceinline__ void attend_units(const AttendArgs& a, const AttendSeq& s, int tile,
                                             int& lo, int& hi) {
    const AttendTile t = attend_tile(a, s, tile * M, M);
    lo = hi = 0;
    if (t.t_hi > t.t_lo) {
        lo = t.t_lo / KT;
        hi = (t.t_hi + KT - 1) / KT;
    }
    if (hi <= lo) hi = lo + 1;
}

template <int M>
__device__ __forceinline__ int attend_tiles(const AttendArgs& a, const AttendSeq& s) {
    return (s.n * a.group + M - 1) / M;
}

// A CTA's place on the line of units.
struct AttendCursor {
    int seq, tile, kvh;
    int unit;         // length of the tile already behind
    int64_t left;     // length of line this CTA still has to do
};

struct AttendScratch {
    int64_t warp_total[16];
    AttendCursor found;
};

// Finds the stretch of CTA `cta` of `ctas`; a short line is cut into no more
// than length / LEAST stretches, rounded up.  A tile is
// COST + units long (COST: what starting and ending it takes, in units; a cut
// inside that part gives the whole tile to the later CTA), once per key/value
// head.  A lane sums
// its share of the sequences, the tiles of a long one being spread over its
// warp; a block scan places the shares, and the warp whose share holds the
// stretch's start walks to it.  Returns in every thread; left = 0: nothing to
// do.  The scratch is shared memory that the caller may use for something else
// afterwards.
template <int M, int KT, int COST, int LEAST, int THREADS>
__device__ AttendCursor attend_place(const AttendArgs& a, AttendScratch& scratch, int cta,
                                     int ctas, unsigned* status) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // consecutive sequences to a warp, and of these to a lane
    constexpr int WARPS = THREADS / 32;
    const int per_warp = (a.b.B + WARPS - 1) / WARPS, share = (per_warp + 31) / 32;
    const int warp_end = min((warp + 1) * per_warp, a.b.B);
    const int b_lane = warp * per_warp + lane * share;
    int64_t mine = 0;
    for (int i = 0; i < share; ++i) {
        const int b = b_lane + i;
        AttendSeq s{};
        int tiles = 0;
        if (b < warp_end) {
            s = attend_seq(a, b, cta == 0 ? status : nullptr);
            tiles = attend_tiles<M>(a, s);
        }
        int64_t sum = 0;
        if (tiles <= 4)
            for (int t = 0; t < tiles; ++t) {
                int lo, hi;
                attend_units<M, KT>(a, s, t, lo, hi);
                sum += hi - lo + COST;
            }
        for (unsigned many = __ballot_sync(0xffffffffu, tiles > 4); many; many &= many - 1) {
            const int from = __ffs(many) - 1;
            AttendSeq q;
            q.q0 = 0;
            q.n = __shfl_sync(0xffffffffu, s.n, from);
            q.len = __shfl_sync(0xffffffffu, s.len, from);
            q.first = __shfl_sync(0xffffffffu, s.first, from);
            const int n = __shfl_sync(0xffffffffu, tiles, from);
            int64_t part = 0;
            for (int t = lane; t < n; t += 32) {
                int lo, hi;
                attend_units<M, KT>(a, q, t, lo, hi);
                part += hi - lo + COST;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
            if (lane == from) sum = part;
        }
        mine += sum * a.c.heads;
    }
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
    }
    if (lane == 31) scratch.warp_total[warp] = before;
    if (tid == 0) scratch.found.left = 0;
    __syncthreads();
    before -= mine;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += scratch.warp_total[w];
        total += scratch.warp_total[w];
    }
    // equal stretches, the first `rest` one longer.  Lines below 2^32, all but
    // the longest, are divided in 32 bits.
    int64_t start = -1, end = -1;
    if (total <= 0xffffffffll) {
        const uint32_t n = (uint32_t)total, most = (n + LEAST - 1) / LEAST;
        const uint32_t active = most < (uint32_t)ctas ? most : (uint32_t)ctas;
        if ((uint32_t)cta < active) {
            const uint32_t each = n / active, rest = n - each * active;
            start = (int64_t)each * cta + ((uint32_t)cta < rest ? (uint32_t)cta : rest);
            end = start + each + ((uint32_t)cta < rest);
        }
    } else {
        const int64_t each = total / ctas, rest = total - each * ctas;
        start = each * cta + (cta < rest ? cta : rest);
        end = start + each + (cta < rest);
    }
    const unsigned owner = __ballot_sync(0xffffffffu, start >= before && start < before + mine);
    if (owner) {
        const int from = __ffs(owner) - 1;
        int64_t skip = start - __shfl_sync(0xffffffffu, before, from);
        const int b0 = warp * per_warp + from * share;
        bool done = false;
        for (int b = b0; b < b0 + share && b < warp_end && !done; ++b) {
            const AttendSeq s = attend_seq(a, b, nullptr);
            const int tiles = attend_tiles<M>(a, s);
            for (int t0 = 0; t0 < tiles && !done; t0 += 32) {
                int64_t n = 0;
                int lo = 0, hi = 0;
                if (t0 + lane < tiles) {
                    attend_units<M, KT>(a, s, t0 + lane, lo, hi);
                    n = (int64_t)(hi - lo + COST) * a.c.heads;
                }
                int64_t upto = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t up = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += up;
                }
                if (skip >= upto - n && skip < upto) {
                    // all heads' units of a long tile may pass 2^31
                    const int64_t at = skip - (upto - n);
                    const int size = hi - lo + COST;
                    scratch.found.seq = b;
                    scratch.found.tile = t0 + lane;
                    scratch.found.kvh = (int)(at / size);
                    scratch.found.unit = (int)(at % size);
                    scratch.found.left = end - start;
                }
                const int64_t all = __shfl_sync(0xffffffffu, upto, 31);
                done = skip < all;
                skip -= all;
            }
        }
    }
    __syncthreads();
    const AttendCursor c = scratch.found;
    __syncthreads();   // the scratch may be overwritten
    return c;
}

// The part of the cursor's tile that falls to this CTA: units u0 ..
// u0 + take - 1 (take may be 0), `begins` / `ends` when these include the
// tile's first and last.  Advance the cursor's `left` by `used`.
struct AttendPart {
    int u0, take;
    int64_t used;
    bool begins, ends;
};

template <int M, int KT, int COST>
__device__ __forceinline__ AttendPart attend_part(const AttendArgs& a, const AttendCursor& c,
                                                  const AttendSeq& s) {
    int lo, hi;
    attend_units<M, KT>(a, s, c.tile, lo, hi);
    const int size = hi - lo + COST;
    const int end = c.left < size - c.unit ? c.unit + (int)c.left : size;
    const int u0 = c.unit > COST ? c.unit - COST : 0, u1 = end > COST ? end - COST : 0;
    AttendPart p;
    p.u0 = lo + u0;
    p.take = u1 - u0;
    p.used = end - c.unit;
    p.begins = u0 == 0;
    p.ends = end == size;
    return p;
}

// Moves to the next tile that has rows (head, then tile, then sequence); `s`
// follows.
template <int M>
__device__ __forceinline__ void attend_next(const AttendArgs& a, AttendCursor& c, AttendSeq& s) {
    c.unit = 0;
    if (++c.kvh < a.c.heads) return;
    c.kvh = 0;
    if (++c.tile < attend_tiles<M>(a, s)) return;
    c.tile = 0;
    while (++c.seq < a.b.B) {
        s = attend_seq(a, c.seq, nullptr);
        if (s.n > 0) return;
    }
    c.left = 0;   // the line ends here
}

#endif

}  // namespace moeb200
