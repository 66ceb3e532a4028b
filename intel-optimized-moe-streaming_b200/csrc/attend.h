// attend.h -- arguments of the attention over a paged cache, and how its work
// is cut into pieces for the GPU.
//
// The rows of a sequence (token, query head of one key/value head's group) are
// cut into tiles of M rows that share a key/value head; a tile walks the keys
// its rows attend in units of KT keys.  The units of all tiles form one line,
// and each CTA takes an equal stretch of it, so a CTA holds at most one tile
// that began in an earlier CTA (its head) and one that ends in a later CTA
// (its tail); such pieces leave their unnormalised sums in the workspace and
// k_attend_join adds them up in CTA order.  The cut balances batches of any
// mixture of lengths, costs at most two partial tiles per CTA, and needs no
// length on the host.
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

// Pieces a CTA left in the workspace.
struct AttendRecord {
    int head;          // 0 none, 1 a middle piece of a tile, 2 its last piece
    int tail;          // 1: the first piece of the tile (seq, tile, kvh)
    int seq, tile, kvh;
    int pad[3];
};

// Workspace: one record per CTA, then two slots per CTA (head, tail) of M rows
// of DP sums with each row's maximum (in units of log 2) and softmax sum.
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

// Tiles of 16 rows (attend_few.cu): decoding and other calls of few rows.
constexpr int kFewRows = 16;
int attend_few_ctas();
cudaError_t launch_attend_few(const AttendArgs& a, void* ws, cudaStream_t s);

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
    lo = window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0;
    if (hi < lo) hi = lo;
}

#ifdef __CUDACC__

struct AttendSeq {
    int q0, n;        // first row of the batch, number of rows
    int len, first;   // cached tokens; position of the first row
};

__device__ __forceinline__ AttendSeq attend_seq(const AttendArgs& a, int b, unsigned* status) {
    AttendSeq s;
    int q0 = __ldg(a.b.q_start + b), q1 = __ldg(a.b.q_start + b + 1);
    const int raw = __ldg(a.b.kv_lens + b);
    q0 = q0 > 0 ? q0 : 0;
    q1 = q1 < a.b.T ? q1 : a.b.T;
    s.q0 = q0;
    s.n = q1 > q0 ? q1 - q0 : 0;
    s.first = raw - s.n;
    const int64_t cap = (int64_t)a.b.max_pages << a.c.page_shift;
    s.len = raw;
    if (raw > cap) {
        kv_flag(status, KV_BAD_LENGTH);
        s.len = (int)cap;
    }
    return s;
}

// Units [lo, hi) of KT keys of a tile of rows r0 .. r0 + M - 1; a tile whose
// rows attend nothing still has one unit, in which its zeros are written.
template <int M, int KT>
__device__ __forceinline__ void attend_units(const AttendArgs& a, const AttendSeq& s, int tile,
                                             int& lo, int& hi) {
    const int r0 = tile * M;
    int r1 = r0 + M - 1;
    const int last = s.n * a.group - 1;
    r1 = r1 < last ? r1 : last;
    int l0, h0, l1, h1;
    attend_range(s.first + r0 / a.group, s.len, a.causal, a.window, l0, h0);
    attend_range(s.first + r1 / a.group, s.len, a.causal, a.window, l1, h1);
    lo = hi = 0;
    if (h1 > l0) {
        lo = l0 / KT;
        hi = (h1 + KT - 1) / KT;
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
    int unit;         // units of the tile already behind
    int64_t left;     // units this CTA still has to do
};

// Finds the stretch of CTA `cta` of `ctas`: every thread sums the units of its
// share of the sequences, a block scan places the shares, and the thread whose
// share holds the stretch's first unit walks to it.  At least `least` units go
// to a CTA.  Returns in every thread; left = 0: nothing to do.  The scratch is
// shared memory that the caller may use for something else afterwards.
struct AttendScratch {
    int64_t warp_total[16];
    AttendCursor found;
};

template <int M, int KT, int THREADS>
__device__ AttendCursor attend_place(const AttendArgs& a, AttendScratch& scratch, int cta,
                                     int ctas, int least, unsigned* status) {
    int64_t* warp_total = scratch.warp_total;
    AttendCursor& found = scratch.found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int share = (a.b.B + THREADS - 1) / THREADS;
    const int b0 = tid * share;
    const int b1 = b0 + share < a.b.B ? b0 + share : a.b.B;
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) {
        const AttendSeq s = attend_seq(a, b, cta == 0 ? status : nullptr);
        const int tiles = attend_tiles<M>(a, s);
        int64_t sum = 0;
        for (int t = 0; t < tiles; ++t) {
            int lo, hi;
            attend_units<M, KT>(a, s, t, lo, hi);
            sum += hi - lo;
        }
        mine += sum * a.c.heads;
    }
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
    }
    if (lane == 31) warp_total[warp] = before;
    if (tid == 0) found.left = 0;
    __syncthreads();
    before -= mine;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += warp_total[w];
        total += warp_total[w];
    }
    int64_t active = (total + least - 1) / least;
    active = active < ctas ? active : ctas;
    if (cta < active) {
        const int64_t start = total * cta / active, end = total * (cta + 1) / active;
        if (start >= before && start < before + mine) {
            int64_t skip = start - before;
            for (int b = b0; b < b1; ++b) {
                const AttendSeq s = attend_seq(a, b, nullptr);
                const int tiles = attend_tiles<M>(a, s);
                int t = 0;
                for (; t < tiles; ++t) {
                    int lo, hi;
                    attend_units<M, KT>(a, s, t, lo, hi);
                    const int64_t n = (int64_t)(hi - lo) * a.c.heads;
                    if (skip < n) {
                        found.seq = b;
                        found.tile = t;
                        found.kvh = (int)(skip / (hi - lo));
                        found.unit = (int)(skip % (hi - lo));
                        found.left = end - start;
                        break;
                    }
                    skip -= n;
                }
                if (t < tiles) break;
            }
        }
    }
    __syncthreads();
    const AttendCursor c = found;
    __syncthreads();   // the scratch may be overwritten
    return c;
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
