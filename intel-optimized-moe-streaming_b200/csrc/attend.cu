// attend.cu -- attention over a paged key/value cache: the choice of kernel,
// the joining of split tiles, and the tensor maps of the cache.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "attend_mma.cuh"
#include "launch.h"

namespace moeb200 {

namespace {

constexpr int kJoinWarps = 8;

// Adds the pieces of the tiles that were split over CTAs, in CTA order: the
// CTA with a tail owns its tile, the pieces are its tail and the heads of the
// CTAs behind it up to the one that finished the tile.  grid (ctas, rows /
// rows of a block); WPR warps share a row, each taking every WPR-th piece,
// and are added in order.  A chain of four dependent loads and one pass over
// the pieces: latency, so rows are spread over as many warps as there are
// (tiles of 256 rows x 128: 19 us, 74 us with eight rows in turn per block).
template <typename TO, int DP, int WPR>
__global__ void __launch_bounds__(kJoinWarps * 32) k_attend_join(AttendArgs a, void* wsp, int ctas,
                                                                 int M) {
    constexpr int V = DP / 64;   // float2 of a lane
    __shared__ float2 part[WPR > 1 ? kJoinWarps : 1][V][32];
    __shared__ float part_l[kJoinWarps], part_m[kJoinWarps];
    pdl_enter();
    const AttendWs ws(wsp, ctas);
    const int cta = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const AttendRecord rec = ws.rec[cta];
    if (!rec.tail) return;
    const AttendSeq s = attend_seq(a, rec.seq, nullptr);
    const int row = blockIdx.y * (kJoinWarps / WPR) + warp / WPR;
    const int sub = warp % WPR;
    const int r = rec.tile * M + row;
    const bool valid = row < M && r < s.n * a.group;
    int pieces = 1;
    for (int i = cta + 1; i < ctas; i += 32) {   // up to the first head that ends the tile
        const bool last = i + lane < ctas && ws.rec[i + lane].head == 2;
        const unsigned found = __ballot_sync(0xffffffffu, last);
        if (found) {
            pieces += __ffs(found);
            break;
        }
        pieces += 32;
    }
    pieces = pieces < ctas - cta ? pieces : ctas - cta;
    float top = -INFINITY, l = 0.f;
    float2 o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = make_float2(0.f, 0.f);
    if (valid) {
        // lane p holds the maximum and the sum of piece p of a group of 32
        for (int p0 = sub; p0 < pieces; p0 += 32 * WPR) {
            const int p = p0 + lane * WPR;
            float2 ml = make_float2(-INFINITY, 0.f);
            if (p < pieces)
                ml = *reinterpret_cast<const float2*>(ws.slot(cta + p, p == 0, M, DP) +
                                                      (size_t)M * DP + 2 * row);
            const float high = fmaxf(top, warp_max(ml.x));
            if (high > top) {
                const float f = exp2f(top - high);
                l *= f;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    o[v].x *= f;
                    o[v].y *= f;
                }
                top = high;
            }
            const float mine = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
            l += warp_sum(mine * ml.y);
            const int left = (pieces - p0 + WPR - 1) / WPR;
            const int n = left < 32 ? left : 32;
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                const int q = p0 + i * WPR;
                const float f = __shfl_sync(0xffffffffu, mine, i);
                const float* sl = ws.slot(cta + q, q == 0, M, DP) + 4 * row + 2 * (lane & 1);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float2 x =
                        *reinterpret_cast<const float2*>(sl + (v * 16 + (lane >> 1)) * 4 * M);
                    o[v].x = fmaf(f, x.x, o[v].x);
                    o[v].y = fmaf(f, x.y, o[v].y);
                }
            }
        }
    }
    if constexpr (WPR > 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) part[warp][v][lane] = o[v];
        if (lane == 0) {
            part_m[warp] = top;
            part_l[warp] = l;
        }
        __syncthreads();
        if (sub) return;
        float high = top;
        for (int w = 1; w < WPR; ++w) high = fmaxf(high, part_m[warp + w]);
        l = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = make_float2(0.f, 0.f);
        for (int w = 0; w < WPR; ++w) {
            const float pm = part_m[warp + w];
            const float f = pm == -INFINITY ? 0.f : exp2f(pm - high);
            l = fmaf(f, part_l[warp + w], l);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float2 x = part[warp + w][v][lane];
                o[v].x = fmaf(f, x.x, o[v].x);
                o[v].y = fmaf(f, x.y, o[v].y);
            }
        }
        top = high;
    }
    if (!valid) return;
    const int tok = a.by_group.div(r), h = rec.kvh * a.group + r - tok * a.group;
    int lo, hi;
    attend_range(s.first + tok, s.len, a.causal, a.window, lo, hi);
    const bool none = lo >= hi;
    const float inv = 1.f / l;
    TO* out = static_cast<TO*>(a.out) + (int64_t)(s.q0 + tok) * a.o_ts + (int64_t)h * a.o_hs;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int d = v * 64 + lane * 2;
        if (d < a.c.dim) {
            TO y[2] = {kv_from_f<TO>(none ? 0.f : o[v].x * inv), kv_from_f<TO>(none ? 0.f : o[v].y * inv)};
            *reinterpret_cast<uint32_t*>(out + d) = *reinterpret_cast<uint32_t*>(y);
        }
    }
    if (a.lse && lane == 0)
        a.lse[(int64_t)(s.q0 + tok) * a.q_heads + h] =
            none ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
}

template <typename TO, int DP, int WPR>
cudaError_t join_as(const AttendArgs& a, void* ws, int ctas, int M, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas, M * WPR / kJoinWarps);
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_attend_join<TO, DP, WPR>, a, ws, ctas, M);
}

// Few rows: up to all CTAs' pieces in a row, four warps share them.  Many
// rows: a few pieces, a warp per row.
template <typename TO, int DP>
cudaError_t join(const AttendArgs& a, void* ws, int ctas, int M, cudaStream_t s) {
    return M <= 16 ? join_as<TO, DP, 4>(a, ws, ctas, M, s)
                         : join_as<TO, DP, 1>(a, ws, ctas, M, s);
}

}  // namespace

cudaError_t launch_attend_join(const AttendArgs& a, void* ws, int ctas, int M, int DP,
                               cudaStream_t s) {
    if (a.type == KV_F16) {
        if (DP == 64) return join<__half, 64>(a, ws, ctas, M, s);
        if (DP == 128) return join<__half, 128>(a, ws, ctas, M, s);
        return join<__half, 256>(a, ws, ctas, M, s);
    }
    if (DP == 64) return join<__nv_bfloat16, 64>(a, ws, ctas, M, s);
    if (DP == 128) return join<__nv_bfloat16, 128>(a, ws, ctas, M, s);
    return join<__nv_bfloat16, 256>(a, ws, ctas, M, s);
}

bool attend_map(void* map, const KvCache& c, const void* base, int cols, int rows) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    });
    if (!encode) return false;
    const int eb = c.type == Q8_0 ? 1 : 2;
    const CUtensorMapDataType dt = c.type == Q8_0    ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : c.type == KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const cuuint64_t dims[3] = {(cuuint64_t)c.dim, (cuuint64_t)c.page_size,
                                (cuuint64_t)c.pages * c.heads};
    const cuuint64_t strides[2] = {(cuuint64_t)c.dim * eb, (cuuint64_t)c.dim * eb * c.page_size};
    const cuuint32_t box[3] = {(cuuint32_t)cols, (cuuint32_t)rows, 1};
    const cuuint32_t es[3] = {1, 1, 1};
    return encode(static_cast<CUtensorMap*>(map), dt, 3, const_cast<void*>(base), dims, strides,
                  box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  cols * eb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

// A Q8_0 cache's pages of the batch's sequences as binary16 (scale * code
// rounded once, what the kernels take them for), laid out by sequence.  Moves
// 3 bytes a value; one block per page, 16 codes a thread.
__global__ void __launch_bounds__(256) k_attend_expand(KvBatch b, KvCache c, __half* k, __half* v,
                                                       int window, unsigned* status) {
    const int seq = blockIdx.y, page = blockIdx.x;
    const int len = __ldg(b.kv_lens + seq);
    const int n = __ldg(b.q_start + seq + 1) - __ldg(b.q_start + seq);
    const int first = page << c.page_shift;
    // pages behind the sequence, or before the first row's window
    if (first >= len || n <= 0) return;
    if (window > 0 && (int64_t)first + c.page_size <= (int64_t)len - n - window + 1) return;
    const int id = kv_page(b, c, seq, page, status);
    if (id < 0) return;
    const int units = (c.heads << c.page_shift) * c.dim >> 4;
    const int64_t from = ((int64_t)id * c.heads << c.page_shift) * c.dim;
    const int64_t to = (((int64_t)seq * b.max_pages + page) * c.heads << c.page_shift) * c.dim;
#pragma unroll 2
    for (int i = threadIdx.x; i < units; i += 256) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int64_t at = from + (int64_t)i * 16;
            const uint4 codes = __ldcs(reinterpret_cast<const uint4*>(
                static_cast<const int8_t*>(w ? c.v : c.k) + at));
            const __half2 d = __half2half2((w ? c.vs : c.ks)[at >> 5]);
            uint32_t x[8];
            codes4(codes.x, d, x[0], x[1]);
            codes4(codes.y, d, x[2], x[3]);
            codes4(codes.z, d, x[4], x[5]);
            codes4(codes.w, d, x[6], x[7]);
            uint4* out = reinterpret_cast<uint4*>((w ? v : k) + to + (int64_t)i * 16);
            out[0] = make_uint4(x[0], x[1], x[2], x[3]);
            out[1] = make_uint4(x[4], x[5], x[6], x[7]);
        }
    }
}

// Rows per sequence and key/value head, on average, up to which attend_few.cu
// is the faster one.  16 sequences of 8000 tokens, two key/value heads, us:
//                  rows   16: few, many    32: few, many    64: few, many
//   16-bit, 64 wide        32, 46           36, 46           46, 46
//   16-bit, 128            46, 52           60, 52           85, 54
//   16-bit, 256            79, 71 (8 rows: 72, 71)           192, 77
//   Q8_0, 128              42, 95           58, 97           91, 97
//   Q8_0, 256              67, 140          97, 142          161, 145 (48: 128, 142)
// One sequence, or 64 of 1000 tokens, give the same order or differ by 2 us.
// The mean decides for the whole call, since the rows of each sequence are known
// on the device only: 200 single tokens and a chunk of 512 rows over 16k tokens
// (4 rows a token, 128 wide) take 965 us in one call, 259 + 145 us in two.
int few_rows(int dp, bool q8) {
    if (q8) return dp > 128 ? 48 : 64;
    return dp > 128 ? 8 : dp > 64 ? 16 : 64;
}

// How a call runs.  Few rows: tiles of 8 up to 8 rows per sequence, of 16 beyond
// (a tile reads the keys again; 16 rows x 128 as above: 56 us in tiles of 8, 46
// in one of 16; 8 rows: 42 and 44).  Many rows: tiles of 128 or 256.  Those
// decode a Q8_0 cache's values as often as a sequence has tiles, on warps that
// the softmax needs (chunks of 2048 rows over 8k keys, 32/8 heads x 128: 444 us,
// expanded first 260 us); from two tiles on the pages are expanded to binary16
// in the workspace, if the table's width bounds that by 1 GB.
struct AttendPlan {
    bool many;
    int rows;             // of a tile
    size_t base, plane;   // workspace of the kernel; bytes of an expanded plane, or 0
    size_t bytes() const { return base + 2 * plane; }
};

AttendPlan attend_plan(const KvBatch& b, const KvCache& c, int group) {
    const int dp = attend_dim(c.dim);
    const int64_t rows = (int64_t)b.T * group;
    AttendPlan p{};
    p.many = rows > few_rows(dp, c.type == Q8_0) * (int64_t)b.B;
    p.rows = p.many ? many_rows(dp) : rows > 8 * (int64_t)b.B ? 16 : 8;
    p.base = align_up(AttendWs::bytes(p.many ? sm_count() : attend_few_ctas(), p.rows, dp));
    if (p.many && c.type == Q8_0 && rows > p.rows * (int64_t)b.B && b.max_pages > 0 &&
        b.B <= 65535) {
        const uint64_t values =
            ((uint64_t)b.B * b.max_pages * c.heads << c.page_shift) * (uint64_t)c.dim;
        if ((uint64_t)b.B * b.max_pages * c.heads <= 0x7fffffffull && values * 4 <= (1ull << 30))
            p.plane = align_up((size_t)values * 2);
    }
    return p;
}

}  // namespace

size_t attend_workspace_bytes(const KvBatch& b, const KvCache& c, int q_heads) {
    return attend_plan(b, c, q_heads / c.heads).bytes();
}

cudaError_t launch_attend(const AttendArgs& a, void* ws, cudaStream_t s) {
    const AttendPlan p = attend_plan(a.b, a.c, a.group);
    if (!p.many) return launch_attend_few(a, p.rows, ws, s);
    if (!p.plane) return launch_attend_many(a, ws, s);
    AttendArgs x = a;
    x.c.type = KV_F16;
    x.c.k = static_cast<char*>(ws) + p.base;
    x.c.v = static_cast<char*>(ws) + p.base + p.plane;
    x.c.ks = x.c.vs = nullptr;
    x.c.pages = a.b.B * a.b.max_pages;
    x.b.table = nullptr;
    k_attend_expand<<<dim3(a.b.max_pages, a.b.B), 256, 0, s>>>(
        a.b, a.c, static_cast<__half*>(x.c.k), static_cast<__half*>(x.c.v), a.window, a.status);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? launch_attend_many(x, ws, s) : e;
}

}  // namespace moeb200
