// attend.cu -- attention over a paged key/value cache: the choice of kernel,
// the joining of split tiles, and the tensor maps of the cache.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "attend.h"
#include "launch.h"
#include "sm100.cuh"

namespace moeb200 {

namespace {

constexpr int kJoinThreads = 256;

// Adds the pieces of the tiles that were split over CTAs, in CTA order: the
// CTA with a tail owns its tile, the pieces are its tail and the heads of the
// CTAs behind it up to the one that finished the tile.  grid (ctas, slices of
// rows); a row is spread over DP / 4 threads, several groups of threads take
// every other piece and are added in order.
template <typename TO, int DP>
__global__ void __launch_bounds__(kJoinThreads) k_attend_join(AttendArgs a, void* wsp, int ctas,
                                                              int M, int rows_per_block) {
    constexpr int kCols = DP / 4;                    // threads of a row
    constexpr int kGroups = kJoinThreads / kCols;    // pieces taken at once
    __shared__ float4 part[kGroups][kCols];
    __shared__ float part_l[kGroups];
    pdl_enter();
    const AttendWs ws(wsp, ctas);
    const int cta = blockIdx.x;
    const AttendRecord rec = ws.rec[cta];
    if (!rec.tail) return;
    int pieces = 1;
    for (int i = cta + 1; i < ctas; ++i) {
        ++pieces;
        if (ws.rec[i].head == 2) break;
    }
    const AttendSeq s = attend_seq(a, rec.seq, nullptr);
    const int col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
    for (int i = 0; i < rows_per_block; ++i) {
        const int row = blockIdx.y * rows_per_block + i;
        const int r = rec.tile * M + row;
        if (row >= M || r >= s.n * a.group) return;
        // the pieces' maxima first, then one pass over their sums
        float top = -INFINITY;
        for (int p = 0; p < pieces; ++p) {
            const float* sl = ws.slot(cta + p, p == 0, M, DP);
            top = fmaxf(top, sl[(size_t)M * DP + 2 * row]);
        }
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
        for (int p = grp; p < pieces; p += kGroups) {
            const float* sl = ws.slot(cta + p, p == 0, M, DP);
            const float m = sl[(size_t)M * DP + 2 * row];
            const float f = m == -INFINITY ? 0.f : exp2f(m - top);
            const float4 v = reinterpret_cast<const float4*>(sl + (size_t)row * DP)[col];
            l += f * sl[(size_t)M * DP + 2 * row + 1];
            o.x += f * v.x;
            o.y += f * v.y;
            o.z += f * v.z;
            o.w += f * v.w;
        }
        part[grp][col] = o;
        if (col == 0) part_l[grp] = l;
        __syncthreads();
        if (grp == 0) {
            for (int g = 1; g < kGroups; ++g) {
                const float4 v = part[g][col];
                o.x += v.x;
                o.y += v.y;
                o.z += v.z;
                o.w += v.w;
                l += part_l[g];
            }
            const int tok = r / a.group, h = rec.kvh * a.group + r % a.group;
            int lo, hi;
            attend_range(s.first + tok, s.len, a.causal, a.window, lo, hi);
            const bool none = lo >= hi;
            const float inv = none ? 0.f : 1.f / l;
            if (none) o = make_float4(0.f, 0.f, 0.f, 0.f);
            if (col * 4 < a.c.dim) {
                TO y[4] = {kv_from_f<TO>(o.x * inv), kv_from_f<TO>(o.y * inv),
                           kv_from_f<TO>(o.z * inv), kv_from_f<TO>(o.w * inv)};
                TO* out = static_cast<TO*>(a.out) + (int64_t)(s.q0 + tok) * a.o_ts +
                          (int64_t)h * a.o_hs + col * 4;
                *reinterpret_cast<uint2*>(out) = *reinterpret_cast<uint2*>(y);
            }
            if (a.lse && col == 0)
                a.lse[(int64_t)(s.q0 + tok) * a.q_heads + h] =
                    none ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
        }
        __syncthreads();
    }
}

template <typename TO, int DP>
cudaError_t join(const AttendArgs& a, void* ws, int ctas, int M, cudaStream_t s) {
    const int rows = M <= 16 ? 4 : 8;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas, (M + rows - 1) / rows);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_attend_join<TO, DP>, a, ws, ctas, M, rows);
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

// Tiles of many rows from 33 rows per sequence on average.
bool use_many(const KvBatch& b, int group) { return (int64_t)b.T * group > 32 * (int64_t)b.B; }

}  // namespace

size_t attend_workspace_bytes(const KvBatch& b, const KvCache& c, int q_heads) {
    const int dp = attend_dim(c.dim);
    return use_many(b, q_heads / c.heads) ? AttendWs::bytes(sm_count(), many_rows(dp), dp)
                                          : AttendWs::bytes(attend_few_ctas(), kFewRows, dp);
}

cudaError_t launch_attend(const AttendArgs& a, void* ws, cudaStream_t s) {
    return use_many(a.b, a.group) ? launch_attend_many(a, ws, s) : launch_attend_few(a, ws, s);
}

}  // namespace moeb200
