// attend_mma.cuh -- pieces that the two attention kernels share.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "attend.h"
#include "umma.cuh"

namespace moeb200 {

enum : int { KIND_F16 = 0, KIND_BF16 = 1, KIND_Q8 = 2 };

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int KIND>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if constexpr (KIND == KIND_BF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&v);
    } else {
        __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&v);
    }
}

// Four codes times their block's scale: binary16 pairs (c0, c1), (c2, c3).
__device__ __forceinline__ void codes4(uint32_t codes, __half2 d, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = codes ^ 0x80808080u;   // code + 128
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140);   // binary16 1024 + 128 + code
    uint32_t b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __float2half2_rn(1152.f);
    __half2 x = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&a), off), d);
    __half2 y = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&b), off), d);
    lo = *reinterpret_cast<uint32_t*>(&x);
    hi = *reinterpret_cast<uint32_t*>(&y);
}

template <int KIND>
__device__ __forceinline__ bool odd16(uint32_t pair) {   // a NaN or an infinity in a pair
    constexpr uint32_t e = KIND == KIND_BF16 ? 0x7f80u : 0x7c00u;
    return (pair & e) == e || ((pair >> 16) & e) == e;
}

template <int KIND>
__device__ __forceinline__ bool odd16x8(const uint4& v) {   // in eight values
    // an exponent of ones carries into the sign bit
    constexpr uint32_t e = KIND == KIND_BF16 ? 0x7f807f80u : 0x7c007c00u;
    constexpr uint32_t one = KIND == KIND_BF16 ? 0x00800080u : 0x04000400u;
    return ((((v.x & e) + one) | ((v.y & e) + one) | ((v.z & e) + one) | ((v.w & e) + one)) &
            0x80008000u) != 0;
}

// Power of two that takes a row maximum of magnitude `top` to [1, 2) (1 for
// zero, subnormal, infinite and NaN rows): a bfloat16 row times it is exact
// in binary16 but for values 2^-14 times smaller than the maximum.  Rows from
// 2^113 on are taken to [2^15, 2^16), below binary16's largest value, so that
// the factor is a normal number and scale / factor finite up to scales of 2^15.
__device__ __forceinline__ float row_factor(float top) {
    const uint32_t e = __float_as_uint(top) >> 23;
    return e > 1 && e < 255 ? __uint_as_float(((e < 240 ? 254u : 269u) - e) << 23) : 1.f;
}

// What takes a score to units of log 2, for a query row held times `factor`.
// Not zero, or keys that a row does not attend (-infinity) would become NaN: at
// 1e-37 all scores are equal, as with 0.  Not infinite: scores of zero stay zero.
__device__ __forceinline__ float score_factor(float scale, float factor) {
    return fminf(fmaxf(fabsf(scale) / factor * kLog2e, 1e-37f), 3.402823466e38f);
}

// 32 lanes x 32 consecutive 32-bit columns of tensor memory.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
        "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
          "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
          "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]),
          "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
        "%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
          "r"(v[15])
        : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
        "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
          "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
          "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
          "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}

__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr));
    return v;
}

__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

}  // namespace moeb200
