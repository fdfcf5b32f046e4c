// pkv_mma.cuh -- register-operand tensor-core tiles (mma.sync) over fp16 (hi, lo) pairs, and the
// loads and byte permutes that build their operands.
#pragma once

#include "pkv_common.cuh"

namespace pkv {

// (hi, lo) fp16 pair of an fp32 value: hi in the low half (k-pair element 2c), lo in the high half
__device__ __forceinline__ uint32_t h2_split(float v) {
    const __half hi = __float2half_rn(v);
    const __half lo = __float2half_rn(v - __half2float(hi));
    return (uint32_t)__half_as_ushort(hi) | ((uint32_t)__half_as_ushort(lo) << 16);
}

// the hi (or lo) fp16 part of v, in both halves
__device__ __forceinline__ uint32_t h2_dup_part(float v, bool lo) {
    const __half hi = __float2half_rn(v);
    const __half pt = lo ? __float2half_rn(v - __half2float(hi)) : hi;
    const uint32_t u = __half_as_ushort(pt);
    return u | (u << 16);
}

// the hi (or lo) parts of a and b as one pair (a low, b high)
__device__ __forceinline__ uint32_t h2_pair_part(float a, float b, bool lo) {
    const __half ah = __float2half_rn(a), bh = __float2half_rn(b);
    const __half ap = lo ? __float2half_rn(a - __half2float(ah)) : ah;
    const __half bp = lo ? __float2half_rn(b - __half2float(bh)) : bh;
    return (uint32_t)__half_as_ushort(ap) | ((uint32_t)__half_as_ushort(bp) << 16);
}

// d += a . b on one m16n8k16 tile, fp16 operands, fp32 accumulators
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint4 lds_u32x4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

__device__ __forceinline__ uint2 lds_u32x2m(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}

// byte permute with the PTX selector semantics (a selector nibble with bit 3 set replicates the
// sign bit of the selected byte)
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}

// (i_a - 8, i_b - 8) as fp16 from the low nibbles of bytes 0 and 2 (the i_z of two codes)
__device__ __forceinline__ uint32_t zc8(uint32_t t) {
    const uint32_t h = (t & 0x000F000Fu) | 0x64006400u;      // 1024 + i, exact
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __halves2half2(__ushort_as_half(0x6408u),
                                                                                  __ushort_as_half(0x6408u)));
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t f2h2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

}  // namespace pkv
