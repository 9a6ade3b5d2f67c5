// mma16.cuh - 16-bit helpers of the kernels on the warp-wide tensor instruction: conversions, the rest of a rounding, fragments
// and asynchronous copies.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace cdclq {

template <bool BF16>
__device__ __forceinline__ uint16_t half_bits(float v) {
    return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
template <bool BF16>
__device__ __forceinline__ float half_value(uint16_t v) {
    return BF16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}
// v - h, rounded: with h = v rounded, h + rest has twice the significand.  An infinity is all in h.
template <bool BF16>
__device__ __forceinline__ uint16_t rest_bits(float v, uint16_t h) {
    const float high = half_value<BF16>(h);
    return half_bits<BF16>(fabsf(high) < INFINITY ? v - high : 0.0f);
}

// D (16 x 8) += A (16 x 16) B (16 x 8)
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four 8 x 8 pieces; lane l gives the address of row l % 8 of piece l / 8.  TRANS: each piece transposed.
template <bool TRANS>
__device__ __forceinline__ void load_pieces(uint32_t (&v)[4], const void* p) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                     : "r"(at)
                     : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                     : "r"(at)
                     : "memory");
}

// A kernel that ran beside the one before it in the stream ends after it, so that what follows finds both done: one CTA waits.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// 16 bytes to shared memory, zeros unless `live` (src is then not read).
__device__ __forceinline__ void copy16(void* dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
                 "r"(live ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace cdclq
