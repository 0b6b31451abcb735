// attn_mfma.h -- what the matrix-core attention kernels share (context_attn.hip, tree_attn.hip): fragment types, the MFMA
// forms, the LDS-DMA issue and the cross-row maximum.
#pragma once
#include "common.h"

namespace mi355q
{
namespace
{

typedef __attribute__((ext_vector_type(8))) __bf16 cbf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 cf16x8_t;
typedef __attribute__((ext_vector_type(4))) float cf32x4_t;
typedef __attribute__((ext_vector_type(16))) float cf32x16_t;
typedef __attribute__((ext_vector_type(4))) short cs16x4_t;
typedef __attribute__((address_space(3))) cs16x4_t lds_cs16x4_t;
typedef __attribute__((address_space(3))) void ctx_lds_void_t;
typedef __attribute__((address_space(1))) const void ctx_gbl_void_t;

// LDS-DMA issued from inline asm: the compiler's waitcnt pass makes every LDS read that follows a
// __builtin_amdgcn_global_load_lds wait for vmcnt(0) (it cannot tell the ring stages apart), which would serialise
// the prefetch with the compute.  Issued this way the DMA is ordered only by the explicit s_waitcnt vmcnt + barrier
// of the tile loop.  lds_off: wave-uniform LDS byte address; lane l's 16 bytes land at lds_off + 16 l.
__device__ __forceinline__ void ctx_dma16(const void* gptr, uint32_t lds_off)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(gptr), "s"(lds_off) : "memory", "m0");
}

// fmaxf on MFMA outputs makes hipcc emit a canonicalising v_max_f32 per operand first; the scores are never sNaN
__device__ __forceinline__ float ctx_max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// max over lane ^ 16 (W = 16) or lane ^ 32 (W = 32) through v_permlane{16,32}_swap: with both operands holding x
// the two results are [x0 x0 x2 x2] / [x1 x1 x3 x3] by rows of 16 lanes (W = 16) or [lo lo] / [hi hi] by halves
// (W = 32), so their max is the pairwise all-reduce.  The swap and the max sit in ONE asm statement: given the builtin,
// hipcc treats the swap's two results as the same value when its operands are copies of each other and emits
// max(r0, r0) -- every lane then ends up with the first row's maximum instead of the column's (a
// consistent but too small running maximum, harmless until a sliding window leaves that row with nothing but masked
// scores).  s_nop 1 either side: a VALU write needs 2 wait states before the swap reads it, and the swap's results
// 2 before a VALU reads them; the compiler cannot see inside the statement to add them.
template <int W>
__device__ __forceinline__ float ctx_swap_max(float x)
{
    float a = x, b = x;
    if constexpr (W == 16)
        asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1\n\tv_max_f32 %0, %0, %1" : "+v"(a), "+v"(b));
    else
        asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1\n\tv_max_f32 %0, %0, %1" : "+v"(a), "+v"(b));
    return a;
}

template <typename T>
__device__ __forceinline__ cf32x4_t ctx_mfma(const uint4& a, const uint4& b, cf32x4_t c);
template <>
__device__ __forceinline__ cf32x4_t ctx_mfma<bf16_t>(const uint4& a, const uint4& b, cf32x4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(cbf16x8_t, a), __builtin_bit_cast(cbf16x8_t, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ cf32x4_t ctx_mfma<f16_t>(const uint4& a, const uint4& b, cf32x4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(cf16x8_t, a), __builtin_bit_cast(cf16x8_t, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ cf32x16_t ctx_mfma32(const uint4& a, const uint4& b, cf32x16_t c);
template <>
__device__ __forceinline__ cf32x16_t ctx_mfma32<bf16_t>(const uint4& a, const uint4& b, cf32x16_t c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(cbf16x8_t, a), __builtin_bit_cast(cbf16x8_t, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ cf32x16_t ctx_mfma32<f16_t>(const uint4& a, const uint4& b, cf32x16_t c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(cf16x8_t, a), __builtin_bit_cast(cf16x8_t, b), c, 0, 0, 0);
}

} // namespace
} // namespace mi355q
