// The instructions of the MX4 kernels that the Q8_0 kernels do not use, one small function each.
#pragma once

#include <stdint.h>

namespace q8 {

// Eight floats to eight E2M1 codes in a word, v[0] in the lowest four bits: nearest, ties to even, saturating at 6.
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float (&v)[8])
{
    uint32_t out;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(out)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return out;
}

// The eight values of a word of codes as pairs of binary16, out[0] the two lowest.
__device__ __forceinline__ void cvt_f16x2_e2m1(uint32_t codes, uint32_t (&out)[4])
{
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3])
        : "r"(codes));
}

// The same for four codes.
__device__ __forceinline__ void cvt_f16x2_e2m1_4(unsigned short codes, uint32_t &low, uint32_t &high)
{
    asm("{\n\t.reg .b8 b0, b1;\n\t"
        "mov.b16 {b0, b1}, %2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t}"
        : "=r"(low), "=r"(high)
        : "h"(codes));
}

// An approximate power of two (within two steps of a float).
__device__ __forceinline__ float ex2_approx(float v)
{
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// A thread's own copy of four bytes, global to shared; zeros where `bytes` is 0 (the source is not read then).
__device__ __forceinline__ void copy_async_4(uint32_t dst, const void *src, uint32_t bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Arrive on a barrier when all of this thread's own copies so far have landed (counted among the barrier's arrivals).
__device__ __forceinline__ void copy_async_arrive(uint32_t bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void st_shared_b8(uint32_t addr, uint32_t value)
{
    asm volatile("{ .reg .b16 h; cvt.u16.u32 h, %1; st.shared.b8 [%0], h; }" ::"r"(addr), "r"(value) : "memory");
}

// Four words into the shared memory of a block of the cluster, counted on that block's barrier `bar` (addresses of mapa_shared,
// 16-byte aligned).
__device__ __forceinline__ void store_counted_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t bar)
{
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr),
                 "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar)
                 : "memory");
}

__device__ __forceinline__ unsigned short ld_shared_u16(uint32_t addr)
{
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
    return v;
}

// 32 rows of 16 bytes from shared memory (a descriptor without swizzle) to four columns of tensor memory, the same in each
// quarter of the lanes: the way a block of scales is laid down for the MMA.
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D[tmem] (+)= A[smem] * B[smem], one 128 x N x 64 step of E2M1 codes with a scale (a power of two) per 32 values of
// either, scales in tensor memory, float sums.
__device__ __forceinline__ void umma_mx4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                         uint32_t b_scales, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
}

// The same two for a pair of blocks (cta_group::2): scales from either block's shared memory into its own tensor memory, the same
// offsets in both; D is 256 x N, each block 128 rows of it with their scales, B half of its columns in either block's shared
// memory and the scales of all of them in both.
__device__ __forceinline__ void pair_tmem_copy_scales(uint32_t taddr, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void pair_mma_mx4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                             uint32_t b_scales, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
}

// Has the phase ended?  Does not wait.
__device__ __forceinline__ uint32_t mbar_test(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done;
}

} // namespace q8
