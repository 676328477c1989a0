// Device code shared by the batched prompt phase's kernels (q4_gemm.hip,
// prefill.hip) and the products of experts (moe.hip).

#pragma once

#include "cw_internal.hpp"

namespace cwi {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kT = 256;

__device__ __forceinline__ float2 add(float2 a, float2 b) {
    return make_float2(a.x + b.x, a.y + b.y);
}
__device__ __forceinline__ float4 add(float4 a, float4 b) {
    return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// The sum in order of the S >= 1 partials at(0), at(1), ...: four requested
// at a time, so that no load waits for another's sum.
template <typename At>
__device__ __forceinline__ auto sum_parts(int S, At at) {
    auto v = at(0);
    int s = 1;
    for (; s + 4 <= S; s += 4) {
        const auto a = at(s), b = at(s + 1), c = at(s + 2), d = at(s + 3);
        v = add(add(add(add(v, a), b), c), d);
    }
    if (s + 3 == S) {
        const auto a = at(s), b = at(s + 1), c = at(s + 2);
        return add(add(add(v, a), b), c);
    }
    if (s + 2 == S) {
        const auto a = at(s), b = at(s + 1);
        return add(add(v, a), b);
    }
    return s < S ? add(v, at(s)) : v;
}

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

constexpr float kUnscale = 0.0625f;  // the factor 16 of products with nibbles()

// 4 quant bytes -> the B fragment of their 8 weights
__device__ __forceinline__ f16x8 nibbles(uint32_t w) {
    const f16x2 o1 = {(_Float16)1032.0f, (_Float16)1032.0f};
    const f16x2 o16 = {(_Float16)1152.0f, (_Float16)1152.0f};
    // v_and_or_b32 takes no literal: the masks in scalar registers, the exponents in
    // a vector register, which the compiler, knowing their values, would not do (it
    // takes an and and an or).  No instruction is written out: the compiler would not
    // see that one writes a register in which a matrix product is still under way.
    uint32_t m1 = 0x000F000Fu, m16 = 0x00F000F0u, one = 0x64006400u;
    asm("" : "+s"(m1));
    asm("" : "+s"(m16));
    asm("" : "+v"(one));
    const uint32_t h = w >> 8;
    auto sub = [&](uint32_t v, uint32_t mask, f16x2 o) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, (v & mask) | one) - o);
    };
    return __builtin_bit_cast(f16x8, (u32x4){sub(w, m1, o1), sub(w, m16, o16), sub(h, m1, o1),
                                             sub(h, m16, o16)});
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

typedef __attribute__((address_space(3))) unsigned char lds_u8;

// 64-lane global -> LDS DMAs of 16 bytes per lane: lane i's bytes land at
// lds_dst + 16 i; lds_dst is wave-uniform (M0, set by the compiler through the
// operand constraint), the source a uniform base plus a lane offset, or an
// address per lane.  Written as asm so the compiler's wait-count pass does not track
// them and adds no wait before the LDS reads of another buffer; the kernel
// orders them itself with counted vmcnt waits and a barrier.
__device__ __forceinline__ uint32_t lds_off(unsigned char *p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_u8 *)p);
}
//
// The compiler puts none of the wait states in front of an asm that the hardware wants:
// one after a write of M0, five after a vector instruction's write (v_readfirstlane,
// v_readlane) of a scalar register that the DMA reads.  dma16 has the one, for bases that
// scalar instructions made (with five a prompt of 512 tokens took 0.8 % longer);
// tests/test_lds_dma.py looks at the built kernels for others.
__device__ __forceinline__ void dma16(const void *base, uint32_t off, unsigned char *lds_dst) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(off), "s"(base), "{m0}"(lds_off(lds_dst))
                 : "memory");
}

// DMAs to an address in LDS (a number: of a pointer each would look whether it is null)
// from a base that is the same in every lane, wherever the compiler has it: 16 bytes a
// lane at lds + 16 i, and 4 bytes at lds + 4 i.
template <typename T>
__device__ __forceinline__ const T *uniform(const T *p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return reinterpret_cast<const T *>((uintptr_t)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ void dma16u(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(off), "s"(uniform(static_cast<const char *>(base))), "{m0}"(lds)
                 : "memory");
}
__device__ __forceinline__ void dma4u(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1"
                 :
                 : "v"(off), "s"(uniform(static_cast<const char *>(base))), "{m0}"(lds)
                 : "memory");
}

// all but the newest N of this wave's loads have completed
template <int N>
__device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
    __builtin_amdgcn_sched_barrier(0);
}

// Workgroup barrier on LDS data only: __syncthreads would also wait for
// every DMA in flight
__device__ __forceinline__ void lds_barrier() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

}  // namespace cwi
