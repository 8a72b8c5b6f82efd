// Device helpers shared by the attention kernels over the q8_0 cache (gfx950).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace qwfn {
namespace {

typedef int      v4i __attribute__((ext_vector_type(4)));
typedef float    v4f __attribute__((ext_vector_type(4)));

// The compiler's hazard recognizer does not see the VALU writes inside inline
// asm, and an MFMA that reads a VGPR needs two wait states after a VALU wrote
// it. Every asm below whose result can feed an MFMA operand therefore ends
// with s_nop 1.

// One V block's A operands for the lane's 4 keys: v[j] holds dims 2m, 2m+1 of
// key j in its low two bytes (one 2-byte LDS read each); a0[q] = f16 pair
// (dim 2m of keys 2q, 2q+1), a1[q] = f16 pair (dim 2m+1). int8 -> f16 is exact.
__device__ __forceinline__ void cvt_v_block(const uint32_t v[4], uint32_t a0[2], uint32_t a1[2]) {
#define QWFN_SDWA(D, S, DSEL, UNUSED, SSEL) "v_cvt_f16_i16_sdwa " D ", sext(" S ") dst_sel:" DSEL " dst_unused:" UNUSED " src0_sel:" SSEL "\n\t"
#define QWFN_PAIR(D, S0, S1, B) QWFN_SDWA(D, S0, "WORD_0", "UNUSED_PAD", B) QWFN_SDWA(D, S1, "WORD_1", "UNUSED_PRESERVE", B)
    asm(QWFN_PAIR("%0", "%4", "%5", "BYTE_0") QWFN_PAIR("%1", "%6", "%7", "BYTE_0")
        QWFN_PAIR("%2", "%4", "%5", "BYTE_1") QWFN_PAIR("%3", "%6", "%7", "BYTE_1")
        "s_nop 1"
        : "=&v"(a0[0]), "=&v"(a0[1]), "=&v"(a1[0]), "=&v"(a1[1])
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]));
#undef QWFN_PAIR
#undef QWFN_SDWA
}

// x * f16 (low or high half of a packed dword), one v_fma_mix_f32.
__device__ __forceinline__ float mul_f16lo(float x, uint32_t h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel:[0,0,0] op_sel_hi:[0,1,0]" : "=v"(r) : "v"(x), "v"(h));
    return r;
}
__device__ __forceinline__ float mul_f16hi(float x, uint32_t h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "=v"(r) : "v"(x), "v"(h));
    return r;
}
// x + f16 * c (f16 in the low or high half of a packed dword), one v_fma_mix_f32.
__device__ __forceinline__ float fma_f16lo(uint32_t h, float c, float x) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(c), "v"(x));
    return r;
}
__device__ __forceinline__ float fma_f16hi(uint32_t h, float c, float x) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(c), "v"(x));
    return r;
}
__device__ __forceinline__ float xmax(float a, float b) { return a > b ? a : b; }
// max of two scores (finite or -inf, never NaN) in one v_max_f32: fmaxf on an
// asm result gets both operands canonicalised first, and the ternary above is
// a compare plus a select
__device__ __forceinline__ float vmax(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// Reductions over the 4 lanes l, l^16, l^32, l^48 (the four lane groups
// holding one MFMA column), with gfx950's cross-row swaps instead of LDS
// permutes: a swap pair holds lanes l and l^16 (or l^32) between its two
// results. The two results pass through an empty asm: without it the
// compiler's IR folds the second result into the first (r[0] op r[1] becomes
// r[0] op r[0]), which silently turns the reduction into x op x.
template <typename Op>
__device__ __forceinline__ float reduce_lanes16_32(float x, Op op) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r16 = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    unsigned a = r16[0], b = r16[1];
    asm volatile("" : "+v"(a), "+v"(b));
    x = op(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    const unsigned w = __builtin_bit_cast(unsigned, x);
    const auto r32 = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    unsigned c = r32[0], d = r32[1];
    asm volatile("" : "+v"(c), "+v"(d));
    return op(__builtin_bit_cast(float, c), __builtin_bit_cast(float, d));
}
__device__ __forceinline__ float xmax_lanes16_32(float x) {
    return reduce_lanes16_32(x, [](float a, float b) { return vmax(a, b); });
}
__device__ __forceinline__ float sum_lanes16_32(float x) {
    return reduce_lanes16_32(x, [](float a, float b) { return a + b; });
}

// LDS writes of this wave become visible to its other lanes (LDS operations of
// one wave complete in order; the fences keep the compiler from moving them).
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wave-wide LDS DMA: lane i copies the 16 bytes at base + off to LDS[at + 16 i] (base and at the same for all lanes).
// Inline asm, so that the compiler neither moves memory operations across it nor waits for it: wait_vmem does. (m0 is
// read one wait state after its write at the earliest; the compiler keeps nothing in it.)
__device__ __forceinline__ void lds_dma16(const void * base, uint32_t off, uint32_t at) {
    const uint64_t b = (uint64_t) (uintptr_t) base;
    const uint64_t s = (uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) (b >> 32)) << 32 |
                       (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) b);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :: "v"(off), "s"(s), "s"(__builtin_amdgcn_readfirstlane((int) at)) : "memory");
}
// Waits for the wave's vector-memory operations.
__device__ __forceinline__ void wait_vmem() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void * p) { return (uint32_t) (uintptr_t) (const __attribute__((address_space(3))) void *) p; }

}  // namespace
}  // namespace qwfn
