// half_split.h - matrix operands as 16-bit fragments (gfx950 MFMA), shared by the kernels that
// multiply fp32 tables on the 16-bit matrix cores.
//
// An fp32 value is held as a pair of halves: x 2^s = hi + lo, hi = fp16(x 2^s) and
// lo = fp16(x 2^s - hi), with s a power of two shared by a row (or by rows of like size), so that the
// largest entry lies in [2^14, 2^15).  hi + lo carries 23 bits of x, down to 2^-39 of that
// largest entry (fp16's smallest subnormal is 2^-24).  A product is three MFMAs,
// hi hi + hi lo + lo hi, summed in fp32; the lo lo term, 2^-22 of the product, is left out.
// That is fp32's accuracy over sums of 64 and more terms at a third of the fp16 rate: 518 TFLOP/s
// of the 1555 that a large library product reaches, against 153 for fp32's own.
#pragma once

#include "common.h"

namespace igr {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));  // 16 bytes that a register array may hold
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

enum : int32_t { kF32 = 0, kBF16 = 1, kF16 = 2 };  // IGR_DTYPE_*

inline int64_t dtype_bytes(int32_t t) { return t == kF32 ? 4 : 2; }

// How a table of each type is fed to the matrix cores: NS 16-bit planes, a block scale 2^(kOff - e).
struct SplitF32 {
    typedef float elem;
    typedef half8_t frag;
    static constexpr int NS = 2, kOff = 14;
    static constexpr bool kScaled = true;
};
struct PlainBF16 {
    typedef __bf16 elem;
    typedef bf16x8_t frag;
    static constexpr int NS = 1, kOff = 0;
    static constexpr bool kScaled = false;
};
struct PlainF16 {
    typedef _Float16 elem;
    typedef half8_t frag;
    static constexpr int NS = 1, kOff = 0;
    static constexpr bool kScaled = false;
};

#ifdef __HIPCC__

__device__ __forceinline__ f32x16_t mfma32(half8_t a, half8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 2^e for |e| <= 126
__device__ __forceinline__ float pow2f(int e) { return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23); }

// floor(log2 a) of a finite a >= 0, held to [-100, 127] (100 below one: 2^(14 + 100) still is
// a float, and a block of zeros must not set the scale that it shares with others).
__device__ __forceinline__ int block_exponent(float amax) {
    const int e = (int)((__builtin_bit_cast(uint32_t, amax) >> 23) & 255u) - 127;
    return e < -100 ? -100 : e;
}

// N 16-byte groups from memory to LDS without passing through registers, `t` of 256 threads; complete after
// copies_done().  (N a multiple of 64: a wave copies 1 KB as it lies.)
template <int N>
__device__ __forceinline__ void copy_to_lds(const u32x4_t *src, u32x4_t *dst, int t) {
    static_assert(N % 64 == 0, "whole waves");
    typedef const __attribute__((address_space(1))) u32x4_t *gptr;
    typedef __attribute__((address_space(3))) u32x4_t *lptr;
#pragma unroll
    for (int i = 0; i < N; i += 256)
        if (N % 256 == 0 || i + (t & ~63) < N)
            __builtin_amdgcn_global_load_lds((gptr)(src + i + t), (lptr)(dst + i + (t & ~63)), 16, 0, 0);
}
__device__ __forceinline__ void copies_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// Eight fp32 values as the NS fragments of one lane.
template <class P>
struct Frags {
    typename P::frag p[P::NS];
};

// x - h[I], the half taken as it lies: one mixed-precision fma, exact (the compiler converts the half
// first, a third instruction for each value).
template <int I>
__device__ __forceinline__ float rest_of(half2_t h, float x) {
    float r;
    if constexpr (I == 0)
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    else
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}

// Both parts rounded to nearest: the pair is off by 2^-23 of the value or half of 2^-24, unbiased.
__device__ __forceinline__ void split8(const float (&v)[8], Frags<SplitF32> &f) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const half2_t h = __builtin_convertvector((float2_t{v[i], v[i + 1]}), half2_t);
        const half2_t l = __builtin_convertvector((float2_t{rest_of<0>(h, v[i]), rest_of<1>(h, v[i + 1])}), half2_t);
        f.p[0][i] = h[0];
        f.p[0][i + 1] = h[1];
        f.p[1][i] = l[0];
        f.p[1][i + 1] = l[1];
    }
}
// Half types: one rounding to nearest, off by at most half a step (2^-8 of the value for bf16, 2^-11 for fp16).
__device__ __forceinline__ void split8(const float (&v)[8], Frags<PlainBF16> &f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.p[0][i] = (__bf16)v[i];
}
__device__ __forceinline__ void split8(const float (&v)[8], Frags<PlainF16> &f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.p[0][i] = (_Float16)v[i];
}

// acc[n] += a b[n] over the planes (hi lo, lo hi, hi hi): the products of one a with NB b's, one part of all of them after the other, so
// that consecutive MFMAs do not wait for each other's sums.
template <class P, int NB, class B>
__device__ __forceinline__ void mfma_row(const Frags<P> &a, const B &b, f32x16_t (&acc)[NB]) {
    if constexpr (P::NS == 2) {
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[n] = mfma32(a.p[0], b(n).p[1], acc[n]);
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[n] = mfma32(a.p[1], b(n).p[0], acc[n]);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[n] = mfma32(a.p[0], b(n).p[0], acc[n]);
}

#endif
}  // namespace igr
