// va_tok.h -- shared device helpers of the token operators (va_tok_linear.hip, va_tok_qk.hip, va_tok_attn.hip): vector
// types, bf16 conversions, the exact three-term split of a float, activations.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/va355.h"
#include "va_dev.h"

namespace tok {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) void lvoid_t;

// the largest side of an operand that the kernels' 32-bit counts take, rounded up to a tile
constexpr int SIDE_MAX = 0x7fffffff - 1023;

// whether a x b workgroups can be launched: a launch counts its threads in 32 bits
inline bool grid_ok(int64_t a, int64_t b, int threads) { return a <= 0xffffffffll / threads / (b > 1 ? b : 1); }

// a kernel's dynamic LDS beyond 64 KiB, once a device
template <auto KERNEL, int LDS>
hipError_t big_lds() {
    static DevFlag attr;
    if (LDS <= 65536 || attr()) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e == hipSuccess) attr() = true;
    return e;
}

// consecutive workgroups go to the 8 XCDs in turn: the i-th workgroup of an XCD takes the i-th tile of a contiguous
// run, so that neighbouring tiles (which read the same operand rows) share that XCD's L2
__device__ __forceinline__ int xcd_tile(int bid, int ntiles) {
    const int q = ntiles / 8, r = ntiles % 8, x = bid % 8, j = bid / 8;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + j;
}

// the same in runs of C: an XCD takes every eighth run, so that tiles of unequal work spread over the XCDs
template <int C>
__device__ __forceinline__ int xcd_runs(int bid, int ntiles) {
    const int x = bid % 8, j = bid / 8;
    return bid < ntiles / (8 * C) * (8 * C) ? (j / C * 8 + x) * C + j % C : bid;
}

// two floats -> packed bf16 (round to nearest even)
__device__ __forceinline__ unsigned pk_bf16(float a, float b) {
    return __builtin_bit_cast(unsigned, (bf16x2){(__bf16)a, (__bf16)b});
}
__device__ __forceinline__ float bf_lo(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

// e4m3 bytes -> bf16, exact (every e4m3 value is a bf16 value)
__device__ __forceinline__ bf16x8 e4m3x8(uint2 q) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)q.x, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)q.x, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)q.y, 1.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)q.y, 1.0f, true);
    return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x = h + m + l exactly, each the round-to-nearest bf16 of what remains (x - h and x - h - m are exact in float: the
// remainders have at most 16 and 8 significant bits).  |m| <= 2^-8 |x| and |l| <= 2^-16 |x|, so the six term products hh, hm,
// mh, hl, mm, lh leave out ml, lm and ll: together at most 2^-23 + 2^-32 of |a b|.  A value whose h would be an infinity (an
// infinity, or from 0x1.ffp127 on) has a NaN for l here, which makes a NaN of every sum that it enters: who finds one forms
// its sums once more with split3_far.
__device__ __forceinline__ void split3(const float (&x)[8], bf16x8 (&t)[3]) {
    unsigned w[3][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a = x[2 * e], b = x[2 * e + 1];
        w[0][e] = pk_bf16(a, b);
        a -= bf_lo(w[0][e]), b -= bf_hi(w[0][e]);
        w[1][e] = pk_bf16(a, b);
        a -= bf_lo(w[1][e]), b -= bf_hi(w[1][e]);
        w[2][e] = pk_bf16(a, b);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) t[k] = __builtin_bit_cast(bf16x8, (u32x4){w[k][0], w[k][1], w[k][2], w[k][3]});
}

// The same for any value.  Beyond bf16's largest, h is that largest one and the remainder is split on.  An infinity is
// (+-1, 0, +-inf): l meets the other factor's h alone, whose sign is the factor's and which is 0 only where the factor is, and
// two infinities meet each other's +-1, so products and their sums are the infinities and NaNs that they have to be.
__device__ __forceinline__ void split3_far(const float (&x)[8], bf16x8 (&t)[3]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = x[e];
        const bool inf = __builtin_isinf(a), far = fabsf(a) >= 0x1.ffp127f;
        const __bf16 h = (__bf16)(far ? copysignf(inf ? 1.0f : 0x1.fep127f, a) : a);
        const float r = inf ? 0.0f : a - (float)h;
        const __bf16 m = (__bf16)r;
        t[0][e] = h, t[1][e] = m, t[2][e] = (__bf16)(inf ? a : r - (float)m);
    }
}

// x Phi(x) = x erfc(-x / sqrt 2) / 2 (the erfc form keeps the left tail's relative accuracy); the tanh form as
// x / (1 + exp(-2 u)), the same function
__device__ __forceinline__ float activate(float x, int act) {
    switch (act) {
        case VA_ACT_SILU: return x / (1.0f + expf(-x));
        case VA_ACT_GELU: return 0.5f * x * erfcf(-0.70710678118654752f * x);
        case VA_ACT_GELU_TANH: return x / (1.0f + expf(-1.5957691216057308f * (x + 0.044715f * x * x * x)));
        case VA_ACT_RELU: return x < 0.0f ? 0.0f : x;
        default: return x;
    }
}

// The same for a result that is rounded to bf16 (2^-8): hardware reciprocal and exponential, and x Phi(x) = max(x, 0) -
// |x| Q(|x|) with the Gaussian tail Q(z) = erfc(z / sqrt 2) / 2 as a polynomial in t = 1 / (1 + 0.376 z) times exp(-z^2 / 2):
// the minimax fit of the relative error over z <= 13.4 (where Q leaves float's range), 2.8e-5, so that the left tail keeps
// what bf16 holds of it.  20 issue slots against erfcf's 60: in a product
// with K = 1024 the activations of a tile would take longer than its MFMAs.
__device__ __forceinline__ float activate_bf16(float x, int act) {
    switch (act) {
        case VA_ACT_SILU:
            return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
        case VA_ACT_GELU: {
            const float z = fminf(fabsf(x), 1e4f), t = __builtin_amdgcn_rcpf(__builtin_fmaf(z, 0.376f, 1.0f));
            const float p = t * __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, -0.09111865f,
                            0.19932078f), 0.08426869f), 0.15805252f), 0.14946288f);
            return __builtin_fmaf(-z, p * __builtin_amdgcn_exp2f(-0.72134752f * x * x), fmaxf(x, 0.0f));
        }
        case VA_ACT_GELU_TANH:
            return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.3022081987f * __builtin_fmaf(0.044715f * x * x, x, x)));
        case VA_ACT_RELU: return x < 0.0f ? 0.0f : x;
        default: return x;
    }
}

// n results at once: one (uniform) branch for all of them
template <bool EXACT, int N>
__device__ __forceinline__ void activate_n(float (&r)[N], int act) {
    switch (act) {
        case VA_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = EXACT ? activate(r[i], VA_ACT_SILU) : activate_bf16(r[i], VA_ACT_SILU);
            break;
        case VA_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = EXACT ? activate(r[i], VA_ACT_GELU) : activate_bf16(r[i], VA_ACT_GELU);
            break;
        case VA_ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = EXACT ? activate(r[i], VA_ACT_GELU_TANH) : activate_bf16(r[i], VA_ACT_GELU_TANH);
            break;
        case VA_ACT_RELU:
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = activate(r[i], VA_ACT_RELU);
            break;
        default: break;
    }
}

}  // namespace tok
