// va_tok_linear.hip -- the matrix product of the token operators: y = act(x w^T + bias) + res (va355.h va_tok_linear).
//
// The weights are the MFMA's A operand (its rows are output channels) and the tokens its B operand, so a lane's
// accumulator registers are consecutive channels of one token: the epilogue stores them as vectors.
#include "va_tok.h"

namespace {
using namespace tok;

// four consecutive channels n .. n + 3 of token m from the accumulator: scale, bias, activation, residual, store.
// vec: y, res rows are aligned for four values and n + 3 < N
struct Out {
    const float *wscale, *bias;
    const void* res;
    void* y;
    int64_t ldr, ldy;
    int32_t M, N, act, f32in, f32out, vec;
};

__device__ __forceinline__ void finish4(const Out& o, int m, int n, f32x4 v) {
    if (m >= o.M || n >= o.N) return;
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = n + i < o.N ? n + i : o.N - 1;
        float t = v[i];
        if (o.wscale) t *= o.wscale[c];
        if (o.bias) t += o.bias[c];
        r[i] = activate(t, o.act);
    }
    if (o.vec && n + 3 < o.N) {
        if (o.res) {
            if (o.f32in) {
                const f32x4 q = *(const f32x4*)((const float*)o.res + (int64_t)m * o.ldr + n);
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] += q[i];
            } else {
                const u32x2 q = *(const u32x2*)((const __bf16*)o.res + (int64_t)m * o.ldr + n);
                r[0] += bf_lo(q[0]), r[1] += bf_hi(q[0]), r[2] += bf_lo(q[1]), r[3] += bf_hi(q[1]);
            }
        }
        if (o.f32out)
            *(f32x4*)((float*)o.y + (int64_t)m * o.ldy + n) = (f32x4){r[0], r[1], r[2], r[3]};
        else
            *(u32x2*)((__bf16*)o.y + (int64_t)m * o.ldy + n) = (u32x2){pk_bf16(r[0], r[1]), pk_bf16(r[2], r[3])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n + i >= o.N) return;
        if (o.res)
            r[i] += o.f32in ? ((const float*)o.res)[(int64_t)m * o.ldr + n + i]
                            : (float)((const __bf16*)o.res)[(int64_t)m * o.ldr + n + i];
        if (o.f32out)
            ((float*)o.y)[(int64_t)m * o.ldy + n + i] = r[i];
        else
            ((__bf16*)o.y)[(int64_t)m * o.ldy + n + i] = (__bf16)r[i];
    }
}

enum Form { BF16, W8, F32 };

// ------------------------------------------------------------------ any shape, stride and alignment
// 64 channels x 64 tokens per workgroup, four waves of 32 x 32, K in steps of 32 through LDS; rows of 40 bf16 keep the
// fragment reads off each other's banks.  F32: three planes, six term products per fragment pair.
constexpr int GB = 64, GK = 32, GLD = GK + 8;

template <Form FORM>
__global__ __launch_bounds__(256) void linear_any(va_tok_linear_args a, Out o, int ntn, int xvec) {
    constexpr int T = FORM == F32 ? 3 : 1;
    __shared__ __align__(16) __bf16 ws[T][GB][GLD], xs[T][GB][GLD];
    const int tile = xcd_tile(blockIdx.x, gridDim.x);
    const int n0 = tile % ntn * GB, m0 = tile / ntn * GB;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, fr = lane & 15, fq = lane >> 4;
    const int wn = wid & 1, wm = wid >> 1;
    const int row = tid >> 2, ch = tid & 3;  // this thread's staged row and 8-value chunk
    const int m = m0 + row;
    f32x4 acc[2][2] = {};
    for (int k0 = 0; k0 < a.Kpad; k0 += GK) {
        const int k = k0 + 8 * ch;
        bf16x8 wt[T], xt[T];
        if constexpr (FORM == F32) {
            const bf16x8* p = (const bf16x8*)a.w + ((int64_t)(n0 + row) * (a.Kpad / 8) + k / 8) * 3;
#pragma unroll
            for (int t = 0; t < 3; ++t) wt[t] = p[t];
        } else if constexpr (FORM == W8) {
            const int c = k / 8, pos = (c & ~7) | ((c & 3) << 1) | ((c >> 2) & 1);
            wt[0] = e4m3x8(*(const uint2*)((const uint8_t*)a.w + (int64_t)(n0 + row) * a.Kpad + 8 * pos));
        } else {
            wt[0] = *(const bf16x8*)((const __bf16*)a.w + (int64_t)(n0 + row) * a.Kpad + k);
        }
        if constexpr (FORM == F32) {
            float x[8];
            const float* p = (const float*)a.x + (int64_t)m * a.ldx + k;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = m < a.M && k + e < a.K ? p[e] : 0.0f;
            split3(x, xt);
        } else {
            const __bf16* p = (const __bf16*)a.x + (int64_t)m * a.ldx + k;
            if (xvec && m < a.M && k + 8 <= a.K) {
                xt[0] = *(const bf16x8*)p;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) xt[0][e] = m < a.M && k + e < a.K ? p[e] : (__bf16)0.0f;
            }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < T; ++t) {
            *(bf16x8*)&ws[t][row][8 * ch] = wt[t];
            *(bf16x8*)&xs[t][row][8 * ch] = xt[t];
        }
        __syncthreads();
        bf16x8 fw[T][2], fx[T][2];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fw[t][i] = *(const bf16x8*)&ws[t][32 * wn + 16 * i + fr][8 * fq];
                fx[t][i] = *(const bf16x8*)&xs[t][32 * wm + 16 * i + fr][8 * fq];
            }
        constexpr int TA[6] = {0, 0, 1, 0, 1, 2}, TB[6] = {0, 1, 0, 2, 1, 0};
#pragma unroll
        for (int t = 0; t < (FORM == F32 ? 6 : 1); ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[TA[t]][i], fx[TB[t]][j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            finish4(o, m0 + 32 * wm + 16 * j + fr, n0 + 32 * wn + 16 * i + 4 * fq, acc[i][j]);
}

bool linear_ok(const va_tok_linear_args& a) {
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || !a.w || !a.y || (a.M > 0 && !a.x)) return false;
    if (a.dtype != VA_DTYPE_BF16 && a.dtype != VA_DTYPE_F32) return false;
    if ((a.w8 != 0 && a.w8 != 1) || (a.w8 && (a.dtype != VA_DTYPE_BF16 || !a.wscale)) || (!a.w8 && a.wscale)) return false;
    if (a.act < VA_ACT_NONE || a.act > VA_ACT_RELU) return false;
    if (a.Npad < a.N || a.Npad % 64 || a.Kpad < a.K || a.Kpad % 64 || ((uintptr_t)a.w & 15)) return false;
    if (a.ldx < a.K || a.ldy < a.N || (a.res && a.ldr < a.N)) return false;
    const uintptr_t e = a.dtype == VA_DTYPE_F32 ? 3 : 1, eo = a.dtype == VA_DTYPE_F32 || a.out_f32 ? 3 : 1;
    return !(((uintptr_t)a.x | (uintptr_t)a.res) & e) && !((uintptr_t)a.y & eo) &&
           !(((uintptr_t)a.bias | (uintptr_t)a.wscale) & 3);
}

}  // namespace

extern "C" int va_tok_linear(void* stream, const va_tok_linear_args* ap) {
    if (!ap || !linear_ok(*ap)) return VA_ERR_ARG;
    const va_tok_linear_args& a = *ap;
    if (a.M == 0) return VA_OK;
    const bool f32 = a.dtype == VA_DTYPE_F32;
    Out o = {a.wscale, a.bias, a.res, a.y, a.ldr, a.ldy, a.M, a.N, a.act, f32, f32 || a.out_f32, 0};
    o.vec = a.ldy % 4 == 0 && !((uintptr_t)a.y & (o.f32out ? 15 : 7)) &&
            (!a.res || (a.ldr % 4 == 0 && !((uintptr_t)a.res & (f32 ? 15 : 7))));
    const int64_t ntn = (a.N + GB - 1) / GB, tiles = ntn * ((a.M + GB - 1) / GB);
    if (tiles > INT32_MAX) return VA_ERR_RANGE;
    const int xvec = a.ldx % 8 == 0 && !((uintptr_t)a.x & 15);
    const dim3 grid((unsigned)tiles), block(256);
    hipStream_t st = (hipStream_t)stream;
    if (f32)
        hipLaunchKernelGGL(linear_any<F32>, grid, block, 0, st, a, o, (int)ntn, xvec);
    else if (a.w8)
        hipLaunchKernelGGL(linear_any<W8>, grid, block, 0, st, a, o, (int)ntn, xvec);
    else
        hipLaunchKernelGGL(linear_any<BF16>, grid, block, 0, st, a, o, (int)ntn, xvec);
    return hipGetLastError() == hipSuccess ? VA_OK : VA_ERR_HIP;
}
