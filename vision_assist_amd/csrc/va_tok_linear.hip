// va_tok_linear.hip -- the matrix product of the token operators: y = act(x w^T + bias) + res (va355.h va_tok_linear).
//
// The weights are the MFMA's A operand (its rows are output channels) and the tokens its B operand, so a lane's
// accumulator registers are consecutive channels of one token: the epilogue stores them as vectors.
//
// float: x = h + m + l exactly in three bf16 terms (so are the weights), and six of the nine term products are kept -- the
// three left out come to 2^-23 of a product's size at most -- so a product runs on the bf16 MFMA at a sixth of its rate, 245 TFLOP/s
// by the library's large bf16 product (1467), where the 32-bit MFMA reaches 154.  e4m3 weights: every e4m3 value is a bf16 value; the
// row's scale is applied to the sum.
#include <type_traits>

#include "va_dev.h"
#include "va_tok.h"

namespace {
using namespace tok;

// four consecutive channels n .. n + 3 of token m from the accumulator: scale, bias, activation, residual, store.
// vec: y and res rows are aligned for four values (1), for eight (2)
struct Out {
    const float *wscale, *bias;
    const void* res;
    void* y;
    int64_t ldr, ldy;
    int32_t M, N, act, vec;
};

template <bool FIN, bool FOUT>
__device__ __forceinline__ void finish4(const Out& o, int m, int n, f32x4 v) {
    if (m >= o.M || n >= o.N) return;
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = n + i < o.N ? n + i : o.N - 1;
        float t = v[i];
        if (o.wscale) t *= o.wscale[c];
        if (o.bias) t += o.bias[c];
        r[i] = t;
    }
    activate_n<FOUT>(r, o.act);
    if (o.vec && n + 3 < o.N) {
        if (o.res) {
            if (FIN) {
                const f32x4 q = *(const f32x4*)((const float*)o.res + (int64_t)m * o.ldr + n);
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] += q[i];
            } else {
                const u32x2 q = *(const u32x2*)((const __bf16*)o.res + (int64_t)m * o.ldr + n);
                r[0] += bf_lo(q[0]), r[1] += bf_hi(q[0]), r[2] += bf_lo(q[1]), r[3] += bf_hi(q[1]);
            }
        }
        if (FOUT)
            *(f32x4*)((float*)o.y + (int64_t)m * o.ldy + n) = (f32x4){r[0], r[1], r[2], r[3]};
        else
            *(u32x2*)((__bf16*)o.y + (int64_t)m * o.ldy + n) = (u32x2){pk_bf16(r[0], r[1]), pk_bf16(r[2], r[3])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n + i >= o.N) return;
        if (o.res)
            r[i] += FIN ? ((const float*)o.res)[(int64_t)m * o.ldr + n + i]
                            : (float)((const __bf16*)o.res)[(int64_t)m * o.ldr + n + i];
        if (FOUT)
            ((float*)o.y)[(int64_t)m * o.ldy + n + i] = r[i];
        else
            ((__bf16*)o.y)[(int64_t)m * o.ldy + n + i] = (__bf16)r[i];
    }
}

// types: bf16 or e4m3 weights with bf16 tensors, the same with a float result, all float
// Packed weights (va355.h): blocks of 32 channels x 32 of K, [Kpad / 32][Npad / 32][32 rows], a row 64 bytes of bf16 (32 of
// e4m3) -- the image that the kernels stage, so that staging is a linear copy.  Row r of a block is channel 16 (r / 4 % 2) +
// 4 (r / 8) + r % 4 of it: an MFMA then leaves a lane 16 consecutive channels in its registers.  Its pieces of 8 values lie in
// place p ^ (r / 4 % 4) (e4m3: p ^ (r / 8 % 4)): the lanes that an LDS read serves at a time (256 bytes: 16 rows' 16 bytes,
// 32 rows' 8) touch every bank once.  With an order that is so for 8 rows alone half of the LDS' cycles were conflicts.
__host__ __device__ constexpr int row_of(int ch) { return 8 * ((ch & 15) >> 2) + 4 * (ch >> 4) + (ch & 3); }

enum Form { BF16, W8, BF16F, W8F, F32 };
constexpr bool is8(Form f) { return f == W8 || f == W8F; }
constexpr bool fin(Form f) { return f == F32; }
constexpr bool fout(Form f) { return f >= BF16F; }

// ------------------------------------------------------------------ any shape, stride and alignment
// 64 channels x 64 tokens per workgroup, four waves of 32 x 32, K in steps of 32 through LDS; rows of 40 bf16 keep the
// fragment reads off each other's banks.  F32: three planes, six term products per fragment pair.
constexpr int GB = 64, GK = 32, GLD = GK + 8;

template <Form FF>
__global__ __launch_bounds__(256) void linear_any(va_tok_linear_args a, Out o, int ntn, int xvec) {
    constexpr int T = FF == F32 ? 3 : 1;
    __shared__ __align__(16) __bf16 ws[T][GB][GLD], xs[T][GB][GLD];
    const int tile = xcd_tile(blockIdx.x, gridDim.x);
    const int n0 = tile % ntn * GB, m0 = tile / ntn * GB;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, fr = lane & 15, fq = lane >> 4;
    const int wn = wid & 1, wm = wid >> 1;
    const int row = tid >> 2, kq = tid & 3;  // this thread's staged row and 8-value chunk
    const int m = m0 + row;
    f32x4 acc[2][2];
    bool far = false;
again:
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i / 2][i % 2] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < a.Kpad; k0 += GK) {
        const int k = k0 + 8 * kq;
        bf16x8 wt[T], xt[T];
        const int ch = n0 + row, r = row_of(ch & 31);
        const int64_t block = (int64_t)(k / 32) * (a.Npad / 32) + ch / 32;
        if constexpr (is8(FF)) {
            wt[0] = e4m3x8(*(const uint2*)((const uint8_t*)a.w + block * 1024 + r * 32 + 8 * ((k % 32 / 8) ^ ((r >> 3) & 3))));
        } else {
#pragma unroll
            for (int t = 0; t < T; ++t)
                wt[t] = *(const bf16x8*)((const __bf16*)a.w + (int64_t)t * a.Npad * a.Kpad + block * 1024 + r * 32 + 8 * ((k % 32 / 8) ^ ((r >> 2) & 3)));
        }
        if constexpr (FF == F32) {
            float x[8];
            const float* p = (const float*)a.x + (int64_t)m * a.ldx + k;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = m < a.M && k + e < a.K ? p[e] : 0.0f;
            if (far)
                split3_far(x, xt);
            else
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
            *(bf16x8*)&ws[t][row][8 * kq] = wt[t];
            *(bf16x8*)&xs[t][row][8 * kq] = xt[t];
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
        for (int t = 0; t < (FF == F32 ? 6 : 1); ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[TA[t]][i], fx[TB[t]][j], acc[i][j], 0, 0, 0);
    }
    if constexpr (FF == F32)  // (as in the tiles below: NaN where split3 does not take a value)
        if (!far && __syncthreads_or(acc[0][0][0] != acc[0][0][0] || acc[0][1][0] != acc[0][1][0])) {
            far = true;
            goto again;
        }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            finish4<fin(FF), fout(FF)>(o, m0 + 32 * wm + 16 * j + fr, n0 + 32 * wn + 16 * i + 4 * fq, acc[i][j]);
}

// the six term products that are kept of (h + m + l)(h + m + l)
constexpr int NTERM = 6, TERM_W[6] = {0, 0, 1, 0, 1, 2}, TERM_X[6] = {0, 1, 0, 2, 1, 0};

// Tile i of ntn x ntm in groups of G rows of token tiles, tokens fastest: the consecutive tiles that an XCD works on at a
// time form a block G high, so that each operand's rows come from beyond its L2 few times (G = 1 at 8192^3: 64 tiles of
// 256 x 128 in two rows fetched 528 KB a step, 937 TFLOP/s).
template <int G>
__device__ __forceinline__ void grouped_tile(int i, int ntn, int ntm, int* tn, int* tm) {
    const int grp = i / (G * ntn), gm = min(G, ntm - G * grp), in = i - G * grp * ntn;
    *tm = G * grp + in % gm;
    *tn = in / gm;
}

// ------------------------------------------------------------------ many tiles: LDS-DMA rings, counted waits
// 64 WN channels x 64 WM tokens per workgroup, four waves of 32 WN x 32 WM on v_mfma_f32_32x32x16_bf16, K in steps of 32.
// Weights go through a ring of NSW stages of a step; tokens in stages of whole 128-byte lines, two steps of bf16 or one of
// float (rows of 64 bytes would fetch each line twice).  A step is two slices of 16; the fragments of a slice are read
// while the MFMAs of the slice before run.  One barrier a step, after its first slice: by then every wave has read the
// whole step, so its stage is free and the weights of step t + NSW (after a token stage's last step: the tokens two stages
// on) are sent into it; and the wait before the barrier has retired what step t + 1 needs -- all but what the barrier
// before sent -- whose fragments are read next.
// KG = 2: two groups of four waves with rings of their own take the first and the second half of K, and the second's sums
// are added to the first's through LDS: two waves a SIMD where there is a workgroup for each CU at most.
// Float: a value that split3 does not take leaves NaN in its token's sums, all channels of them (0 x NaN too), so one sum of
// each token is looked at, and the tile is formed once more with split3_far if it is one, by a loop of its own (a test of
// every split value was 4 to 5 % of the time, split3_far in the loop itself 0 to 6 %).
// Two workgroups of 256 x 128 share a CU: the epilogue of one (activations: VALU, stores) runs beside the MFMAs of the
// other.  (One workgroup of 256 x 256 a CU, without that: 1222 TFLOP/s where this form had 1198 at 8192^3, but 334 us
// instead of 304 with GELU at 25600 x 1024 x 4096; deeper rings: no faster, and one workgroup a CU.)
// Bound by the MFMAs and the issue around them, on one GPU: 8192^3 in bf16 1157 TFLOP/s (the library's product: 1467); 25600 x
// 1024 x 4096 216 us, 995 TFLOP/s (the library's: 184 us), with bias and GELU 241 to 254 us, whose vector instructions the
// MFMAs of the other workgroup cover in part; with e4m3 weights, which both waves that read a fragment convert, 262 us, with
// GELU 302; float 1603 x 520 x 1000 with a residual 18.7 us: 208 workgroups, two waves a SIMD.
constexpr int LIN_OOB = 0x7ffffff0;      // an offset that a descriptor of that many bytes answers with zeros
constexpr int LIN_ROW = 1 << 21;         // longest rows in values: the offsets of 256 of them stay within 31 bits

__device__ __forceinline__ void dma16(const void* base, void* lds, int off, int uniform) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, LIN_OOB, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lvoid_t*)lds, 16, off, uniform, 0, 0);
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// eight consecutive channels of a token, through every type and alignment
template <bool FIN, bool FOUT>
__device__ __forceinline__ void finish8(const Out& o, int m, int n, float (&r)[8], const float (&scale)[8], const float (&bias)[8],
                                        const u32x4 (&res)[FIN ? 2 : 1]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __builtin_fmaf(r[i], scale[i], bias[i]);
    activate_n<FOUT>(r, o.act);
    if (o.vec == 2 && n + 7 < o.N) {
        if (o.res) {
            if constexpr (FIN) {
#pragma unroll
                for (int i = 0; i < 8; ++i) r[i] += __uint_as_float(res[i / 4][i % 4]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) r[2 * e] += bf_lo(res[0][e]), r[2 * e + 1] += bf_hi(res[0][e]);
            }
        }
        if (FOUT) {
            f32x4* y = (f32x4*)((float*)o.y + (int64_t)m * o.ldy + n);
            y[0] = (f32x4){r[0], r[1], r[2], r[3]}, y[1] = (f32x4){r[4], r[5], r[6], r[7]};
        } else {
            *(u32x4*)((__bf16*)o.y + (int64_t)m * o.ldy + n) =
                (u32x4){pk_bf16(r[0], r[1]), pk_bf16(r[2], r[3]), pk_bf16(r[4], r[5]), pk_bf16(r[6], r[7])};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (n + i >= o.N) return;
        const int64_t at = (int64_t)m * o.ldy + n + i;
        if (o.res) r[i] += FIN ? ((const float*)o.res)[(int64_t)m * o.ldr + n + i]
                                   : (float)((const __bf16*)o.res)[(int64_t)m * o.ldr + n + i];
        if (FOUT)
            ((float*)o.y)[at] = r[i];
        else
            ((__bf16*)o.y)[at] = (__bf16)r[i];
    }
}

// A wave's 32 WN channels x 32 WM tokens from n, m on: 32 tokens at a time through the wave's part of LDS, so that its
// stores are whole runs of a token's channels -- 4 WN lanes hold a token's channels, eight each, whose bias and scale are
// loaded once.  Register e of a block: channel 16 lh + e (the staged order of the weight rows).
template <Form FF, int WN, int WM>
__device__ __forceinline__ void store_tile(const Out& o, const f32x16 (&acc)[WN][WM], unsigned char* es, int m, int n, int lane) {
    constexpr int EROW = (32 * WN + 4) * 4, LR = 4 * WN, RI = 64 / LR;  // lanes of a token, tokens an iteration
    const int lc = lane & 31, lh = lane >> 5, er = lane / LR, ec = lane % LR * 8;
    float scale[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) scale[e] = 1.0f, bias[e] = 0.0f;
    if (is8(FF)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) scale[e] = o.wscale[min(n + ec + e, o.N - 1)];
    }
    if (o.bias) {
#pragma unroll
        for (int e = 0; e < 8; ++e) bias[e] = o.bias[min(n + ec + e, o.N - 1)];
    }
    // (waited for here: in the loops below the wait would be for the stores before it as well)
#pragma unroll
    for (int e = 0; e < 8; ++e) asm volatile("" ::"v"(scale[e]), "v"(bias[e]));
#pragma unroll
    for (int j = 0; j < WM; ++j) {
#pragma unroll
        for (int i = 0; i < WN; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *(f32x4*)(es + lc * EROW + (32 * i + 16 * lh + e) * 4) =
                    (f32x4){acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
        // the residuals of U iterations are on their way before the first store: res may be y, so no load passes a store
        constexpr int U = 32 / RI < 4 ? 32 / RI : 4, NR = fin(FF) ? 2 : 1;
#pragma unroll 1
        for (int it = 0; it < 32 / RI; it += U) {
            u32x4 res[U][NR];
            if (o.res && o.vec == 2 && n + ec + 7 < o.N) {
#pragma unroll
                for (int t = 0; t < U; ++t) {
                    const int64_t at = (int64_t)min(m + 32 * j + (it + t) * RI + er, o.M - 1) * o.ldr + n + ec;
#pragma unroll
                    for (int q = 0; q < NR; ++q) res[t][q] = *(const u32x4*)((const unsigned char*)o.res + at * (fin(FF) ? 4 : 2) + 16 * q);
                }
            }
#pragma unroll
            for (int t = 0; t < U; ++t) {
                const int row = (it + t) * RI + er, mr = m + 32 * j + row;
                const f32x4 u = *(const f32x4*)(es + row * EROW + ec * 4), v = *(const f32x4*)(es + row * EROW + ec * 4 + 16);
                float r[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
                if (mr < o.M && n + ec < o.N) finish8<fin(FF), fout(FF)>(o, mr, n + ec, r, scale, bias, res[t]);
            }
        }
    }
}

template <Form F, int WN, int WM, int KG>
struct TileCfg {
    static constexpr int BN = 64 * WN, BM = 64 * WM, T = F == F32 ? 3 : 1;
    static constexpr int WROW = is8(F) ? 32 : 64, XP = F == F32 ? 1 : 2;        // bytes of a weight row; steps of a token stage
    static constexpr int WPL = BN * WROW, WB = T * WPL, XB = BM * 128;          // bytes of a plane, of the stages
    static constexpr int NSW = 3 * WB + (F == F32 ? 3 : 2) * XB <= 80 * 1024 ? 3 : 2, NSX = F == F32 ? NSW : 2;
    static constexpr int DW = WB / 4096, DX = XB / 4096;                        // DMAs of a wave
    static constexpr int EROW = (32 * WN + 4) * 4, EPI = 4 * 32 * EROW;         // the epilogue's blocks (store_tile)
    static constexpr int RING = NSW * WB + NSX * XB, LDS = KG * (RING > EPI ? RING : EPI);
    static_assert(WB % 4096 == 0 && XB % 4096 == 0 && WPL % 1024 == 0 && LDS <= KG * 80 * 1024, "eight waves a CU");
    static_assert(KG == 1 || 4 * WN * WM * 16 * 64 * 4 <= LDS / 2, "");
};

template <Form F, int WN, int WM, int KG>
__global__ __launch_bounds__((256 * KG), 2) void linear_tile(va_tok_linear_args a, Out o, int ntn, int ntm) {
    using C = TileCfg<F, WN, WM, KG>;
    constexpr int T = C::T, XE = F == F32 ? 4 : 2;
    extern __shared__ __align__(16) unsigned char lds[];  // [KG]: [NSW] weights, [NSX] tokens
    int tn, tm;
    grouped_tile<8>(xcd_tile(blockIdx.x, gridDim.x), ntn, ntm, &tn, &tm);
    const int n0 = tn * C::BN, m0 = tm * C::BM;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grp = wave >> 2, wid = wave & 3, lane = threadIdx.x & 63, lc = lane & 31, lh = lane >> 5;
    const int wn = wid & 1, wm = wid >> 1;
    const int nk = 2 * ((a.K + 63) / 64), nl = KG == 1 ? nk : 2 * ((nk / 2 + KG - 1) / KG), k0 = grp * nl;  // steps: all, a group's, from
    unsigned char* sm = lds + grp * (C::LDS / KG);
    // weights: DMA d of a stage's plane copies its bytes [1024 d, 1024 d + 1024); blocks from channel Npad on are not there
    const unsigned char* wb = (const unsigned char*)a.w + (int64_t)(n0 / 32) * 32 * C::WROW;
    const int64_t wstep = (int64_t)a.Npad * C::WROW, plane = wstep * (a.Kpad / 32);
    const int wend = min(a.Npad - n0, C::BN) * C::WROW;
    auto issue_w = [&](int t) {
        unsigned char* to = sm + t % C::NSW * C::WB;
        const unsigned char* from = wb + min(t + k0, nk - 1) * wstep;
        const bool on = t < nl && t + k0 < nk;
#pragma unroll
        for (int j = 0; j < C::DW; ++j) {
            const int d = (wid * C::DW + j) * 1024, in = d % C::WPL;  // uniform
            dma16(from + (T > 1 ? d / C::WPL * plane : 0), to + d, on && in < wend ? lane * 16 : LIN_OOB, in);
        }
    };
    // tokens: DMA j takes rows 8 (wid DX + j) .. + 7, lane l row l / 8, place l % 8: piece place ^ (row / 2 % 8), so rows of
    // odd DMAs (4 more) have the other half of the pieces
    static_assert(C::DX % 2 == 0, "");
    const int l8 = lane >> 3, piece = (lane & 7) ^ (l8 >> 1);
    const unsigned char* xb = (const unsigned char*)a.x + (int64_t)m0 * a.ldx * XE;
    const int xrow = 8 * wid * C::DX + l8, xmore = a.M - m0 - xrow;
    const int xoff[2] = {(int)(xrow * a.ldx) * XE + 16 * piece, (int)(xrow * a.ldx) * XE + 16 * (piece ^ 4)};
    auto issue_x = [&](int st) {
        unsigned char* to = sm + C::NSW * C::WB + st % C::NSX * C::XB + wid * C::DX * 1024;
        const int g = st + k0 / C::XP;
        const bool in[2] = {g * (128 / XE) + piece * (16 / XE) < a.K, g * (128 / XE) + (piece ^ 4) * (16 / XE) < a.K};
#pragma unroll
        for (int j = 0; j < C::DX; ++j)
            dma16(xb, to + j * 1024, in[j & 1] && 8 * j < xmore ? xoff[j & 1] : LIN_OOB, (int)(8 * j * a.ldx) * XE + g * 128);
    };
    f32x16 acc[WN][WM];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < WN; ++i)
#pragma unroll
            for (int j = 0; j < WM; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    };
    struct Frag {
        bf16x8 w[WN][T], x[WM][T];
        f32x4 raw[F == F32 ? WM : 1][2];
    };
    auto read = [&](Frag& f, int t, int ks) {
        const unsigned char* ws = sm + t % C::NSW * C::WB;
        const unsigned char* xs = sm + C::NSW * C::WB + t / C::XP % C::NSX * C::XB;
#pragma unroll
        for (int i = 0; i < WN; ++i) {
            const unsigned char* wr = ws + (32 * (wn * WN + i) + lc) * C::WROW;
            if constexpr (is8(F)) {
                f.w[i][0] = e4m3x8(*(const uint2*)(wr + 8 * ((2 * ks + lh) ^ (lc >> 3))));
            } else {
#pragma unroll
                for (int p = 0; p < T; ++p) f.w[i][p] = *(const bf16x8*)(wr + p * C::WPL + 16 * ((2 * ks + lh) ^ ((lc >> 2) & 3)));
            }
        }
#pragma unroll
        for (int j = 0; j < WM; ++j) {
            const unsigned char* xr = xs + (32 * (wm * WM + j) + lc) * 128;
            if constexpr (F == F32) {
                const int p = 2 * (2 * ks + lh);
                const int q = (lc >> 1) & 7;
                f.raw[j][0] = *(const f32x4*)(xr + 16 * (p ^ q)), f.raw[j][1] = *(const f32x4*)(xr + 16 * ((p + 1) ^ q));
            } else {
                f.x[j][0] = *(const bf16x8*)(xr + 16 * ((4 * (t & 1) + 2 * ks + lh) ^ ((lc >> 1) & 7)));
            }
        }
    };
    auto mma = [&](const Frag& f) {
#pragma unroll
        for (int t = 0; t < (T > 1 ? NTERM : 1); ++t)
#pragma unroll
            for (int i = 0; i < WN; ++i)
#pragma unroll
                for (int j = 0; j < WM; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.w[i][T > 1 ? TERM_W[t] : 0], f.x[j][T > 1 ? TERM_X[t] : 0],
                                                                        acc[i][j], 0, 0, 0);
    };
    auto split = [&](Frag& f) {  // F32: the tokens' terms
        if constexpr (F == F32) {
#pragma unroll
            for (int j = 0; j < WM; ++j) {
                const f32x4 u = f.raw[j][0], v = f.raw[j][1];
                const float e[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
                split3(e, f.x[j]);
            }
        }
    };
    // the next slice's fragments are read before this slice's MFMAs; F32: and split beside the second half of them
    auto slice = [&](Frag& next, const Frag& f) {
        if constexpr (F == F32) {
            mma(f);
            split(next);
            constexpr int NM = NTERM * WN * WM, NV = 52 * WM;
            __builtin_amdgcn_sched_group_barrier(0x100, WN * T + 2 * WM, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, NM / 2, 0);
#pragma unroll
            for (int i = 0; i < NM - NM / 2; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x002, NV / (NM - NM / 2), 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            }
        } else {
            __builtin_amdgcn_sched_barrier(0);
            mma(f);
        }
    };
    clear();
    // in the order in which the steps need them; past the last step they run on, on offsets out of range
    issue_x(0);
    issue_w(0);
    issue_w(1);
    issue_x(1);
    if constexpr (C::NSW == 3) {
        issue_w(2);
        if constexpr (C::XP == 1) issue_x(2);
    }
    wait_vm<C::NSW == 3 ? 2 * C::DW + C::DX * (C::XP == 1 ? 2 : 1) : C::DW + C::DX>();
    asm volatile("s_barrier" ::: "memory");
    Frag f0, f1;
    read(f0, 0, 0);
    split(f0);
    for (int t2 = 0; t2 < nl; t2 += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int t = t2 + u;
            read(f1, t, 1);
            slice(f1, f0);
            __builtin_amdgcn_sched_barrier(0);
            constexpr int XS = C::XP == 1 ? C::DX : 0;
            if (u == 0)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(C::NSW == 3 ? C::DW + C::DX : 0) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(C::NSW == 3 ? C::DW + XS : 0) : "memory");
            issue_w(t + C::NSW);
            if (C::XP == 1 || u == 1) issue_x(t / C::XP + C::NSX);
            read(f0, t + 1, 0);
            slice(f0, f1);
            if constexpr (F == F32) __builtin_amdgcn_sched_barrier(0);
        }
    }
    wait_vm<0>();
    if constexpr (F == F32) {
        __shared__ int nans[4 * KG];
        bool nan = false;
#pragma unroll
        for (int j = 0; j < WM; ++j) nan |= acc[0][j][0] != acc[0][j][0];
        nan = __any(nan);
        if (lane == 0) nans[wave] = nan;
        __syncthreads();
        bool far = false;
#pragma unroll
        for (int i = 0; i < 4 * KG; ++i) far |= nans[i] != 0;
        if (far) {  // (the whole workgroup, step by step)
            clear();
#pragma unroll 1
            for (int t = 0; t < nl; ++t) {
                issue_w(t);
                issue_x(t);
                wait_vm<0>();
                __syncthreads();
#pragma unroll 1
                for (int ks = 0; ks < 2; ++ks) {
                    read(f0, t, ks);
#pragma unroll
                    for (int j = 0; j < WM; ++j) {
                        const f32x4 u = f0.raw[j][0], v = f0.raw[j][1];
                        const float e[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
                        split3_far(e, f0.x[j]);
                    }
                    mma(f0);
                }
                __syncthreads();
            }
        }
    } else {
        __syncthreads();
    }
    if constexpr (KG == 2) {  // the second group's sums into the first's
        f32x4* part = (f32x4*)(lds + C::LDS / 2) + wid * WN * WM * 4 * 64 + lane;
        if (grp) {
#pragma unroll
            for (int i = 0; i < WN; ++i)
#pragma unroll
                for (int j = 0; j < WM; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        part[((i * WM + j) * 4 + e) * 64] =
                            (f32x4){acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
        }
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int i = 0; i < WN; ++i)
#pragma unroll
            for (int j = 0; j < WM; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f32x4 v = part[((i * WM + j) * 4 + e) * 64];
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[i][j][4 * e + q] += v[q];
                }
    }
    store_tile<F, WN, WM>(o, acc, sm + wid * 32 * C::EROW, m0 + 32 * wm * WM, n0 + 32 * wn * WN, lane);
}

// ------------------------------------------------------------------ few tiles: K over the waves of a workgroup
// 16 channels x 16 MB tokens per workgroup; its eight waves take every eighth step of 128 bytes of the tokens' rows, each
// through two slots of its own in LDS and without a barrier, and their sums are joined in LDS in the waves' order.
// v_mfma_f32_16x16x32_bf16.
// 32 x 4096 x 4096 over 24 sets of weights: bf16 11.0 us, e4m3 9.3; x 16384: 36.2 and 30.6 us.  bf16 is bound by the weights'
// bytes, 3.7 TB/s; e4m3, at 2.2 TB/s of weights, by the tokens: 16 channels are 64 KB of e4m3 weights and read 256 KB of
// tokens through L2 and LDS, so half the bytes saves 15 % of the time.  One token, 1024 x 4096: 4.3.  Float weights are 6
// bytes a value: 32 x 4096 x 4096 22 us, 4.6 TB/s of them.
// The tokens come by LDS-DMA, eight lanes to a row's 128 bytes: loaded straight into the fragments neighbouring lanes held
// different rows, so that each lane's 16 bytes was a request of its own, and the tokens, not the weights, took the time
// (12.9, 14.1; 49.0 and 52.9 us).  Three or four slots: 1 to 9 us slower where workgroups queue, as fewer fit a CU.
template <Form F, int MB>
struct FewCfg {
    static constexpr int NW = 8, XE = F == F32 ? 4 : 2, KS = 128 / XE;  // waves; K of a step
    static constexpr int NS = 2;                                        // steps in LDS
    static constexpr int DX = 2 * MB, DW = is8(F) ? 1 : F == F32 ? 3 : 2;  // loads of a step: tokens', weights'
    static constexpr int XB = DX * 1024, LDS = NW * NS * XB;
};
template <Form F, int MB>
__global__ __launch_bounds__(512) void linear_few(va_tok_linear_args a, Out o, int ntn) {
    using C = FewCfg<F, MB>;
    constexpr int T = F == F32 ? 3 : 1, NW = C::NW, XE = C::XE, NS = C::NS;
    extern __shared__ __align__(16) unsigned char sm[];  // a wave: [NS][16 MB tokens][128]; then its sums
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fq = lane >> 4;
    const int n0 = blockIdx.x % ntn * 16, m0 = blockIdx.x / ntn * 16 * MB;
    const int nk = (a.K + C::KS - 1) / C::KS, count = (nk - wid + NW - 1) / NW;  // steps wid, wid + NW, ... are this wave's
    const int64_t wrow = (n0 / 32) * 32 + row_of((n0 & 16) + fr);                // this lane's weight row among a step's
    unsigned char* mine = sm + wid * NS * C::XB;
    f32x4 acc[MB];
    auto clear = [&]() {
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    };
    u32x4 w[NS][C::DW];
    // DMA j takes rows 8 j .. 8 j + 7, lane l row l / 8, place l % 8: piece place ^ (row / 2 % 8)
    const int l8 = lane >> 3, piece = (lane & 7) ^ (l8 >> 1), xmore = a.M - m0 - l8;
    const unsigned char* xb = (const unsigned char*)a.x + (int64_t)m0 * a.ldx * XE;
    const int xoff[2] = {(int)(l8 * a.ldx) * XE + 16 * piece, (int)(l8 * a.ldx) * XE + 16 * (piece ^ 4)};
    auto issue = [&](int i, int s) {  // (steps past the last one: no tokens, and the last one's weights, which no product uses)
        const int kb = wid + i * NW, kw = min(kb, nk - 1);
        if constexpr (is8(F)) {  // one 16-byte piece: 16 of K
            w[s][0] = *(const u32x4*)((const uint8_t*)a.w + ((int64_t)(2 * kw + fq / 2) * (a.Npad / 32)) * 1024 + wrow * 32 +
                                      16 * ((fq & 1) ^ ((wrow >> 4) & 1)));
        } else if constexpr (F == F32) {
#pragma unroll
            for (int t = 0; t < T; ++t)
                w[s][t] = *(const u32x4*)((const __bf16*)a.w + (int64_t)t * a.Npad * a.Kpad + (int64_t)kw * (a.Npad / 32) * 1024 +
                                          wrow * 32 + 8 * (fq ^ ((wrow >> 2) & 3)));
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                w[s][h] = *(const u32x4*)((const __bf16*)a.w + (int64_t)(2 * kw + h) * (a.Npad / 32) * 1024 + wrow * 32 +
                                          8 * (fq ^ ((wrow >> 2) & 3)));
        }
        const int k = kb * C::KS;
        const bool in[2] = {k + piece * (16 / XE) < a.K, k + (piece ^ 4) * (16 / XE) < a.K};
#pragma unroll
        for (int j = 0; j < C::DX; ++j)
            dma16(xb, mine + s * C::XB + j * 1024, in[j & 1] && 8 * j < xmore ? xoff[j & 1] : LIN_OOB,
                  (int)(8 * j * a.ldx) * XE + min(kb, nk) * 128);
    };
    const int turn = (fr >> 1) & 7;
    auto mma = [&](int s, auto far) {  // (far: with split3_far)
        const unsigned char* xs = mine + s * C::XB + fr * 128;
        if constexpr (F == F32) {
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                const f32x4 u = *(const f32x4*)(xs + j * 2048 + 16 * ((2 * fq) ^ turn));
                const f32x4 v = *(const f32x4*)(xs + j * 2048 + 16 * ((2 * fq + 1) ^ turn));
                const float e[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
                bf16x8 x[T];
                if constexpr (decltype(far)::value)
                    split3_far(e, x);
                else
                    split3(e, x);
#pragma unroll
                for (int t = 0; t < NTERM; ++t)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16((bf16x8)w[s][TERM_W[t]], x[TERM_X[t]], acc[j], 0, 0, 0);
            }
        } else {
            u32x4 r = w[s][0];
            if (is8(F) && (wrow & 8)) r = (u32x4){r[2], r[3], r[0], r[1]};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                bf16x8 wh;
                if constexpr (is8(F))
                    wh = e4m3x8(make_uint2(r[2 * h], r[2 * h + 1]));
                else
                    wh = (bf16x8)w[s][h];
                const int pc = is8(F) ? 2 * fq + h : 4 * h + fq;
#pragma unroll
                for (int j = 0; j < MB; ++j)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wh, *(const bf16x8*)(xs + j * 2048 + 16 * (pc ^ turn)), acc[j], 0, 0, 0);
            }
        }
    };
    clear();
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) issue(s, s);
    int i = 0;
    for (; i + NS <= count; i += NS) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            // the slot that is filled next was read in the step before: those reads are done
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            issue(i + s + NS - 1, (s + NS - 1) % NS);
            wait_vm<(NS - 1) * (C::DX + C::DW)>();
            mma(s, std::false_type());
        }
    }
    wait_vm<0>();
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
        if (i + s < count) mma(s, std::false_type());
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (F == F32) {  // (as in the tiles: NaN where split3 does not take a value)
        bool nan = false;
#pragma unroll
        for (int j = 0; j < MB; ++j) nan |= acc[j][0] != acc[j][0];
        if (__any(nan)) {
            clear();
#pragma unroll 1
            for (i = 0; i < count; ++i) {
                issue(i, 0);
                wait_vm<0>();
                mma(0, std::true_type());
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        }
    }
    f32x4* part = (f32x4*)mine;
#pragma unroll
    for (int j = 0; j < MB; ++j) part[j * 64 + lane] = acc[j];
    __syncthreads();
    for (int i = threadIdx.x; i < MB * 64; i += 64 * NW) {
        const int j = i / 64;
        f32x4 v = *(const f32x4*)(sm + i * 16);
#pragma unroll
        for (int q = 1; q < NW; ++q) v += *(const f32x4*)(sm + q * NS * C::XB + i * 16);
        finish4<fin(F), fout(F)>(o, m0 + 16 * j + fr, n0 + 4 * fq, v);
    }
}

bool linear_ok(const va_tok_linear_args& a) {
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || !a.w || !a.y || (a.M > 0 && !a.x)) return false;
    if (a.M > SIDE_MAX || a.Npad > SIDE_MAX || a.Kpad > SIDE_MAX) return false;
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

namespace {
template <Form F, int WN, int WM, int KG>
hipError_t go_tile(const va_tok_linear_args& a, const Out& o, hipStream_t st) {
    using C = TileCfg<F, WN, WM, KG>;
    constexpr int lds = C::LDS;
    const int ntn = (a.N + C::BN - 1) / C::BN, ntm = (a.M + C::BM - 1) / C::BM;
    if (!grid_ok(ntn, ntm, 256 * KG)) return hipErrorInvalidConfiguration;
    if (hipError_t e = big_lds<linear_tile<F, WN, WM, KG>, lds>()) return e;
    hipLaunchKernelGGL((linear_tile<F, WN, WM, KG>), dim3((unsigned)(ntn * ntm)), dim3(256 * KG), lds, st, a, o, ntn, ntm);
    return hipGetLastError();
}

template <Form F, int MB>
hipError_t go_few(const va_tok_linear_args& a, const Out& o, hipStream_t st) {
    const int ntn = (a.N + 15) / 16, ntm = (a.M + 16 * MB - 1) / (16 * MB);
    if (!grid_ok(ntn, ntm, 512)) return hipErrorInvalidConfiguration;
    constexpr int lds = FewCfg<F, MB>::LDS;
    if (hipError_t e = big_lds<linear_few<F, MB>, lds>()) return e;
    hipLaunchKernelGGL((linear_few<F, MB>), dim3((unsigned)(ntn * ntm)), dim3(512), lds, st, a, o, ntn);
    return hipGetLastError();
}

template <Form F>
hipError_t go_any(const va_tok_linear_args& a, const Out& o, hipStream_t st, int xvec) {
    const int ntn = (a.N + GB - 1) / GB, ntm = (a.M + GB - 1) / GB;
    if (!grid_ok(ntn, ntm, 256)) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL(linear_any<F>, dim3((unsigned)(ntn * ntm)), dim3(256), 0, st, a, o, ntn, xvec);
    return hipGetLastError();
}

template <Form F>
int form_of(const va_tok_linear_args& a) {
    constexpr int E = F == F32 ? 4 : 8;
    if (a.K % E || a.ldx % E || ((uintptr_t)a.x & 15) || a.ldx > LIN_ROW || a.Kpad > LIN_ROW) return VA_TOK_LINEAR_ANY;
    const int64_t t64 = (int64_t)((a.N + 63) / 64) * ((a.M + 63) / 64);
    // Measured (us, graph replays, K 1024; few | tiles): 112 tiles of 64 x 64: bf16 8.5 | 10.4, e4m3 8.7 | 16.0, float
    // 16.2 | 23.3; 128: 8.6 | 10.2, 8.9 | 16.1, 17.3 | 23.4; 208: 15.4 | 10.6, 15.8 | 16.4, 31.1 | 24.7; 256: 16.1 | 10.7,
    // 16.2 | 16.3, 31.7 | 25.5
    if (a.M <= 64 || t64 <= (is8(F) ? 256 : 128)) return VA_TOK_LINEAR_FEW;
    // Tiles of 128 x 64 | of 256 x 128, by the number of large ones: bf16 208 25.2 | 25.5, 400 42.0 | 37.4; e4m3 208
    // 28.9 | 33.4, 400 50.1 | 44.5.
    // Up to 256 tiles of 128 x 64, a workgroup a CU: one group of four waves | K halved between two, by the number of 64 x 64
    // (K 1024): float 256 24.3 | 23.5, 400 30.9 | 26.5, 448 31.7 | 27.8, 832 51.9 | 56.4; e4m3 400 16.6 |
    // 13.1, 448 16.6 | 13.1, 800 19.2 | 19.0; bf16, whose steps are short, 400 11.1 | 10.6, at K 520 8.2 | 8.5: one group.
    if constexpr (F != F32) {
        const int64_t big = (int64_t)((a.N + 255) / 256) * ((a.M + 127) / 128);
        if (big >= (is8(F) ? 320 : 224)) return VA_TOK_LINEAR_LARGE;
    }
    return (F == F32 || is8(F)) && t64 <= 512 ? VA_TOK_LINEAR_TILE_2K : VA_TOK_LINEAR_TILE;
}

template <Form F>
hipError_t go(const va_tok_linear_args& a, const Out& o, hipStream_t st) {
    switch (form_of<F>(a)) {
        case VA_TOK_LINEAR_FEW:
            return a.M <= 16 ? go_few<F, 1>(a, o, st) : a.M <= 32 ? go_few<F, 2>(a, o, st) : go_few<F, 4>(a, o, st);
        case VA_TOK_LINEAR_TILE: return go_tile<F, 2, 1, 1>(a, o, st);
        case VA_TOK_LINEAR_TILE_2K:
            if constexpr (F == F32 || is8(F)) return go_tile<F, 2, 1, 2>(a, o, st);
            break;
        case VA_TOK_LINEAR_LARGE:
            if constexpr (F != F32) return go_tile<F, 4, 2, 1>(a, o, st);
            break;
    }
    return go_any<F>(a, o, st, a.ldx % 8 == 0 && !((uintptr_t)a.x & 15));
}
}  // namespace

extern "C" int va_tok_linear(void* stream, const va_tok_linear_args* ap) {
    if (!ap || !linear_ok(*ap)) return VA_ERR_ARG;
    const va_tok_linear_args& a = *ap;
    if (a.M == 0) return VA_OK;
    const bool f32 = a.dtype == VA_DTYPE_F32;
    const bool f32out = f32 || a.out_f32;
    Out o = {a.wscale, a.bias, a.res, a.y, a.ldr, a.ldy, a.M, a.N, a.act, 0};
    // stores of 4 channels (1), of 8 (2)
    const auto rows = [&](int n) {
        const int eo = f32out ? 4 : 2, ei = f32 ? 4 : 2, bo = n * eo < 16 ? n * eo : 16, bi = n * ei < 16 ? n * ei : 16;
        return a.ldy * eo % bo == 0 && !((uintptr_t)a.y & (uintptr_t)(bo - 1)) &&
               (!a.res || (a.ldr * ei % bi == 0 && !((uintptr_t)a.res & (uintptr_t)(bi - 1))));
    };
    o.vec = rows(8) ? 2 : rows(4) ? 1 : 0;
    hipStream_t st = (hipStream_t)stream;
    const hipError_t e = f32         ? go<F32>(a, o, st)
                         : a.out_f32 ? (a.w8 ? go<W8F>(a, o, st) : go<BF16F>(a, o, st))
                                     : (a.w8 ? go<W8>(a, o, st) : go<BF16>(a, o, st));
    return e == hipSuccess ? VA_OK : e == hipErrorInvalidConfiguration ? VA_ERR_RANGE : VA_ERR_HIP;
}

extern "C" int va_tok_linear_form(const va_tok_linear_args* ap) {
    if (!ap || !linear_ok(*ap)) return VA_ERR_ARG;
    const va_tok_linear_args& a = *ap;
    if (a.dtype == VA_DTYPE_F32) return form_of<F32>(a);
    return a.w8 ? form_of<W8>(a) : form_of<BF16>(a);
}
