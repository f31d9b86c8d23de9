// va_tok_attn.hip -- attention with frames, a sliding window and sinks over a stream's cache (va355.h va_tok_attn).
//
// The G query heads of a key head and the positions are one list of rows, row = position * G + head, so one staged tile
// of keys and values serves all of them and the rows of a workgroup span few positions.  A wave holds 32 rows as MFMA
// columns: S^T = K Q^T leaves a lane the scores of ONE row (its lane & 31), so maximum and sum are in-lane plus one
// exchange with lane ^ 32, and O^T = V^T P^T takes those registers as its B operand without any exchange: the sum over
// keys may run in any order, so V^T is read in the order in which the scores lie in the registers.
//   bf16: v_mfma_f32_32x32x16_bf16, V^T by the transposing LDS read (16 lanes x 8 bytes: 4 keys x 16 columns)
//   f32:  v_mfma_f32_32x32x2_f32 (exact products), V^T by plain 4-byte reads
// One pass over the keys with the running maximum and sum of the softmax (base 2: the scale is folded with log2 e).
#include <math.h>

#include "va_tok.h"

namespace {
using namespace tok;

// keys that any row of a position sees: [0, sinks) and [low, top) in positions
struct Span {
    int low, top;
};

struct AttnSeq {  // one sequence's lengths, clamped to what the call holds
    int ql, kv, first;  // queries, cached positions, position of query 0
    int held;           // oldest position behind the sinks that no later one has overwritten
};

__device__ __forceinline__ AttnSeq attn_seq(const va_tok_attn_args& a, int b) {
    AttnSeq q;
    q.ql = a.q_len ? min(max(a.q_len[b], 0), a.S) : a.S;
    q.kv = a.kv_len && a.slots ? max(a.kv_len[b], 0) : a.slots;
    q.first = q.kv - q.ql;
    q.held = max(a.sinks, q.kv - (a.slots - a.sinks));
    return q;
}

// visible positions of the query at position i: [0, min(sinks, top)) and [low, top), low >= sinks; nothing for i < 0
__device__ __forceinline__ Span attn_span(const va_tok_attn_args& a, const AttnSeq& q, int i) {
    if (i < 0) return {a.sinks, 0};
    int64_t e = 0x7fffffff;
    if (a.frame) e = ((int64_t)(i / a.frame) + 1) * a.frame;
    int low = q.held;
    if (a.window && e - a.window > low) low = (int)min(e - a.window, (int64_t)0x7fffffff);
    return {low, (int)min(e, (int64_t)q.kv)};
}

template <typename T>
struct Tr;
template <>
struct Tr<__bf16> {
    static constexpr int VE = 8;   // values of a 16-byte piece
    static constexpr int KT = 64;  // keys of a tile
};
template <>
struct Tr<float> {
    static constexpr int VE = 4;
    static constexpr int KT = 32;
};

// LDS image of a tile: KT rows of CS 16-byte pieces, piece c of row r in place c ^ swz(r).  K is read by 8 lanes of
// consecutive rows at one piece, V by 4 rows at 4 pieces: both spread over the banks.
template <int CS>
__device__ __forceinline__ int swz(int r) {
    if constexpr (CS >= 16)
        return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (CS == 8)
        return ((r & 1) << 2) | ((r >> 1) & 3);
    else
        return (r >> 1) & 3;
}

// Tile walk: keys [t0, t0 + KT) of [lo, hi), positions -> slots
__device__ __forceinline__ int slot_of(const va_tok_attn_args& a, int p) {
    if (p < a.slots) return p;
    return a.sinks + (p - a.sinks) % (a.slots - a.sinks);
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_kernel(va_tok_attn_args a, int ntiles) {
    constexpr int VE = Tr<T>::VE, KT = Tr<T>::KT;
    constexpr bool BF = sizeof(T) == 2;
    constexpr int NC = DP / VE;                                       // pieces of a row
    constexpr int CS = NC <= 4 ? 4 : NC <= 8 ? 8 : NC <= 16 ? 16 : 32;  // ... as laid out (a power of two)
    constexpr int KB = KT / 32, NV = DP / 32;
    __shared__ __align__(16) unsigned char ks[KT * CS * 16], vs[KT * CS * 16];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, lc = lane & 31, lh = lane >> 5;
    const int G = a.Hq / a.Hk;
    int bid = blockIdx.x;
    const int tile = bid % ntiles;
    bid /= ntiles;
    const int hk = bid % a.Hk, b = bid / a.Hk;
    const AttnSeq sq = attn_seq(a, b);
    const int rows = sq.ql * G, r0 = tile * 128;
    if (r0 >= rows) return;
    // this lane's row
    const int row = r0 + 32 * wid + lc, s = row / G, g = row - s * G;
    const bool there = row < rows;
    const Span sp = there ? attn_span(a, sq, sq.first + s) : Span{a.sinks, 0};
    // the workgroup's keys: spans grow with the position
    const int s0 = r0 / G, s1 = (min(r0 + 128, rows) - 1) / G;
    const Span w0 = attn_span(a, sq, max(sq.first + s0, 0)), w1 = attn_span(a, sq, sq.first + s1);
    const int top = w1.top, low = max(w0.low, a.sinks), ntop = min(a.sinks, top);

    // Q^T fragments
    const T* qp = (const T*)a.q + b * a.q_sb + s * a.q_ss + (int64_t)(hk * G + g) * a.q_sh;
    u32x4 qf[DP / (2 * VE)];
#pragma unroll
    for (int c = 0; c < DP / (2 * VE); ++c) {
        const int d = (2 * c + lh) * VE;
        qf[c] = there && d < a.D ? *(const u32x4*)(qp + d) : (u32x4){0, 0, 0, 0};
    }
    const float cexp = a.scale * 1.4426950408889634f;
    float mx = -INFINITY, sum = 0.0f;
    f32x16 acc[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[v][i] = 0.0f;

    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    for (int part = 0; part < 2; ++part) {
        const int beg = part ? low : 0, end = part ? top : ntop;
        for (int t0 = beg; t0 < end; t0 += KT) {
            __syncthreads();
            for (int i = tid; i < KT * NC; i += 256) {
                const int r = i / NC, c = i % NC, p = t0 + r;
                const int slot = p < end ? slot_of(a, p) : 0;
                const bool kin = p < end && c * VE < a.D, vin = p < end && c * VE < a.Dv;
                const int at = (r * CS + (c ^ swz<CS>(r))) * 16;
                *(u32x4*)(ks + at) = kin ? *(const u32x4*)(kb + slot * a.k_ss + c * VE) : (u32x4){0, 0, 0, 0};
                *(u32x4*)(vs + at) = vin ? *(const u32x4*)(vb + slot * a.v_ss + c * VE) : (u32x4){0, 0, 0, 0};
            }
            __syncthreads();
            f32x16 sc[KB];
#pragma unroll
            for (int kb_ = 0; kb_ < KB; ++kb_) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[kb_][i] = 0.0f;
                const int r = 32 * kb_ + lc;
#pragma unroll
                for (int c = 0; c < NC / 2; ++c) {
                    const u32x4 kf = *(const u32x4*)(ks + (r * CS + ((2 * c + lh) ^ swz<CS>(r))) * 16);
                    if constexpr (BF) {
                        sc[kb_] = __builtin_amdgcn_mfma_f32_32x32x16_bf16((bf16x8)kf, (bf16x8)qf[c], sc[kb_], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            sc[kb_] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kf[e]), __uint_as_float(qf[c][e]),
                                                                          sc[kb_], 0, 0, 0);
                    }
                }
            }
            // register i of block kb: key 32 kb + 8 (i / 4) + 4 lh + i % 4
            float nm = mx;
#pragma unroll
            for (int kb_ = 0; kb_ < KB; ++kb_)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int p = t0 + 32 * kb_ + 8 * (i / 4) + 4 * lh + i % 4;
                    const bool see = p < sp.top && p < end && (part ? p >= sp.low : true);
                    sc[kb_][i] = see ? sc[kb_][i] * cexp : -INFINITY;
                    nm = fmaxf(nm, sc[kb_][i]);
                }
            nm = fmaxf(nm, __shfl_xor(nm, 32));
            const float base = nm == -INFINITY ? 0.0f : nm;
            const float alpha = __builtin_amdgcn_exp2f(mx - base);
            mx = nm;
            sum *= alpha;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[v][i] *= alpha;
            bool seen[KB][16];
#pragma unroll
            for (int kb_ = 0; kb_ < KB; ++kb_)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    seen[kb_][i] = sc[kb_][i] != -INFINITY;
                    sc[kb_][i] = __builtin_amdgcn_exp2f(sc[kb_][i] - base);
                    sum += sc[kb_][i];
                }
            // O^T += V^T P^T: a step takes the keys of 8 (bf16) or 1 (f32) registers
            constexpr int PR = BF ? 8 : 1;
#pragma unroll
            for (int kb_ = 0; kb_ < KB; ++kb_)
#pragma unroll
                for (int c = 0; c < 16; c += PR) {
                    u32x4 pf, one;
                    if constexpr (BF) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            pf[e] = pk_bf16(sc[kb_][c + 2 * e], sc[kb_][c + 2 * e + 1]);
                            one[e] = (seen[kb_][c + 2 * e] ? 0x3f80u : 0u) | (seen[kb_][c + 2 * e + 1] ? 0x3f800000u : 0u);
                        }
                    }
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        if constexpr (BF) {
                            // lane group (lh, column half): rows 4 lh + (i / 4) of the step's two 8-key groups
                            const int q = lane & 15, ch = (lane >> 4) & 1;
                            u32x4 vf;
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const int r = 32 * kb_ + 2 * c + 8 * u + 4 * lh + (q >> 2);
                                const int pc = 4 * v + 2 * ch + ((q & 3) >> 1);
                                const unsigned char* at = vs + (r * CS + (pc ^ swz<CS>(r))) * 16 + 8 * (q & 1);
                                const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (__attribute__((address_space(3))) s16x4*)at);
                                const u32x2 tt = __builtin_bit_cast(u32x2, t);
                                vf[2 * u] = tt[0], vf[2 * u + 1] = tt[1];
                            }
                            // values that are not finite would reach rows that do not see their key (0 x inf): they
                            // are taken out, and added where they are seen
                            unsigned bad = 0;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                bad |= (vf[e] & 0x7f80u) == 0x7f80u;
                                bad |= (vf[e] & 0x7f800000u) == 0x7f800000u;
                            }
                            if (__any(bad)) {
                                u32x4 fin, up, dn;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    fin[e] = up[e] = dn[e] = 0;
#pragma unroll
                                    for (int w = 0; w < 32; w += 16) {
                                        const unsigned x = vf[e] >> w & 0xffffu;
                                        const bool nf = (x & 0x7f80u) == 0x7f80u, nan = nf && (x & 0x7fu);
                                        fin[e] |= (nf ? 0u : x) << w;
                                        up[e] |= (nf && (nan || !(x >> 15)) ? 0x3f80u : 0u) << w;
                                        dn[e] |= (nf && (nan || x >> 15) ? 0x3f80u : 0u) << w;
                                    }
                                }
                                f32x16 nu, nd;
#pragma unroll
                                for (int i = 0; i < 16; ++i) nu[i] = nd[i] = 0.0f;
                                acc[v] = __builtin_amdgcn_mfma_f32_32x32x16_bf16((bf16x8)fin, (bf16x8)pf, acc[v], 0, 0, 0);
                                nu = __builtin_amdgcn_mfma_f32_32x32x16_bf16((bf16x8)up, (bf16x8)one, nu, 0, 0, 0);
                                nd = __builtin_amdgcn_mfma_f32_32x32x16_bf16((bf16x8)dn, (bf16x8)one, nd, 0, 0, 0);
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    if (nu[i] > 0.0f) acc[v][i] += INFINITY;
                                    if (nd[i] > 0.0f) acc[v][i] -= INFINITY;
                                }
                            } else {
                                acc[v] = __builtin_amdgcn_mfma_f32_32x32x16_bf16((bf16x8)vf, (bf16x8)pf, acc[v], 0, 0, 0);
                            }
                        } else {
                            const int r = 32 * kb_ + 8 * (c / 4) + 4 * lh + c % 4, d = 32 * v + lc;
                            const float x = *(const float*)(vs + (r * CS + ((d / 4) ^ swz<CS>(r))) * 16 + 4 * (d % 4));
                            const bool nf = !(fabsf(x) < INFINITY);
                            acc[v] = __builtin_amdgcn_mfma_f32_32x32x2f32(nf ? 0.0f : x, sc[kb_][c], acc[v], 0, 0, 0);
                            if (__any(nf)) {
                                f32x16 nu, nd;
#pragma unroll
                                for (int i = 0; i < 16; ++i) nu[i] = nd[i] = 0.0f;
                                const float w = seen[kb_][c] ? 1.0f : 0.0f;
                                nu = __builtin_amdgcn_mfma_f32_32x32x2f32(nf && !(x < 0.0f) ? 1.0f : 0.0f, w, nu, 0, 0, 0);
                                nd = __builtin_amdgcn_mfma_f32_32x32x2f32(nf && !(x > 0.0f) ? 1.0f : 0.0f, w, nd, 0, 0, 0);
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    if (nu[i] > 0.0f) acc[v][i] += INFINITY;
                                    if (nd[i] > 0.0f) acc[v][i] -= INFINITY;
                                }
                            }
                        }
                    }
                }
        }
    }
    if (!there) return;
    const float total = sum + __shfl_xor(sum, 32);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    // register i of block v: column 32 v + 8 (i / 4) + 4 lh + i % 4 of this lane's row
    T* op = (T*)a.o + b * a.o_sb + s * a.o_ss + (int64_t)(hk * G + g) * a.o_sh;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = 32 * v + 2 * i + 4 * lh;
            if (d >= a.Dv) continue;
            const float x[4] = {acc[v][i] * inv, acc[v][i + 1] * inv, acc[v][i + 2] * inv, acc[v][i + 3] * inv};
            if constexpr (BF)
                *(u32x2*)(op + d) = (u32x2){pk_bf16(x[0], x[1]), pk_bf16(x[2], x[3])};
            else
                *(f32x4*)(op + d) = (f32x4){x[0], x[1], x[2], x[3]};
        }
}

bool attn_ok(const va_tok_attn_args& a) {
    if (a.B < 0 || a.S < 0 || a.Hk < 1 || a.Hq < a.Hk || a.Hq % a.Hk || a.slots < 0) return false;
    if (a.dtype != VA_DTYPE_BF16 && a.dtype != VA_DTYPE_F32) return false;
    if (a.D < 8 || a.D > 128 || a.D % 8 || a.Dv < 8 || a.Dv > 128 || a.Dv % 8) return false;
    if (a.frame < 0 || a.window < 0 || a.sinks < 0 || (a.slots && a.sinks >= a.slots)) return false;
    if (!a.frame && (a.window || a.sinks)) return false;
    if (!(a.scale > 0.0f) || !(a.scale < INFINITY)) return false;
    if ((int64_t)a.S * (a.Hq / a.Hk) > INT32_MAX - 256) return false;
    const int64_t st = a.q_sb | a.q_ss | a.q_sh | a.k_sb | a.k_ss | a.k_sh | a.v_sb | a.v_ss | a.v_sh | a.o_sb | a.o_ss | a.o_sh;
    if (st % 8) return false;
    const bool some = a.B > 0 && a.S > 0;
    if (some && (!a.q || !a.o || (a.slots && (!a.k || !a.v)))) return false;
    return !(((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.o) & 15);
}

template <typename T>
hipError_t attn_go(const va_tok_attn_args& a, hipStream_t st, dim3 grid, int ntiles) {
    switch ((max(a.D, a.Dv) + 31) / 32) {
        case 1: hipLaunchKernelGGL((attn_kernel<T, 32>), grid, dim3(256), 0, st, a, ntiles); break;
        case 2: hipLaunchKernelGGL((attn_kernel<T, 64>), grid, dim3(256), 0, st, a, ntiles); break;
        case 3: hipLaunchKernelGGL((attn_kernel<T, 96>), grid, dim3(256), 0, st, a, ntiles); break;
        default: hipLaunchKernelGGL((attn_kernel<T, 128>), grid, dim3(256), 0, st, a, ntiles);
    }
    return hipGetLastError();
}

}  // namespace

extern "C" {

int64_t va_tok_attn_workspace_bytes(const va_tok_attn_args* a) { return a && attn_ok(*a) ? 0 : VA_ERR_ARG; }

int va_tok_attn(void* stream, const va_tok_attn_args* ap) {
    if (!ap || !attn_ok(*ap)) return VA_ERR_ARG;
    const va_tok_attn_args& a = *ap;
    if (a.B == 0 || a.S == 0) return VA_OK;
    const int64_t ntiles = ((int64_t)a.S * (a.Hq / a.Hk) + 127) / 128, blocks = ntiles * a.Hk * a.B;
    if (blocks > INT32_MAX) return VA_ERR_RANGE;
    const dim3 grid((unsigned)blocks);
    const hipError_t e = a.dtype == VA_DTYPE_F32 ? attn_go<float>(a, (hipStream_t)stream, grid, (int)ntiles)
                                                 : attn_go<__bf16>(a, (hipStream_t)stream, grid, (int)ntiles);
    return e == hipSuccess ? VA_OK : VA_ERR_HIP;
}

}  // extern "C"
