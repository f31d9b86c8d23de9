// va_tok_qk.hip -- norms of queries and keys for each head and the rotation by position, in one pass (va355.h
// va_tok_qk), with the key and the value written into a stream's cache where the call has one.
//
// A wave takes one token (or a share of its heads): its angles once, one pair a lane, into LDS -- every head of the
// token turns by the same angles -- then its heads, several at a time.  A lane holds P pairs (lo, hi) of a head, so the
// rotation needs no exchange; the mean of squares is one butterfly over the head's lanes.
#include "va_tok.h"

namespace {
using namespace tok;

constexpr int QK_WAVES = 4, QK_PAIRS = 128;  // D <= 256
constexpr int QK_U = 4;

template <typename T, int P>
__device__ __forceinline__ void load_p(const T* p, float (&v)[P]) {
    if constexpr (P == 1) {
        v[0] = (float)*p;
    } else if constexpr (sizeof(T) == 2) {
        static_assert(P == 4 || P == 8, "");
        if constexpr (P == 4) {
            const u32x2 u = *(const u32x2*)p;
            v[0] = bf_lo(u[0]), v[1] = bf_hi(u[0]), v[2] = bf_lo(u[1]), v[3] = bf_hi(u[1]);
        } else {
            const u32x4 u = *(const u32x4*)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[2 * i] = bf_lo(u[i]), v[2 * i + 1] = bf_hi(u[i]);
        }
    } else {
        static_assert(P == 2 || P == 4, "");
        if constexpr (P == 2) {
            const f32x2 u = *(const f32x2*)p;
            v[0] = u[0], v[1] = u[1];
        } else {
            const f32x4 u = *(const f32x4*)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = u[i];
        }
    }
}

template <typename T, int P>
__device__ __forceinline__ void store_p(T* p, const float (&v)[P]) {
    if constexpr (P == 1) {
        *p = (T)v[0];
    } else if constexpr (sizeof(T) == 2) {
        if constexpr (P == 4)
            *(u32x2*)p = (u32x2){pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])};
        else
            *(u32x4*)p = (u32x4){pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7])};
    } else {
        if constexpr (P == 2)
            *(f32x2*)p = (f32x2){v[0], v[1]};
        else
            *(f32x4*)p = (f32x4){v[0], v[1], v[2], v[3]};
    }
}

// Pair f of a head: values (lo, hi).  The first rot / 2 pairs are the rotated ones; the rest of the head is paired up
// the same way (its pairs are not turned), a last single value of an odd rest has hi = -1.
__device__ __forceinline__ void pair_at(int f, int D, int rot, int layout, int* lo, int* hi) {
    const int half = rot / 2;
    if (f < half) {
        *lo = layout ? 2 * f : f;
        *hi = layout ? 2 * f + 1 : f + half;
        return;
    }
    const int g = f - half, rest = D - rot, up = (rest + 1) / 2;
    *lo = rot + (layout ? 2 * g : g);
    *hi = layout ? *lo + 1 : *lo + up;
    if (*hi >= D) *hi = -1;
}

// P = 1: any size, stride and alignment, a head per wave pass, IT pairs a lane.  P > 1 (4 bf16 / 2 float pairs a lane,
// IT = 1): the launcher has checked that every group of P pairs is aligned and lies on one side of `rot`.
template <typename T, int P, int IT>
__global__ __launch_bounds__(64 * QK_WAVES) void qk_kernel(va_tok_qk_args a, int lph, int parts) {
    __shared__ float cs[QK_WAVES][2][QK_PAIRS];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int64_t unit = (int64_t)blockIdx.x * QK_WAVES + wid;  // (token, share of its heads)
    const int64_t tok = unit / parts;
    const int part = (int)(unit - tok * parts);
    const int b = (int)(tok / a.S), s = (int)(tok - (int64_t)b * a.S);
    bool live = b < a.B;
    int slot = s;
    bool keep = true;
    if (live && a.q_len) live = s < a.q_len[b];
    if (live && a.slots) {
        const int ql = a.q_len ? a.q_len[b] : a.S, kv = a.kv_len ? a.kv_len[b] : ql, ring = a.slots - a.sinks;
        const int64_t p = (int64_t)kv - ql + s;
        keep = p >= 0 && p < kv && (p < a.sinks || p >= (int64_t)kv - ring);
        if (keep) slot = p < a.sinks ? (int)p : a.sinks + ((int)p - a.sinks) % ring;
    }
    if (live) {
        const int32_t* pos = a.pos + b * a.pos_sb + s * a.pos_ss;
        for (int f = lane; f < a.rot / 2; f += 64) {
            // whole turns are dropped in float64: a position of 2^24 keeps 2^-29 of a turn
            const double t = a.turns[f] * (double)pos[a.axis[f]];
            float sn, c;
            sincospif(2.0f * (float)(t - rint(t)), &sn, &c);
            cs[wid][0][f] = c;
            cs[wid][1][f] = sn;
        }
    }
    __syncthreads();
    if (!live) return;
    const int hpw = 64 / lph, sub = lane / lph, c0 = lane - sub * lph, npair = (a.D + 1) / 2;
    constexpr int U = P == 1 ? 1 : QK_U;
    const int heads = a.Hq + a.Hk, groups = (heads + hpw - 1) / hpw;
    const float inv_d = 1.0f / (float)a.D;
    int lo[IT], hi[IT];
    float cc[IT][P], ss[IT][P], wl[2][IT][P], wh[2][IT][P];
    bool on[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int f = (i * lph + c0) * P;
        on[i] = f < npair;
        pair_at(on[i] ? f : 0, a.D, a.rot, a.layout, &lo[i], &hi[i]);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const bool turned = on[i] && f < a.rot / 2;
            cc[i][p] = turned ? cs[wid][0][f + p] : 1.0f;
            ss[i][p] = turned ? cs[wid][1][f + p] : 0.0f;
            int l = lo[i], h = hi[i];
            if (P > 1) l = lo[i] + (a.layout ? 2 * p : p), h = hi[i] + (a.layout ? 2 * p : p);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const float* g = w ? a.k_weight : a.q_weight;
                wl[w][i][p] = g && on[i] ? g[l] : 1.0f;
                wh[w][i][p] = g && on[i] && h >= 0 ? g[h] : 1.0f;
            }
        }
    }
    for (int g0 = part; g0 < groups; g0 += parts * U) {
        // U groups of heads are read before the first is stored: a wave's loads in flight, not its latency, set the rate
        float x[U][IT][P], y[U][IT][P];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = (g0 + u * parts) * hpw + sub;
            const bool isq = h < a.Hq, mine = h < heads;
            const T* src = isq ? (const T*)a.q + b * a.q_sb + s * a.q_ss + h * a.q_sh
                               : (const T*)a.k + b * a.k_sb + s * a.k_ss + (h - a.Hq) * a.k_sh;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
#pragma unroll
                for (int p = 0; p < P; ++p) x[u][i][p] = y[u][i][p] = 0.0f;
                if (!mine || !on[i]) continue;
                if constexpr (P == 1) {
                    load_p<T, 1>(src + lo[i], x[u][i]);
                    if (hi[i] >= 0) load_p<T, 1>(src + hi[i], y[u][i]);
                } else if (a.layout) {
                    float t[2 * P];
                    load_p<T, 2 * P>(src + lo[i], t);
#pragma unroll
                    for (int p = 0; p < P; ++p) x[u][i][p] = t[2 * p], y[u][i][p] = t[2 * p + 1];
                } else {
                    load_p<T, P>(src + lo[i], x[u][i]);
                    load_p<T, P>(src + hi[i], y[u][i]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = (g0 + u * parts) * hpw + sub;
            const bool isq = h < a.Hq, mine = h < heads;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int p = 0; p < P; ++p) sum += x[u][i][p] * x[u][i][p] + y[u][i][p] * y[u][i][p];
            for (int d = 1; d < lph; d <<= 1) sum += __shfl_xor(sum, d);
            const bool normed = isq ? a.q_weight != nullptr : a.k_weight != nullptr;
            const float inv = normed ? 1.0f / sqrtf(sum * inv_d + a.eps) : 1.0f;
            if (!mine || (!isq && !keep)) continue;
            T* dst = isq ? (T*)a.q_out + b * a.qo_sb + s * a.qo_ss + h * a.qo_sh
                         : (T*)a.k_out + b * a.ko_sb + (int64_t)slot * a.ko_ss + (h - a.Hq) * a.ko_sh;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                if (!on[i]) continue;
                float l[P], r[P];
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const float m = x[u][i][p] * inv * (isq ? wl[0][i][p] : wl[1][i][p]);
                    const float n = y[u][i][p] * inv * (isq ? wh[0][i][p] : wh[1][i][p]);
                    l[p] = m * cc[i][p] - n * ss[i][p];
                    r[p] = n * cc[i][p] + m * ss[i][p];
                }
                if constexpr (P == 1) {
                    store_p<T, 1>(dst + lo[i], l);
                    if (hi[i] >= 0) store_p<T, 1>(dst + hi[i], r);
                } else if (a.layout) {
                    float t[2 * P];
#pragma unroll
                    for (int p = 0; p < P; ++p) t[2 * p] = l[p], t[2 * p + 1] = r[p];
                    store_p<T, 2 * P>(dst + lo[i], t);
                } else {
                    store_p<T, P>(dst + lo[i], l);
                    store_p<T, P>(dst + hi[i], r);
                }
            }
        }
    }
    if (a.slots && keep) {  // the value, as it is
        constexpr int VE = P == 1 ? 1 : 16 / (int)sizeof(T);
        const T* src = (const T*)a.v + b * a.v_sb + s * a.v_ss;
        T* dst = (T*)a.v_out + b * a.vo_sb + (int64_t)slot * a.vo_ss;
        const int per = a.Dv / VE, n = a.Hk * per;
        for (int i = part * 64 + lane; i < n; i += parts * 64) {
            const int h = i / per, c = (i - h * per) * VE;
            if constexpr (P == 1)
                dst[h * a.vo_sh + c] = src[h * a.v_sh + c];
            else
                *(u32x4*)(dst + h * a.vo_sh + c) = *(const u32x4*)(src + h * a.v_sh + c);
        }
    }
}

bool qk_ok(const va_tok_qk_args& a) {
    if (a.B < 0 || a.S < 0 || a.Hq < 0 || a.Hk < 0 || a.Hq > (1 << 20) || a.Hk > (1 << 20) || a.D < 1 || a.D > 2 * QK_PAIRS)
        return false;
    if (a.dtype != VA_DTYPE_BF16 && a.dtype != VA_DTYPE_F32) return false;
    if (a.rot < 0 || a.rot % 2 || a.rot > a.D || (a.layout != 0 && a.layout != 1)) return false;
    if (a.rot && (!a.turns || !a.axis || !a.pos || a.axes < 1 || ((uintptr_t)a.turns & 7))) return false;
    if (!(a.eps >= 0.0f)) return false;
    const bool some = a.B > 0 && a.S > 0;
    if (some && ((a.Hq && (!a.q || !a.q_out)) || (a.Hk && (!a.k || !a.k_out)))) return false;
    if (a.slots < 0 || a.sinks < 0 || (a.slots && a.sinks >= a.slots)) return false;
    if (a.slots && a.Hk && some && (!a.v || !a.v_out || a.Dv < 1)) return false;
    return true;
}

// whether every lane's P pairs can be read and written as vectors: 8 bytes of each half (layout 0) or 16 bytes (1); the
// values of a cached token in 16 bytes
bool qk_wide(const va_tok_qk_args& a) {
    const int e = a.dtype == VA_DTYPE_F32 ? 4 : 2, P = 8 / e, n = a.layout ? 2 * P : P;
    if (a.D % (2 * P) || (a.rot / 2) % P || ((a.D - a.rot) / 2) % P) return false;
    int64_t st = a.q_sb | a.q_ss | a.q_sh | a.k_sb | a.k_ss | a.k_sh | a.qo_sb | a.qo_ss | a.qo_sh | a.ko_sb | a.ko_ss | a.ko_sh;
    if (st % n || (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.q_out | (uintptr_t)a.k_out) & (uintptr_t)(n * e - 1))) return false;
    if (!a.slots) return true;
    st = a.v_sb | a.v_ss | a.v_sh | a.vo_sb | a.vo_ss | a.vo_sh | a.Dv;
    return st % (16 / e) == 0 && !(((uintptr_t)a.v | (uintptr_t)a.v_out) & 15);
}

}  // namespace

extern "C" int va_tok_qk(void* stream, const va_tok_qk_args* ap) {
    if (!ap || !qk_ok(*ap)) return VA_ERR_ARG;
    const va_tok_qk_args& a = *ap;
    if (a.B == 0 || a.S == 0 || a.Hq + a.Hk == 0) return VA_OK;
    const bool f32 = a.dtype == VA_DTYPE_F32;
    const int64_t tokens = (int64_t)a.B * a.S;
    const bool wide = qk_wide(a);
    const int P = wide ? (f32 ? 2 : 4) : 1;
    int lph = 64;  // lanes of a head: a power of two that holds its pairs
    while (wide && lph > 1 && (lph / 2) * P >= a.D / 2) lph /= 2;
    // few tokens: a token's heads over several waves, up to eight waves for each of the 256 CUs
    const int groups = (a.Hq + a.Hk + 64 / lph - 1) / (64 / lph);
    const int parts = (int)max((int64_t)1, min((int64_t)groups, 2048 / tokens));
    const int64_t blocks = (tokens * parts + QK_WAVES - 1) / QK_WAVES;
    if (blocks > INT32_MAX) return VA_ERR_RANGE;
    const dim3 grid((unsigned)blocks), block(64 * QK_WAVES);
    hipStream_t st = (hipStream_t)stream;
    if (f32 && wide)
        hipLaunchKernelGGL((qk_kernel<float, 2, 1>), grid, block, 0, st, a, lph, parts);
    else if (f32)
        hipLaunchKernelGGL((qk_kernel<float, 1, 2>), grid, block, 0, st, a, lph, parts);
    else if (wide)
        hipLaunchKernelGGL((qk_kernel<__bf16, 4, 1>), grid, block, 0, st, a, lph, parts);
    else
        hipLaunchKernelGGL((qk_kernel<__bf16, 1, 2>), grid, block, 0, st, a, lph, parts);
    return hipGetLastError() == hipSuccess ? VA_OK : VA_ERR_HIP;
}
