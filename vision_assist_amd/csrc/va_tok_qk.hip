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
    for (int g = part; g < groups; g += parts) {
        const int h = g * hpw + sub;
        const bool isq = h < a.Hq, mine = h < heads;
        const T* src = isq ? (const T*)a.q + b * a.q_sb + s * a.q_ss + h * a.q_sh
                           : (const T*)a.k + b * a.k_sb + s * a.k_ss + (h - a.Hq) * a.k_sh;
        float x[IT][P], y[IT][P], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
#pragma unroll
            for (int p = 0; p < P; ++p) x[i][p] = y[i][p] = 0.0f;
            if (mine && on[i]) {
                if constexpr (P == 1) {
                    load_p<T, 1>(src + lo[i], x[i]);
                    if (hi[i] >= 0) load_p<T, 1>(src + hi[i], y[i]);
                } else if (a.layout) {
                    float t[2 * P];
                    load_p<T, 2 * P>(src + lo[i], t);
#pragma unroll
                    for (int p = 0; p < P; ++p) x[i][p] = t[2 * p], y[i][p] = t[2 * p + 1];
                } else {
                    load_p<T, P>(src + lo[i], x[i]);
                    load_p<T, P>(src + hi[i], y[i]);
                }
            }
#pragma unroll
            for (int p = 0; p < P; ++p) sum += x[i][p] * x[i][p] + y[i][p] * y[i][p];
        }
        for (int d = 1; d < lph; d <<= 1) sum += __shfl_xor(sum, d);
        const bool normed = isq ? a.q_weight != nullptr : a.k_weight != nullptr;
        const float inv = normed ? 1.0f / sqrtf(sum * inv_d + a.eps) : 1.0f;
        if (!mine || (!isq && !keep)) continue;
        T* dst = isq ? (T*)a.q_out + b * a.qo_sb + s * a.qo_ss + h * a.qo_sh
                     : (T*)a.k_out + b * a.ko_sb + (int64_t)slot * a.ko_ss + (h - a.Hq) * a.ko_sh;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            if (!on[i]) continue;
            float u[P], v[P];
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float l = x[i][p] * inv * (isq ? wl[0][i][p] : wl[1][i][p]);
                const float r = y[i][p] * inv * (isq ? wh[0][i][p] : wh[1][i][p]);
                u[p] = l * cc[i][p] - r * ss[i][p];
                v[p] = r * cc[i][p] + l * ss[i][p];
            }
            if constexpr (P == 1) {
                store_p<T, 1>(dst + lo[i], u);
                if (hi[i] >= 0) store_p<T, 1>(dst + hi[i], v);
            } else if (a.layout) {
                float t[2 * P];
#pragma unroll
                for (int p = 0; p < P; ++p) t[2 * p] = u[p], t[2 * p + 1] = v[p];
                store_p<T, 2 * P>(dst + lo[i], t);
            } else {
                store_p<T, P>(dst + lo[i], u);
                store_p<T, P>(dst + hi[i], v);
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

}  // namespace

extern "C" int va_tok_qk(void* stream, const va_tok_qk_args* ap) {
    if (!ap || !qk_ok(*ap)) return VA_ERR_ARG;
    const va_tok_qk_args& a = *ap;
    if (a.B == 0 || a.S == 0 || a.Hq + a.Hk == 0) return VA_OK;
    const bool f32 = a.dtype == VA_DTYPE_F32;
    const int64_t tokens = (int64_t)a.B * a.S;
    const int64_t blocks = (tokens + QK_WAVES - 1) / QK_WAVES;
    if (blocks > INT32_MAX) return VA_ERR_RANGE;
    const dim3 grid((unsigned)blocks), block(64 * QK_WAVES);
    hipStream_t st = (hipStream_t)stream;
    if (f32)
        hipLaunchKernelGGL((qk_kernel<float, 1, 2>), grid, block, 0, st, a, 64, 1);
    else
        hipLaunchKernelGGL((qk_kernel<__bf16, 1, 2>), grid, block, 0, st, a, 64, 1);
    return hipGetLastError() == hipSuccess ? VA_OK : VA_ERR_HIP;
}
