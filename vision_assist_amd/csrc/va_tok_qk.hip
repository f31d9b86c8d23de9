// va_tok_qk.hip -- norms of queries and keys for each head and the rotation by position, in one pass (va355.h
// va_tok_qk), with the key and the value written into a stream's cache where the call has one.
//
// A wave takes one token (or a share of its heads): its angles once, one pair a lane, into LDS -- every head of the
// token turns by the same angles -- then its heads, several at a time.  A lane holds P pairs (lo, hi) of a head, so the
// rotation needs no exchange; the mean of squares is one butterfly over the head's lanes.
//
// Bound by memory: the tensors are read and written once.  8 x 1600 tokens, 12 + 12 heads of 64, three axes, bf16: 21.7 us,
// 3.6 TB/s (a large copy: 4.8); one token of 64 streams into their caches: 7 us, a launch and two dependent loads.
#include "va_tok.h"

namespace {
using namespace tok;

constexpr int QK_WAVES = 4, QK_PAIRS = 128;  // D <= 256

template <typename T, int P>
__device__ __forceinline__ void store_p(T* p, const float (&v)[P]) {
    if constexpr (sizeof(T) == 2) {
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

// the slot of token s of sequence b, or -1: not kept
__device__ __forceinline__ int kept_slot(const va_tok_qk_args& a, int b, int s) {
    const int ql = a.q_len ? min(a.q_len[b], a.S) : a.S, kv = a.kv_len ? a.kv_len[b] : ql, ring = a.slots - a.sinks;
    const int64_t p = (int64_t)kv - ql + s;
    if (p < 0 || p >= kv || (p >= a.sinks && p < (int64_t)kv - ring)) return -1;
    return p < a.sinks ? (int)p : a.sinks + ((int)p - a.sinks) % ring;
}

// cos and sin of the token's angles: whole turns are dropped in float64, so a position of 2^24 keeps 2^-29 of a turn; what
// the rest loses as a float (up to 2^-26 of a turn, l in radians) is added to first order for float tensors, which leaves
// 2^-48
template <typename T>
__device__ __forceinline__ void angles(const va_tok_qk_args& a, int b, int s, int lane, float (&cs)[2][QK_PAIRS]) {
    const int32_t* pos = a.pos + b * a.pos_sb + s * a.pos_ss;
    for (int f = lane; f < a.rot / 2; f += 64) {
        double t = a.turns[f] * (double)pos[a.axis[f]];
        t -= rint(t);
        const float h = (float)t, l = sizeof(T) == 4 ? 6.2831853f * (float)(t - (double)h) : 0.0f;
        float sn, c;
        sincospif(2.0f * h, &sn, &c);
        cs[0][f] = sizeof(T) == 4 ? c - l * sn : c;
        cs[1][f] = sizeof(T) == 4 ? sn + l * c : sn;
    }
}

// any size, stride and alignment: a wave per token, a head at a time, up to two pairs a lane
template <typename T>
__global__ __launch_bounds__(64 * QK_WAVES) void qk_any(va_tok_qk_args a) {
    __shared__ float cs[QK_WAVES][2][QK_PAIRS];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tok = (int64_t)blockIdx.x * QK_WAVES + wid;
    const int b = (int)(tok / a.S), s = (int)(tok - (int64_t)b * a.S);
    if (b >= a.B || (a.q_len && s >= a.q_len[b])) return;  // (whole waves, and no barrier follows)
    const int slot = a.slots ? kept_slot(a, b, s) : s;
    angles<T>(a, b, s, lane, cs[wid]);
    const int npair = (a.D + 1) / 2;
    const float inv_d = 1.0f / (float)a.D;
    int lo[2], hi[2];
    bool on[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        on[i] = lane + 64 * i < npair;
        pair_at(on[i] ? lane + 64 * i : 0, a.D, a.rot, a.layout, &lo[i], &hi[i]);
    }
    for (int h = 0; h < a.Hq + a.Hk; ++h) {
        const bool isq = h < a.Hq;
        const T* src = isq ? (const T*)a.q + b * a.q_sb + s * a.q_ss + h * a.q_sh
                           : (const T*)a.k + b * a.k_sb + s * a.k_ss + (h - a.Hq) * a.k_sh;
        const float* w = isq ? a.q_weight : a.k_weight;
        float x[2], y[2], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = on[i] ? (float)src[lo[i]] : 0.0f;
            y[i] = on[i] && hi[i] >= 0 ? (float)src[hi[i]] : 0.0f;
            sum += x[i] * x[i] + y[i] * y[i];
        }
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
        const float inv = w ? 1.0f / sqrtf(sum * inv_d + a.eps) : 1.0f;
        if (!isq && slot < 0) continue;
        T* dst = isq ? (T*)a.q_out + b * a.qo_sb + s * a.qo_ss + h * a.qo_sh
                     : (T*)a.k_out + b * a.ko_sb + (int64_t)slot * a.ko_ss + (h - a.Hq) * a.ko_sh;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (!on[i]) continue;
            const int f = lane + 64 * i;
            const float c = f < a.rot / 2 ? cs[wid][0][f] : 1.0f, n = f < a.rot / 2 ? cs[wid][1][f] : 0.0f;
            const float l = x[i] * inv * (w ? w[lo[i]] : 1.0f), r = y[i] * inv * (w && hi[i] >= 0 ? w[hi[i]] : 1.0f);
            dst[lo[i]] = (T)(l * c - r * n);
            if (hi[i] >= 0) dst[hi[i]] = (T)(r * c + l * n);
        }
    }
    if (a.slots && slot >= 0) {  // the value, as it is
        const T* src = (const T*)a.v + b * a.v_sb + s * a.v_ss;
        T* dst = (T*)a.v_out + b * a.vo_sb + (int64_t)slot * a.vo_ss;
        for (int i = lane; i < a.Hk * a.Dv; i += 64) {
            const int h = i / a.Dv, c = i - h * a.Dv;
            dst[h * a.vo_sh + c] = src[h * a.v_sh + c];
        }
    }
}

// P pairs a lane (4 of bf16, 2 of float), 64 / lph heads at a time, L = the layout; the launcher has checked that every
// group of P pairs is aligned and lies on one side of `rot`.  A token's heads may be shared by `parts` waves.  The first U
// groups of heads are on their way while the angles are formed: loads in flight, not latencies, set the rate.  Lanes and
// groups that are not there read what their neighbours read, so that no load is conditional.
template <typename T, int P, int L>
__global__ __launch_bounds__(64 * QK_WAVES) void qk_wide(va_tok_qk_args a, int lph, int parts) {
    constexpr int U = 4;
    __shared__ float cs[QK_WAVES][2][QK_PAIRS];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t unit = (int64_t)blockIdx.x * QK_WAVES + wid;  // (token, share of its heads)
    const int64_t tok = unit / parts;
    const int part = (int)(unit - tok * parts);
    const int b = (int)(tok / a.S), s = (int)(tok - (int64_t)b * a.S);
    if (b >= a.B || (a.q_len && s >= a.q_len[b])) return;  // (whole waves, and no barrier follows)
    const int hpw = 64 / lph, sub = lane / lph, f = (lane - sub * lph) * P;  // this lane's head of a group, and first pair
    const bool on = f < a.D / 2;
    int lo, hi;
    pair_at(on ? f : 0, a.D, a.rot, L, &lo, &hi);
    const int heads = a.Hq + a.Hk, groups = (heads + hpw - 1) / hpw;
    const T* qb = (const T*)a.q + b * a.q_sb + s * a.q_ss;
    const T* kb = (const T*)a.k + b * a.k_sb + s * a.k_ss;
    typedef __attribute__((ext_vector_type(2))) unsigned int half_t;  // P values
    half_t raw[U][2];
    auto load = [&](int g, half_t (&r)[2]) {
        const int h = min(g * hpw + sub, heads - 1);
        const T* src = (h < a.Hq ? qb + h * a.q_sh : kb + (h - a.Hq) * a.k_sh) + lo;
        if constexpr (L) {
            const u32x4 x = *(const u32x4*)src;
            r[0] = (half_t){x[0], x[1]}, r[1] = (half_t){x[2], x[3]};
        } else {
            r[0] = *(const half_t*)src, r[1] = *(const half_t*)(src + (hi - lo));
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) load(part + u * parts, raw[u]);
    const int slot = a.slots ? kept_slot(a, b, s) : s;
    float w[2][2][P];  // weights of queries and keys for the pairs' two values
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float* g = k ? a.k_weight : a.q_weight;
#pragma unroll
        for (int p = 0; p < P; ++p) w[k][0][p] = w[k][1][p] = 1.0f;
        if (g) {
#pragma unroll
            for (int p = 0; p < P; ++p) w[k][0][p] = g[lo + (L ? 2 * p : p)], w[k][1][p] = g[hi + (L ? 2 * p : p)];
        }
    }
    angles<T>(a, b, s, lane, cs[wid]);  // (a wave's LDS operations run in order: its own reads need no barrier)
    float c[P], n[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const bool turned = on && f < a.rot / 2;
        c[p] = turned ? cs[wid][0][f + p] : 1.0f;
        n[p] = turned ? cs[wid][1][f + p] : 0.0f;
    }
    const float inv_d = 1.0f / (float)a.D;
    T* qo = (T*)a.q_out + b * a.qo_sb + s * a.qo_ss;
    T* ko = (T*)a.k_out + b * a.ko_sb + (int64_t)max(slot, 0) * a.ko_ss;
    auto value = [](const half_t& r, int p) {
        if constexpr (sizeof(T) == 2)
            return p & 1 ? bf_hi(r[p / 2]) : bf_lo(r[p / 2]);
        else
            return __uint_as_float(r[p]);
    };
    for (int g0 = part; g0 < groups; g0 += parts * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = (g0 + u * parts) * hpw + sub;
            const bool isq = h < a.Hq;
            float x[P], y[P], sum = 0.0f;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                // layout 1: the two values of a pair lie side by side
                const float v0 = L ? value(raw[u][2 * p / P], 2 * p % P) : value(raw[u][0], p);
                const float v1 = L ? value(raw[u][(2 * p + 1) / P], (2 * p + 1) % P) : value(raw[u][1], p);
                x[p] = on ? v0 : 0.0f, y[p] = on ? v1 : 0.0f;
                sum += x[p] * x[p] + y[p] * y[p];
            }
            for (int d = 1; d < lph; d <<= 1) sum += __shfl_xor(sum, d);
            const bool normed = isq ? a.q_weight != nullptr : a.k_weight != nullptr;
            const float inv = normed ? 1.0f / sqrtf(sum * inv_d + a.eps) : 1.0f;
            float l[P], r[P];
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float m = x[p] * inv * (isq ? w[0][0][p] : w[1][0][p]), q = y[p] * inv * (isq ? w[0][1][p] : w[1][1][p]);
                l[p] = m * c[p] - q * n[p];
                r[p] = q * c[p] + m * n[p];
            }
            if (on && h < heads && (isq || slot >= 0)) {
                T* dst = isq ? qo + h * a.qo_sh : ko + (h - a.Hq) * a.ko_sh;
                if constexpr (L) {
                    float t[2 * P];
#pragma unroll
                    for (int p = 0; p < P; ++p) t[2 * p] = l[p], t[2 * p + 1] = r[p];
                    store_p<T, 2 * P>(dst + lo, t);
                } else {
                    store_p<T, P>(dst + lo, l);
                    store_p<T, P>(dst + hi, r);
                }
            }
        }
        // (after this batch's stores: in place, a later head may not be read ahead of an earlier one's store by its owner)
#pragma unroll
        for (int u = 0; u < U; ++u) load(min(g0 + (U + u) * parts, groups - 1), raw[u]);
    }
    if (a.slots && slot >= 0) {  // the value, as it is
        constexpr int VE = 16 / (int)sizeof(T);
        const T* src = (const T*)a.v + b * a.v_sb + s * a.v_ss;
        T* dst = (T*)a.v_out + b * a.vo_sb + (int64_t)slot * a.vo_ss;
        const int per = a.Dv / VE, m = a.Hk * per;
        for (int i = part * 64 + lane; i < m; i += parts * 64) {
            const int h = i / per, d = (i - h * per) * VE;
            *(u32x4*)(dst + h * a.vo_sh + d) = *(const u32x4*)(src + h * a.v_sh + d);
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
    if (a.slots && a.Hk && some && (!a.v || !a.v_out || a.Dv < 1 || (int64_t)a.Hk * a.Dv > SIDE_MAX)) return false;
    return true;
}

// whether every lane's P pairs can be read and written as vectors: 8 bytes of each half (layout 0) or 16 bytes (1); the
// values of a cached token in 16 bytes
bool wide_ok(const va_tok_qk_args& a) {
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
    hipStream_t st = (hipStream_t)stream;
    const dim3 block(64 * QK_WAVES);
    if (!wide_ok(a)) {
        const int64_t blocks = (tokens + QK_WAVES - 1) / QK_WAVES;
        if (!grid_ok(blocks, 1, 64 * QK_WAVES)) return VA_ERR_RANGE;
        if (f32)
            hipLaunchKernelGGL(qk_any<float>, dim3((unsigned)blocks), block, 0, st, a);
        else
            hipLaunchKernelGGL(qk_any<__bf16>, dim3((unsigned)blocks), block, 0, st, a);
        return hipGetLastError() == hipSuccess ? VA_OK : VA_ERR_HIP;
    }
    const int P = f32 ? 2 : 4;
    int lph = 64;  // lanes of a head: a power of two that holds its pairs
    while (lph > 1 && (lph / 2) * P >= a.D / 2) lph /= 2;
    // few tokens: a token's heads over several waves, up to eight waves for each of the 256 CUs
    const int groups = (a.Hq + a.Hk + 64 / lph - 1) / (64 / lph);
    const int parts = (int)max((int64_t)1, min((int64_t)groups, 2048 / tokens));
    const int64_t blocks = (tokens * parts + QK_WAVES - 1) / QK_WAVES;
    if (!grid_ok(blocks, 1, 64 * QK_WAVES)) return VA_ERR_RANGE;
    const dim3 grid((unsigned)blocks);
    if (f32 && a.layout)
        hipLaunchKernelGGL((qk_wide<float, 2, 1>), grid, block, 0, st, a, lph, parts);
    else if (f32)
        hipLaunchKernelGGL((qk_wide<float, 2, 0>), grid, block, 0, st, a, lph, parts);
    else if (a.layout)
        hipLaunchKernelGGL((qk_wide<__bf16, 4, 1>), grid, block, 0, st, a, lph, parts);
    else
        hipLaunchKernelGGL((qk_wide<__bf16, 4, 0>), grid, block, 0, st, a, lph, parts);
    return hipGetLastError() == hipSuccess ? VA_OK : VA_ERR_HIP;
}
