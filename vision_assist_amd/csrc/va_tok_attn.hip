// va_tok_attn.hip -- attention with frames, a sliding window and sinks over a stream's cache (va355.h va_tok_attn).
//
// The G query heads of a key head and the positions are one list of rows, row = position * G + head, so one staged tile
// of keys and values serves all of them and the rows of a workgroup span few positions.  A wave holds 32 rows as MFMA
// columns: S^T = K Q^T leaves a lane the scores of ONE row (its lane & 31), so maximum and sum are in-lane plus one
// exchange with lane ^ 32, and O^T = V^T P^T takes those registers as its B operand without any exchange: the sum over
// keys may run in any order, so V^T is read in the order in which the scores lie in the registers.
//   bf16: v_mfma_f32_32x32x16_bf16, V^T by the transposing LDS read (16 lanes x 8 bytes: 4 keys x 16 columns)
//   f32:  v_mfma_f32_32x32x2_f32 (exact products), V^T by plain 4-byte reads
// One pass over the keys with the running maximum and sum of the softmax (base 2: the scale is folded with log2 e).  A row's
// running maximum is only raised where a score passes it by more than 8 (in powers of two): its sums stay below 2^8 times
// the keys, and few tiles rescale.  bf16, many rows: the probabilities are rounded to bf16 for the second product (half a
// step, 2^-8 of each at most), and the sum is of the rounded ones, which is what the product weighs by.  Few rows (single
// tokens over a cache) are bound by the cache's bytes, so there a probability enters as two bf16 terms (2^-16 of it is left
// out) and the sum is of the floats: 1 % of the time (161.1 us against 159.4 for 32 streams over 6800 slots, graph
// replays), and the error against float64 is the output's own rounding (0.0017 instead of 0.0023, relative L2).  For many
// rows the second term's MFMAs and conversions were 23 to 27 % of the time (116 -> 143 us, 136 -> 168, 254 -> 324).
//
// What is not finite in a value that no row of a tile's part sees must not meet a probability of 0 in an MFMA: in tiles
// that some row does not see whole, such values are replaced by 0 as the tile arrives (take_out) and added afterwards by
// the rows that do see them (add_nonfinite); whole tiles need neither.  Every probability of a seen key is positive, so what a
// row sees of a column alone says which infinity it is or that it is NaN; but a probability, or the factor that rescales a
// sum, may come out 0, and 0 x inf is NaN.  Results that are not finite are therefore settled by the column's values (settle).
#include <math.h>

#include "va_dev.h"
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

// visible positions of the query at position i (up to 2^31 - 2: what follows forms differences of positions, no sums): [0, min(sinks, top)) and [low, top), low >= sinks; nothing for i < 0
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
    static constexpr int KT = 64;  // keys of a staged tile
};
template <>
struct Tr<float> {
    static constexpr int VE = 4;
    static constexpr int KT = 32;
};
// rows of D values (a multiple of 32) as they are staged: NC pieces, laid out as CS (a power of two)
template <typename T, int D>
struct Dims {
    static constexpr int NC = D / Tr<T>::VE, CS = NC <= 4 ? 4 : NC <= 8 ? 8 : NC <= 16 ? 16 : 32;
};
// attn_split: waves of a workgroup (two buffers of K and V tiles each within the LDS), and its bytes
template <typename T, int DQ, int DV>
struct Split {
    static constexpr int CK = Dims<T, DQ>::CS, CV = Dims<T, DV>::CS, SW = CK + CV > 32 ? 2 : 4, LDS = SW * 2 * 32 * (CK + CV) * 16;
    static_assert(LDS <= 128 * 1024 && SW / 2 * (DV / 32) * 16 * 64 * 4 <= LDS, "");
};

// LDS image of a tile: rows of CS 16-byte pieces, piece c of row r in place c ^ swz(r), so that the lanes that a read
// serves at a time (256 bytes) touch every bank once: K is read at one piece of 16 consecutive rows; V by the transposing
// read at 4 pieces of 4 rows (bf16), or at 8 pieces of two rows 4 apart (float).
template <typename T, int CS>
__device__ __forceinline__ int swz(int r) {
    if constexpr (CS >= 16)
        return sizeof(T) == 2 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r & 4) << 1) | ((r & 3) << 1) | ((r >> 3) & 1);
    else if constexpr (CS == 8)
        return ((r & 2) << 1) | ((r >> 2) & 3);
    else
        return (r >> 2) & 3;
}

__device__ __forceinline__ int slot_of(const va_tok_attn_args& a, int p) {
    if (p < a.slots) return p;
    return a.sinks + (p - a.sinks) % (a.slots - a.sinks);
}

// sc = K Q^T of KB blocks of 32 keys x 32 rows; kf(k, c): piece 2 c + lh of this lane's key in block k.  bf16: a block's
// fragments are read beside the MFMAs of the block before.
template <typename T, int DQ, int KB, typename F>
__device__ __forceinline__ void scores(f32x16 (&sc)[KB], const u32x4 (&qf)[DQ / (2 * Tr<T>::VE)], F kf) {
    constexpr int NF = DQ / (2 * Tr<T>::VE);
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[k][i] = 0.0f;
    if constexpr (sizeof(T) == 2) {
        u32x4 f[KB][NF];
#pragma unroll
        for (int c = 0; c < NF; ++c) f[0][c] = kf(0, c);
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int c = 0; c < NF; ++c) {
                if (k + 1 < KB) f[k + 1][c] = kf(k + 1, c);
                sc[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16((bf16x8)f[k][c], (bf16x8)qf[c], sc[k], 0, 0, 0);
            }
        __builtin_amdgcn_sched_group_barrier(0x100, NF, 0);
#pragma unroll
        for (int i = 0; i < KB * NF; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (i < (KB - 1) * NF) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    } else {
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int c = 0; c < NF; ++c) {
                const u32x4 f = kf(k, c);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sc[k] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(f[e]), __uint_as_float(qf[c][e]), sc[k], 0, 0, 0);
            }
    }
}

// the key of register i of a block of 32 scores
__device__ __forceinline__ int key_of(int i, int lh) { return 8 * (i / 4) + 4 * lh + i % 4; }

// the larger of this lane's value and its partner's (lane ^ 32): the swap of x with itself leaves both lanes' values in both
__device__ __forceinline__ float pair_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The running softmax of one row (a lane and its partner lane ^ 32): mx is the reference of the exponents in units of
// the raw scores, kept while the maximum grows by less than 2^8 in the result (the sums are float, and a probability
// rounded to bf16 has the same relative error at any size).  Exponents: 2^((s - mx) c).
template <int NV>
struct Row {
    float mx = -INFINITY, sum = 0.0f;
    f32x16 acc[NV];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[v][i] = 0.0f;
    }
};

// keys from .. to - 1 of a tile are this row's (the bounds moved by the lane's 4 lh, so that they meet constants)
template <int KB>
__device__ __forceinline__ void mask(f32x16 (&sc)[KB], int from, int to, int lh) {
    from -= 4 * lh, to -= 4 * lh;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int p = 32 * k + key_of(i, 0);
            sc[k][i] = ((from <= p) & (p < to)) ? sc[k][i] : -INFINITY;
        }
}

// (FSUM: the sum is formed here, of the floats)
template <typename T, int KB, int NV, bool FSUM>
__device__ __forceinline__ void softmax(Row<NV>& r, f32x16 (&sc)[KB], float c) {
    float nm = -INFINITY;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) nm = fmaxf(nm, sc[k][i]);
    nm = pair_max(nm);
    const bool up = nm > r.mx && !((nm - r.mx) * c <= 8.0f);
    if (__any(up)) {  // (each row by its own maximum alone: a row's result does not depend on the others')
        const float alpha = up ? __builtin_amdgcn_exp2f((r.mx - nm) * c) : 1.0f;
        r.mx = up ? nm : r.mx;
        r.sum *= alpha;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 16; ++i) r.acc[v][i] *= alpha;
    }
    const float off = r.mx == -INFINITY ? 0.0f : -r.mx * c;
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            sc[k][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[k][i], c, off));
            if constexpr (FSUM) part[i % 4] += sc[k][i];
        }
    if constexpr (FSUM) r.sum += (part[0] + part[1]) + (part[2] + part[3]);
}

// This lane's LDS addresses in a tile's image, formed once: K of row lane & 31, piece 2 c + lh; V for the reads of block v.
// bf16: 16 lanes read 4 keys of 16 columns (rows 4 lh + 0 .. 3 of the 8-key group u, columns 32 v + 16 (lane / 16 % 2) ..)
// and lane q of them gets column q's 4 keys.  Later keys of a tile are a constant away (32 rows' swizzles are 0 .. 31's).
template <typename T, int DQ, int DV>
struct Addr {
    static constexpr int CK = Dims<T, DQ>::CS, CV = Dims<T, DV>::CS, NV = DV / 32, NF = DQ / (2 * Tr<T>::VE), U = sizeof(T) == 2 ? 2 : 1;
    int k[NF], v[U][NV];
    __device__ __forceinline__ Addr(int lane) {
        const int lc = lane & 31, lh = lane >> 5, q = lane & 15, ch = (lane >> 4) & 1;
#pragma unroll
        for (int c = 0; c < NF; ++c) k[c] = (lc * CK + ((2 * c + lh) ^ swz<T, CK>(lc))) * 16;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int row = 8 * u + 4 * lh + (q >> 2), pc = 4 * i + 2 * ch + ((q & 3) >> 1);
                    v[u][i] = (row * CV + (pc ^ swz<T, CV>(row))) * 16 + 8 * (q & 1);
                }
        }
    }
};

template <typename T, int DQ, int DV>
__device__ __forceinline__ u32x4 values_bf16(const Addr<T, DQ, DV>& ad, const unsigned char* vs, int row0, int v) {
    u32x4 vf;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const unsigned char* at = vs + ad.v[u][v] + row0 * (Dims<T, DV>::CS * 16);
        const u32x2 t = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
        vf[2 * u] = t[0], vf[2 * u + 1] = t[1];
    }
    return vf;
}

// V^T of step st (16 keys) of a tile, block v of columns
template <typename T, int DQ, int DV>
struct Values {
    u32x4 f[DV / 32];
    __device__ __forceinline__ void read(const Addr<T, DQ, DV>& ad, const unsigned char* vs, int st) {
#pragma unroll
        for (int v = 0; v < DV / 32; ++v) f[v] = values_bf16<T, DQ, DV>(ad, vs, 16 * st, v);
    }
};

// O^T += V^T P^T over the KB blocks of 32 keys of a tile; bf16: first = step 0's values, read before the softmax, and each
// step's are read beside the MFMAs of the step before; TWO: the probabilities as two bf16 terms, else their rounded sum too
template <typename T, int DQ, int DV, int KB, bool TWO>
__device__ __forceinline__ void add_values(Row<DV / 32>& r, const f32x16 (&p)[KB], const Values<T, DQ, DV>& first,
                                           const Addr<T, DQ, DV>& ad, const unsigned char* vs, int lane) {
    constexpr int CS = Dims<T, DV>::CS, NV = DV / 32;
    if constexpr (sizeof(T) == 2) {
        Values<T, DQ, DV> cur = first, next;
        const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
        float part[2] = {0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < 2 * KB; ++st) {
            if (st + 1 < 2 * KB) next.read(ad, vs, st + 1);
            u32x4 pf, pl;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f32x16& w = p[st / 2];
                const int i = 8 * (st & 1) + 2 * e;
                const bf16x2 two = {(__bf16)w[i], (__bf16)w[i + 1]};
                pf[e] = __builtin_bit_cast(unsigned, two);
                if constexpr (TWO)
                    pl[e] = pk_bf16(w[i] - bf_lo(pf[e]), w[i + 1] - bf_hi(pf[e]));
                else
                    part[e & 1] = __builtin_amdgcn_fdot2_f32_bf16(two, one, part[e & 1], false);
            }
            if constexpr (!TWO) asm volatile("" : "+v"(part[0]), "+v"(part[1]));  // (summed here, beside the MFMAs)
#pragma unroll
            for (int v = 0; v < NV; ++v)
                r.acc[v] = __builtin_amdgcn_mfma_f32_32x32x16_bf16((bf16x8)cur.f[v], (bf16x8)pf, r.acc[v], 0, 0, 0);
            if constexpr (TWO) {
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    r.acc[v] = __builtin_amdgcn_mfma_f32_32x32x16_bf16((bf16x8)cur.f[v], (bf16x8)pl, r.acc[v], 0, 0, 0);
            }
            cur = next;
        }
        if constexpr (!TWO) r.sum += part[0] + part[1];
    } else {
        const int lc = lane & 31, lh = lane >> 5;
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = 32 * k + key_of(i, lh);
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const int d = 32 * v + lc;
                    const float x = *(const float*)(vs + (row * CS + ((d / 4) ^ swz<T, CS>(row))) * 16 + 4 * (d % 4));
                    r.acc[v] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[k][i], r.acc[v], 0, 0, 0);
                }
            }
    }
}

// Values that are not finite, in tiles that some row does not see whole: the product would carry them, as 0 x inf, into
// rows that do not see their key.  A wave takes them out of the pieces that it has staged -- zeros in their places, two
// bits a value of what stood there (1 +inf, 2 -inf, 3 NaN) in kinds, one word a piece -- and after the product each row
// adds those of the keys it sees.
template <typename T>
__device__ __forceinline__ bool take_out(unsigned char* piece, unsigned short* kind) {
    u32x4 x = *(const u32x4*)piece;
    unsigned k = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned y = x[e] >> (16 * h) & 0xffffu;
                if ((y & 0x7f80u) == 0x7f80u) {
                    k |= (y & 0x7fu ? 3u : y >> 15 ? 2u : 1u) << (4 * e + 2 * h);
                    x[e] &= h ? 0xffffu : 0xffff0000u;
                }
            }
        } else if ((x[e] & 0x7f800000u) == 0x7f800000u) {
            k |= (x[e] & 0x7fffffu ? 3u : x[e] >> 31 ? 2u : 1u) << (2 * e);
            x[e] = 0;
        }
    }
    *kind = (unsigned short)k;
    if (k) *(u32x4*)piece = x;
    return k != 0;
}

// ... positions from .. to - 1 of the tile's n keys are seen
template <typename T, int DV>
__device__ __forceinline__ void add_nonfinite(Row<DV / 32>& r, const unsigned short* kinds, int from, int to, int n, int lh) {
    constexpr int CS = Dims<T, DV>::CS, NV = DV / 32, VE = Tr<T>::VE;
#pragma unroll 1
    for (int k = max(from, 0); k < min(to, n); ++k) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {  // four values of one piece
                const int d = 32 * v + key_of(i, lh);
                const unsigned w = kinds[k * CS + ((d / VE) ^ swz<T, CS>(k))] >> (2 * (d % VE));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned q = w >> (2 * e) & 3u;
                    if (q) r.acc[v][i + e] += q == 1 ? INFINITY : q == 2 ? -INFINITY : NAN;
                }
                __builtin_amdgcn_sched_barrier(0);  // few registers, not speed
            }
    }
}

// What is not finite in a row's NB blocks of columns from block v0 on is what the values that it sees make it: an infinity,
// or NaN where it sees both or a NaN; not where the scores made the row NaN (sum), nor where finite values passed the range.
template <typename T, int NB>
__device__ __forceinline__ void settle(const va_tok_attn_args& a, f32x16 (&x)[NB], float sum, const T* vb, Span sp, int v0, int lh) {
    float z = 0.0f;
#pragma unroll
    for (int v = 0; v < NB; ++v)
#pragma unroll
        for (int i = 0; i < 16; ++i) z = __builtin_fmaf(x[v][i], 0.0f, z);
    if (__builtin_expect(z == z || sum != sum, 1)) return;
    // U keys at a time, so that their loads run together, until every such column has shown that it is NaN
    constexpr int U = NB == 1 ? 8 : NB == 2 ? 4 : 2;
    unsigned plus[NB], minus[NB], open[NB];
#pragma unroll
    for (int v = 0; v < NB; ++v) {
        plus[v] = minus[v] = open[v] = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) open[v] |= (unsigned)!(fabsf(x[v][i]) < INFINITY) << i;
    }
    bool more = true;
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        const int end = part ? sp.top : min(a.sinks, sp.top);
#pragma unroll 1
        for (int p = part ? sp.low : 0; p < end && more; p += min(U, end - p)) {
            const T* row[U];  // (the last one's again where there are fewer)
#pragma unroll
            for (int u = 0; u < U; ++u) row[u] = vb + (int64_t)slot_of(a, p + min(u, end - 1 - p)) * a.v_ss;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int v = 0; v < NB; ++v)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const int d = min(32 * (v0 + v) + key_of(i, lh), a.Dv - 4);  // (columns from Dv on are not stored)
                        float four[4];
                        if constexpr (sizeof(T) == 2) {
                            const u32x2 y = *(const u32x2*)(row[u] + d);
                            four[0] = bf_lo(y[0]), four[1] = bf_hi(y[0]), four[2] = bf_lo(y[1]), four[3] = bf_hi(y[1]);
                        } else {
                            const f32x4 y = *(const f32x4*)(row[u] + d);
                            four[0] = y[0], four[1] = y[1], four[2] = y[2], four[3] = y[3];
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            plus[v] |= (unsigned)!(four[e] < INFINITY) << (i + e);  // (NaN: both)
                            minus[v] |= (unsigned)!(four[e] > -INFINITY) << (i + e);
                        }
                    }
            more = false;
#pragma unroll
            for (int v = 0; v < NB; ++v) more |= (open[v] & ~(plus[v] & minus[v])) != 0;
        }
    }
#pragma unroll
    for (int v = 0; v < NB; ++v)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const bool p = plus[v] >> i & 1, m = minus[v] >> i & 1;
            x[v][i] = p && m ? NAN : p ? INFINITY : m ? -INFINITY : x[v][i];
        }
}

// 16 registers of block v -> columns 32 v + key_of(i, lh) of this lane's row
template <typename T>
__device__ __forceinline__ void store_block(T* op, const f32x16& x, float by, int v, int lh, int Dv) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const int d = 32 * v + key_of(i, lh);
        if (d >= Dv) continue;
        if constexpr (sizeof(T) == 2)
            *(u32x2*)(op + d) = (u32x2){pk_bf16(x[i] * by, x[i + 1] * by), pk_bf16(x[i + 2] * by, x[i + 3] * by)};
        else
            *(f32x4*)(op + d) = (f32x4){x[i] * by, x[i + 1] * by, x[i + 2] * by, x[i + 3] * by};
    }
}

template <typename T, int DQ>
__device__ __forceinline__ void load_q(const va_tok_attn_args& a, const T* qp, bool there, int lh,
                                       u32x4 (&qf)[DQ / (2 * Tr<T>::VE)]) {
    constexpr int VE = Tr<T>::VE;
#pragma unroll
    for (int c = 0; c < DQ / (2 * VE); ++c) {
        const int d = (2 * c + lh) * VE;
        qf[c] = there && d < a.D ? *(const u32x4*)(qp + d) : (u32x4){0, 0, 0, 0};
    }
}

// The walk over a row block's keys: positions [0, ntop), [low, mid) and [mid, top) -- the sinks, and what its rows see
// behind them, cut where the ring begins anew so that a tile's slots are consecutive -- in tiles of KT.
template <int KT>
struct Walk {
    int ntop, low, mid, top, n0, n1, nt;
    __device__ __forceinline__ Walk(const va_tok_attn_args& a, Span first, Span last) {
        top = last.top, low = max(first.low, a.sinks), ntop = min(a.sinks, top), mid = top;
        if (top > a.slots && top > low) {
            const int ring = a.slots - a.sinks;
            const int64_t m = a.sinks + ((int64_t)(low - a.sinks) + ring - 1) / ring * ring;
            mid = m < top ? (int)m : top;
        }
        n0 = (ntop + KT - 1) / KT;
        n1 = n0 + (mid > low ? (mid - low + KT - 1) / KT : 0);
        nt = n1 + (top > mid && top > low ? (top - max(mid, low) + KT - 1) / KT : 0);
    }
    // tile t holds positions t0 .. min(t0 + KT, end) - 1
    __device__ __forceinline__ void tile(int t, int* t0, int* end) const {
        *t0 = t < n0 ? t * KT : t < n1 ? low + (t - n0) * KT : mid + (t - n1) * KT;
        *end = t < n0 ? ntop : t < n1 ? mid : top;
    }
};

// ------------------------------------------------------------------ many rows: 128 a workgroup, keys through LDS
// Tiles of KT keys in two LDS buffers: the next tile is on its way into one by LDS-DMA while the other is worked on, and
// one wait and barrier a tile publish it.  Tiles of 64 keys (bf16) or 32: the scores of twice as many would not fit the
// registers of three waves a SIMD at D <= 64, of two at 128.  A tile's slots are consecutive (the walk is cut at the ring's end), so its
// rows are offsets from one address; rows and pieces that are not there take an offset out of range and load zeros.
// Bound by the instructions between the products: at D = 128 MFMAs and vector instructions (an exp2 of four issue slots,
// a multiply-add, half a maximum, half a conversion and half a sum for each score) take half of a SIMD's time each, and two
// waves overlap them in part.  Measured, bf16: 16 heads over 2 key heads, 8192 tokens, window 4096, D 128: 258 us, 799
// TFLOP/s; 8 streams, 400 queries over 3200 keys, D 128: 119 us, 704 TFLOP/s; two clips of 6400 tokens, frames of 400, D
// 64: 138 us, 570 TFLOP/s.  One stream's 400 queries alone (16 over 8 heads) are 56 workgroups for 256 CUs, each of which
// walks all keys: 92 us.  Float (32-bit MFMA, 154 TFLOP/s at most): 16 x 8 heads of 400 x 400, D 32, Dv 64: 53 us, 74
// TFLOP/s.
constexpr int TILE_OOB = 0x7ffffff0;

// (a plain function: the host pass drops the stub of a kernel template that names the builtin)
__device__ __forceinline__ void dma16(const void* base, void* lds, int off, int uniform) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, TILE_OOB, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lvoid_t*)lds, 16, off, uniform, 0, 0);
}

// waves of a SIMD: three where the registers of D <= 64 allow it
template <typename T, int DQ, int DV>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (DV <= 64 ? 3 : 2) : (DV <= 64 ? 2 : 1)) void attn_kernel(va_tok_attn_args a, int ntiles) {
    constexpr int VE = Tr<T>::VE, KT = Tr<T>::KT, CK = Dims<T, DQ>::CS, CV = Dims<T, DV>::CS, KB = KT / 32, NV = DV / 32;
    constexpr int NK = KT * CK / 256, NP = KT * CV / 256;             // DMAs of a wave for K, for V
    constexpr int KBUF = KT * CK * 16, BUF = KBUF + KT * CV * 16;      // bytes of a tile of K, of both
    extern __shared__ __align__(16) unsigned char sm[];    // [2][K | V]
    __shared__ unsigned short kinds[2][KT * CV];
    __shared__ int bad_tile[2];  // the tile of a buffer, if values were taken out of it
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), lc = lane & 31, lh = lane >> 5;
    const int G = a.Hq / a.Hk;
    // Four row blocks of a unit (a sequence's key head) are a run on one XCD, which share its keys in that L2; those that
    // see most come first, over all units.  (A contiguous eighth for each XCD, unit after unit: 162 us instead of 136 for
    // two clips, 288 instead of 255 for a long prompt, as the XCDs' shares differ in work.  Runs of 8, 16: the same.)
    constexpr int RUN = 4;
    const int at = xcd_runs<RUN>(blockIdx.x, gridDim.x), units = a.B * a.Hk, run = at / (units * RUN);
    const int in = at - run * units * RUN, width = min(RUN, ntiles - run * RUN);
    const int unit = in / width, tile = ntiles - 1 - (run * RUN + in % width), hk = unit % a.Hk, b = unit / a.Hk;
    const AttnSeq sq = attn_seq(a, b);
    const int rows = sq.ql * G, r0 = tile * 128;
    if (r0 >= rows) return;
    const int row = r0 + 32 * wid + lc, s = row / G, g = row - s * G;  // this lane's row
    const bool there = row < rows;
    const Span sp = there ? attn_span(a, sq, sq.first + s) : Span{a.sinks, 0};
    // spans grow with the position: the workgroup's keys, and this wave's
    const Span g0 = attn_span(a, sq, sq.first + r0 / G), g1 = attn_span(a, sq, sq.first + (min(r0 + 128, rows) - 1) / G);
    const Walk<KT> w(a, attn_span(a, sq, max(sq.first + r0 / G, 0)), g1);
    const Span f0 = attn_span(a, sq, sq.first + min(r0 + 32 * wid, rows - 1) / G);
    const Span f1 = attn_span(a, sq, sq.first + min(r0 + 32 * wid + 31, rows - 1) / G);
    const bool idle = r0 + 32 * wid >= rows;

    u32x4 qf[DQ / (2 * VE)];
    load_q<T, DQ>(a, (const T*)a.q + b * a.q_sb + s * a.q_ss + (int64_t)(hk * G + g) * a.q_sh, there, lh, qf);
    const float cexp = a.scale * 1.4426950408889634f;
    Row<NV> r;
    r.clear();
    const Addr<T, DQ, DV> ad(lane);

    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    // this lane's DMAs: place i = (wid * N + j) * 64 + lane of an operand's image, row i / CS = r_0 + j 64 / CS, piece i % CS ^ swz
    const int kr = wid * NK * (64 / CK) + lane / CK, vr = wid * NP * (64 / CV) + lane / CV;
    const int krow = (int)(kr * a.k_ss) * (int)sizeof(T), vrow = (int)(vr * a.v_ss) * (int)sizeof(T);
    auto fetch = [&](int t, int buf) {
        int t0, end;
        w.tile(t, &t0, &end);
        const int64_t slot = slot_of(a, t0);
        const T *kt = kb + slot * a.k_ss, *vt = vb + slot * a.v_ss;
        unsigned char *ks = sm + buf * BUF + wid * NK * 1024, *vs = sm + buf * BUF + KBUF + wid * NP * 1024;
        const bool whole = end - t0 >= KT;  // (uniform) no row is missing
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            const int rj = kr + j * (64 / CK), c = lane % CK ^ swz<T, CK>(rj);
            const int out = whole ? 0 : (int)(rj >= end - t0);  // (no short cuts: a branch would split the DMA)
            dma16(kt, ks + j * 1024, (out | (int)(c * VE >= a.D)) ? TILE_OOB : krow + 16 * c,
                  j * (64 / CK) * (int)a.k_ss * (int)sizeof(T));
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int rj = vr + j * (64 / CV), c = lane % CV ^ swz<T, CV>(rj);
            const int out = whole ? 0 : (int)(rj >= end - t0);
            dma16(vt, vs + j * 1024, (out | (int)(c * VE >= a.Dv)) ? TILE_OOB : vrow + 16 * c,
                  j * (64 / CV) * (int)a.v_ss * (int)sizeof(T));
        }
    };
    // whether some row of the workgroup does not see a tile whole
    auto partial = [&](int t) {
        int t0, end;
        w.tile(t, &t0, &end);
        return min(g0.top, end) - t0 < KT || (t >= w.n0 && t0 < g1.low);
    };
    // this wave's pieces of tile t are there: what is not finite leaves them before the barrier shows them to the others
    auto clean = [&](int t) {
        const int buf = t & 1, first = wid * NP * 64 + lane;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < NP; ++j)
            bad |= take_out<T>(sm + buf * BUF + KBUF + (first + j * 64) * 16, &kinds[buf][first + j * 64]);
        if (bad) bad_tile[buf] = t;
    };
    if (tid < 2) bad_tile[tid] = -1;
    __syncthreads();
    __builtin_amdgcn_s_setprio(1);
    if (w.nt > 0) {
        fetch(0, 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (partial(0)) clean(0);
    }
    __syncthreads();
    for (int t = 0; t < w.nt; ++t) {
        const int buf = t & 1;
        if (t + 1 < w.nt) fetch(t + 1, buf ^ 1);
        const unsigned char *ks = sm + buf * BUF, *vs = ks + KBUF;
        int t0, end;
        w.tile(t, &t0, &end);
        const bool sink = t < w.n0;
        if (!idle && t0 < f1.top && (sink || f0.low - t0 < KT)) {
            f32x16 sc[KB];
            scores<T, DQ, KB>(sc, qf, [&](int k, int c) { return *(const u32x4*)(ks + ad.k[c] + k * 32 * CK * 16); });
            Values<T, DQ, DV> v0;
            if constexpr (sizeof(T) == 2) v0.read(ad, vs, 0);
            const int from = (sink ? 0 : sp.low) - t0, upto = min(sp.top, end) - t0;
            if (min(f0.top, end) - t0 < KT || (!sink && t0 < f1.low)) mask<KB>(sc, from, upto, lh);  // not all see all
            __builtin_amdgcn_s_setprio(0);  // (beside the other waves' products, which go first)
            softmax<T, KB, NV, sizeof(T) == 4>(r, sc, cexp);
            __builtin_amdgcn_s_setprio(1);
            add_values<T, DQ, DV, KB, false>(r, sc, v0, ad, vs, lane);
            if (bad_tile[buf] == t) add_nonfinite<T, DV>(r, kinds[buf], from, upto, KT, lh);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (t + 1 < w.nt && partial(t + 1)) clean(t + 1);
        __syncthreads();
    }
    const float total = r.sum + __shfl_xor(r.sum, 32);
    if (!there) return;
    settle<T, NV>(a, r.acc, total, vb, sp, 0, lh);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    T* op = (T*)a.o + b * a.o_sb + s * a.o_ss + (int64_t)(hk * G + g) * a.o_sh;
#pragma unroll
    for (int v = 0; v < NV; ++v) store_block<T>(op, r.acc[v], inv, v, lh, a.Dv);
}

// ------------------------------------------------------------------ few rows: the keys split over waves and workgroups
// A workgroup takes 32 rows and one of nsplit shares of their tiles of 32 keys; its waves walk the share's tiles in
// turn, each through two buffers of its own in LDS and without a barrier, until their sums are joined.  A tile comes by
// LDS-DMA while the one before is worked on, whole rows at a time (a load covers complete cache lines: reading each key's
// row by its own lane instead, 32 lines at a time, ran at 1.7 TB/s).  Bound by the bytes of the keys and values: 32
// streams over 6800 slots, 8 key heads of 128: 153 us, 4.2 TB/s (a large copy: 4.8).
// A share's result: [NV * 16][64] registers as they lie in the wave, then the 32 rows' maxima and sums.
__device__ __forceinline__ int64_t part_floats(int NV) { return NV * 16 * 64 + 64; }

template <typename T, int DQ, int DV>
__global__ __launch_bounds__((64 * Split<T, DQ, DV>::SW), 1) void attn_split(va_tok_attn_args a, int nrb, int nsplit) {
    constexpr int VE = Tr<T>::VE, CK = Dims<T, DQ>::CS, CV = Dims<T, DV>::CS, NV = DV / 32, SW = Split<T, DQ, DV>::SW;
    constexpr int NK = 32 * CK / 64, NP = 32 * CV / 64, KBUF = 32 * CK * 16, BUF = KBUF + 32 * CV * 16, ACC = NV * 16 * 64 * 4;
    extern __shared__ __align__(16) unsigned char sm[];  // a wave: [2][K | V]; then the waves' registers
    __shared__ unsigned short kinds[SW][32 * CV];
    __shared__ float sms[2][2][64];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), lc = lane & 31, lh = lane >> 5;
    const int G = a.Hq / a.Hk;
    int bid = xcd_tile(blockIdx.x, gridDim.x);
    const int split = bid % nsplit;
    bid /= nsplit;
    const int rb = bid % nrb;
    const int unit = bid / nrb, hk = unit % a.Hk, b = unit / a.Hk;
    const AttnSeq sq = attn_seq(a, b);
    const int rows = sq.ql * G, r0 = rb * 32;
    if (r0 >= rows) return;
    const int row = r0 + lc, s = row / G, g = row - s * G;
    const bool there = row < rows;
    const Span sp = there ? attn_span(a, sq, sq.first + s) : Span{a.sinks, 0};
    const Span f0 = attn_span(a, sq, sq.first + r0 / G), f1 = attn_span(a, sq, sq.first + (min(r0 + 32, rows) - 1) / G);
    const Walk<32> w(a, attn_span(a, sq, max(sq.first + r0 / G, 0)), f1);
    const int per = (w.nt + nsplit - 1) / nsplit, t1 = min((split + 1) * per, w.nt);

    u32x4 qf[DQ / (2 * VE)];
    load_q<T, DQ>(a, (const T*)a.q + b * a.q_sb + s * a.q_ss + (int64_t)(hk * G + g) * a.q_sh, there, lh, qf);
    const float cexp = a.scale * 1.4426950408889634f;
    Row<NV> r;
    r.clear();
    const Addr<T, DQ, DV> ad(lane);
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    // this lane's DMAs: place j * 64 + lane of an operand's image, row lane / CS + j 64 / CS
    const int kr = lane / CK, vr = lane / CV;
    const int krow = (int)(kr * a.k_ss) * (int)sizeof(T), vrow = (int)(vr * a.v_ss) * (int)sizeof(T);
    unsigned char* mine = sm + wid * 2 * BUF;
    auto fetch = [&](int t, int buf) {
        int t0, end;
        w.tile(t, &t0, &end);
        const int64_t slot = slot_of(a, t0);
        const T *k = kb + slot * a.k_ss, *v = vb + slot * a.v_ss;
        unsigned char* to = mine + buf * BUF;
        const bool whole = end - t0 >= 32;
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            const int rj = kr + j * (64 / CK), c = lane % CK ^ swz<T, CK>(rj);
            const int out = whole ? 0 : (int)(rj >= end - t0);
            dma16(k, to + j * 1024, (out | (int)(c * VE >= a.D)) ? TILE_OOB : krow + 16 * c, j * (64 / CK) * (int)a.k_ss * (int)sizeof(T));
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int rj = vr + j * (64 / CV), c = lane % CV ^ swz<T, CV>(rj);
            const int out = whole ? 0 : (int)(rj >= end - t0);
            dma16(v, to + KBUF + j * 1024, (out | (int)(c * VE >= a.Dv)) ? TILE_OOB : vrow + 16 * c,
                  j * (64 / CV) * (int)a.v_ss * (int)sizeof(T));
        }
    };
    int t = split * per + wid, buf = 0;
    if (t < t1) fetch(t, 0);
    for (; t < t1; t += SW, buf ^= 1) {
        // this tile is there (the wave's own loads, and its reads of the other buffer are done: their values were used)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (t + SW < t1) fetch(t + SW, buf ^ 1);
        unsigned char *ks = mine + buf * BUF, *vs = ks + KBUF;
        int t0, end;
        w.tile(t, &t0, &end);
        const bool sink = t < w.n0, partial = min(f0.top, end) - t0 < 32 || (!sink && t0 < f1.low);  // for some row
        bool bad = false;
        if (partial) {
#pragma unroll
            for (int j = 0; j < NP; ++j) bad |= take_out<T>(vs + (j * 64 + lane) * 16, &kinds[wid][j * 64 + lane]);
            bad = __any(bad);
        }
        f32x16 sc[1];
        scores<T, DQ, 1>(sc, qf, [&](int, int c) { return *(const u32x4*)(ks + ad.k[c]); });
        Values<T, DQ, DV> v0;
        if constexpr (sizeof(T) == 2) v0.read(ad, vs, 0);
        const int from = (sink ? 0 : sp.low) - t0, upto = min(sp.top, end) - t0;
        if (partial) mask<1>(sc, from, upto, lh);
        softmax<T, 1, NV, true>(r, sc, cexp);
        add_values<T, DQ, DV, 1, true>(r, sc, v0, ad, vs, lane);
        if (bad) add_nonfinite<T, DV>(r, kinds[wid], from, upto, 32, lh);
    }
    // the upper half of the waves into the lower, until one is left
    r.sum += __shfl_xor(r.sum, 32);
    float* regs = (float*)sm;
#pragma unroll
    for (int half = SW / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (wid >= half && wid < 2 * half) {
            float* to = regs + (wid - half) * (ACC / 4);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 16; ++i) to[(v * 16 + i) * 64 + lane] = r.acc[v][i];
            sms[wid - half][0][lane] = r.mx;
            sms[wid - half][1][lane] = r.sum;
        }
        __syncthreads();
        if (wid < half) {
            const float* of = regs + wid * (ACC / 4);
            const float m2 = sms[wid][0][lane], s2 = sms[wid][1][lane], mx = fmaxf(r.mx, m2);
            const float base = mx == -INFINITY ? 0.0f : mx;
            const float x = __builtin_amdgcn_exp2f((r.mx - base) * cexp), y = __builtin_amdgcn_exp2f((m2 - base) * cexp);
            r.mx = mx;
            r.sum = r.sum * x + s2 * y;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 16; ++i) r.acc[v][i] = r.acc[v][i] * x + of[(v * 16 + i) * 64 + lane] * y;
        }
    }
    if (wid || !there) return;
    if (nsplit == 1) {
        settle<T, NV>(a, r.acc, r.sum, vb, sp, 0, lh);
        const float inv = r.sum == 0.0f ? 0.0f : 1.0f / r.sum;
        T* op = (T*)a.o + b * a.o_sb + s * a.o_ss + (int64_t)(hk * G + g) * a.o_sh;
#pragma unroll
        for (int v = 0; v < NV; ++v) store_block<T>(op, r.acc[v], inv, v, lh, a.Dv);
        return;
    }
    float* ws = (float*)a.ws + ((int64_t)(unit * nrb + rb) * nsplit + split) * part_floats(NV);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 16; ++i) ws[(v * 16 + i) * 64 + lane] = r.acc[v][i];
    if (lh == 0) {
        ws[NV * 16 * 64 + lc] = r.mx;
        ws[NV * 16 * 64 + 32 + lc] = r.sum;
    }
}

// the shares of 32 rows, in their order: a wave per block of 32 columns
template <typename T, int DV>
__global__ __launch_bounds__(64 * (DV / 32)) void attn_join(va_tok_attn_args a, int nrb, int nsplit) {
    constexpr int NV = DV / 32;
    const int lane = threadIdx.x & 63, v = threadIdx.x >> 6, lc = lane & 31, lh = lane >> 5, G = a.Hq / a.Hk;
    const int rb = blockIdx.x % nrb, unit = blockIdx.x / nrb, hk = unit % a.Hk, b = unit / a.Hk;
    const AttnSeq sq = attn_seq(a, b);
    const int row = rb * 32 + lc, s = row / G, g = row - s * G;
    if (row >= sq.ql * G) return;
    const float cexp = a.scale * 1.4426950408889634f;
    const float* ws = (const float*)a.ws + (int64_t)(unit * nrb + rb) * nsplit * part_floats(NV);
    float mx = -INFINITY;
    for (int i = 0; i < nsplit; ++i) mx = fmaxf(mx, ws[i * part_floats(NV) + NV * 16 * 64 + lc]);
    const float base = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
    f32x16 acc[1];
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[0][j] = 0.0f;
    for (int i = 0; i < nsplit; ++i) {
        const float* p = ws + i * part_floats(NV);
        const float y = __builtin_amdgcn_exp2f((p[NV * 16 * 64 + lc] - base) * cexp);
        sum += p[NV * 16 * 64 + 32 + lc] * y;
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[0][j] += p[(v * 16 + j) * 64 + lane] * y;
    }
    settle<T, 1>(a, acc, sum, (const T*)a.v + b * a.v_sb + hk * a.v_sh, attn_span(a, sq, sq.first + s), v, lh);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    store_block<T>((T*)a.o + b * a.o_sb + s * a.o_ss + (int64_t)(hk * G + g) * a.o_sh, acc[0], inv, v, lh, a.Dv);
}

constexpr int64_t ROW_MAX = 1 << 22;  // elements between slots: a tile's offsets stay within 31 bits

bool attn_ok(const va_tok_attn_args& a) {
    if (a.B < 0 || a.S < 0 || a.Hk < 1 || a.Hq < a.Hk || a.Hq % a.Hk || a.slots < 0) return false;
    if (a.dtype != VA_DTYPE_BF16 && a.dtype != VA_DTYPE_F32) return false;
    if (a.D < 8 || a.D > 128 || a.D % 8 || a.Dv < 8 || a.Dv > 128 || a.Dv % 8) return false;
    if (a.frame < 0 || a.window < 0 || a.sinks < 0 || (a.slots && a.sinks >= a.slots) || a.slots > SIDE_MAX) return false;
    if (!a.frame && (a.window || a.sinks)) return false;
    if (!(a.scale > 0.0f) || !(a.scale < INFINITY)) return false;
    if ((int64_t)a.S * (a.Hq / a.Hk) > INT32_MAX - 256) return false;
    const int64_t st = a.q_sb | a.q_ss | a.q_sh | a.k_sb | a.k_ss | a.k_sh | a.v_sb | a.v_ss | a.v_sh | a.o_sb | a.o_ss | a.o_sh;
    if (st % 8 || min(a.k_ss, a.v_ss) < 0 || max(a.k_ss, a.v_ss) >= ROW_MAX) return false;
    const bool some = a.B > 0 && a.S > 0;
    if (some && (!a.q || !a.o || (a.slots && (!a.k || !a.v)))) return false;
    return !(((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.o) & 15);
}

// How a call is split: rows of 128 through LDS (nsplit 0), or 32 rows a workgroup with the keys in nsplit shares.
struct Plan {
    int nrb, nsplit;
};

Plan attn_plan(const va_tok_attn_args& a) {
    const int64_t rows = (int64_t)a.S * (a.Hq / a.Hk), units = (int64_t)a.B * a.Hk;
    if (rows > 32) return {(int)((rows + 127) / 128), 0};
    int64_t keys = a.slots;  // the most that a row block can see
    if (a.window) keys = min(keys, (int64_t)a.sinks + a.window + a.S + a.frame);
    const int64_t nrb = (rows + 31) / 32;
    // two workgroups for each of the 256 CUs, and 256 keys at least to a share
    const int64_t want = (512 + units * nrb - 1) / (units * nrb), most = (keys + 255) / 256;
    return {(int)nrb, (int)max((int64_t)1, min(want, most))};
}

int padded(int d) { return (d + 31) / 32 * 32; }

int64_t part_bytes(const va_tok_attn_args& a) { return (padded(max(a.D, a.Dv)) / 2 * 64 + 64) * 4; }

template <typename T, int DQ, int DV>
hipError_t attn_go(const va_tok_attn_args& a, hipStream_t st, Plan p) {
    const unsigned units = (unsigned)(a.B * a.Hk);
    if (p.nsplit == 0) {
        constexpr int lds = 2 * Tr<T>::KT * (Dims<T, DQ>::CS + Dims<T, DV>::CS) * 16;
        if (hipError_t e = big_lds<attn_kernel<T, DQ, DV>, lds>()) return e;
        hipLaunchKernelGGL((attn_kernel<T, DQ, DV>), dim3(units * p.nrb), dim3(256), lds, st, a, p.nrb);
        return hipGetLastError();
    }
    using S = Split<T, DQ, DV>;
    hipError_t e = big_lds<attn_split<T, DQ, DV>, S::LDS>();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((attn_split<T, DQ, DV>), dim3(units * p.nrb * p.nsplit), dim3(64 * S::SW), S::LDS, st, a, p.nrb, p.nsplit);
    e = hipGetLastError();
    if (e == hipSuccess && p.nsplit > 1) {
        hipLaunchKernelGGL((attn_join<T, DV>), dim3(units * p.nrb), dim3(64 * (DV / 32)), 0, st, a, p.nrb, p.nsplit);
        e = hipGetLastError();
    }
    return e;
}

// heads whose keys are half as wide as their values are staged as they are, others at the wider of both widths
template <typename T>
hipError_t attn_type(const va_tok_attn_args& a, hipStream_t st, Plan p) {
    if (a.D <= 32 && a.Dv > 32 && a.Dv <= 64) return attn_go<T, 32, 64>(a, st, p);
    switch (padded(max(a.D, a.Dv))) {
        case 32: return attn_go<T, 32, 32>(a, st, p);
        case 64: return attn_go<T, 64, 64>(a, st, p);
        case 96: return attn_go<T, 96, 96>(a, st, p);
        default: return attn_go<T, 128, 128>(a, st, p);
    }
}

}  // namespace

extern "C" {

int64_t va_tok_attn_workspace_bytes(const va_tok_attn_args* a) {
    if (!a || !attn_ok(*a)) return VA_ERR_ARG;
    if (a->B == 0 || a->S == 0) return 0;
    const Plan p = attn_plan(*a);
    return p.nsplit > 1 ? (int64_t)a->B * a->Hk * p.nrb * p.nsplit * part_bytes(*a) : 0;
}

int va_tok_attn(void* stream, const va_tok_attn_args* ap) {
    if (!ap || !attn_ok(*ap)) return VA_ERR_ARG;
    const va_tok_attn_args& a = *ap;
    if (a.B == 0 || a.S == 0) return VA_OK;
    const Plan p = attn_plan(a);
    if (!grid_ok((int64_t)a.B * a.Hk, p.nrb * max(p.nsplit, 1), 256)) return VA_ERR_RANGE;
    const int64_t need = va_tok_attn_workspace_bytes(ap);
    if (need > 0 && (!a.ws || a.ws_bytes < need || ((uintptr_t)a.ws & 15))) return VA_ERR_ARG;
    const hipError_t e = a.dtype == VA_DTYPE_F32 ? attn_type<float>(a, (hipStream_t)stream, p)
                                                 : attn_type<__bf16>(a, (hipStream_t)stream, p);
    return e == hipSuccess ? VA_OK : VA_ERR_HIP;
}

}  // extern "C"
