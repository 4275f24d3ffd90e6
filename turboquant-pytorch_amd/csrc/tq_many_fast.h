// Attention of tiles of queries over packed tokens at head dimensions 64, 65 to 96, 128 and 256, codes of one, two or four to a byte (tq_many.hip).
// One source file per padded head dimension instantiates it.
#pragma once
#include <type_traits>

#include "tq_many.h"
#include "tq_lut.h"

namespace {

constexpr int FAST_WAVES = 8;                // one block per compute unit, two waves per SIMD, which share the tables
constexpr int FAST_THREADS = 64 * FAST_WAVES;
static_assert(FAST_THREADS == LUT_THREADS, "threads that stage the tables");
constexpr int FAST_APART = 12;               // queries of a block are scaled together unless one is smaller than the largest by 2^12 or more
constexpr int FAST_SLACK = 8;                // a column's reference moves when a logit exceeds it by more than this
constexpr int FAST_P = 14 - FAST_SLACK;      // weights enter the products times 2^FAST_P, at most 2^14; value norms below 2 in their unit

// A head dimension as the kernels work on it: DP, the next multiple of 32.  64, 128 and 256 are taken as they are; for others (EVEN false, a.D below DP possible) packed
// bytes go through LDS, where they may lie anywhere.  On the value side a lane has NC coordinates in a row, NC n ... NC n + NC - 1, of which the first LANES lanes' exist.
template <int DP>
struct Shape {
    static constexpr bool EVEN = DP == 64 || DP == 128 || DP == 256;
    static constexpr int NC = EVEN ? DP / 32 : DP <= 128 ? 4 : 8, LANES = DP / NC, TILES = DP / 32, STEPS = DP / 16;
};

// A table of two fp16 terms a level: an entry is the byte's leading terms, then the rests; spread over the banks as Lut does.
template <int IPB>
struct Lut2 {
    static constexpr int ROWS = 4;
    uint32_t t[ROWS][IPB];
    __device__ __forceinline__ void load(const uint8_t *table, uint32_t bits, uint32_t D, uint32_t tid) {
        const TQ_GLOBAL float *level = (const TQ_GLOBAL float *)(table + TQ_OFF_LUT(D) + 512u * IPB);
        const uint32_t mask = (1u << bits) - 1u;
#pragma unroll
        for (int k = 0; k < ROWS; ++k)
#pragma unroll
            for (int c = 0; c < IPB; ++c) t[k][c] = __float_as_uint(level[((((tid >> 3) * ROWS + k) >> (bits * (IPB - 1 - c))) & mask)]);
    }
    __device__ __forceinline__ void store(uint8_t *lds, uint32_t tid) {
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            uint32_t e[IPB];
#pragma unroll
            for (int c = 0; c < IPB; ++c) e[c] = fp16_terms(__uint_as_float(t[k][c]) * (float)(1 << LEVEL_SHIFT));
            tq_u4 x;
            if constexpr (IPB == 1) x = tq_u4{e[0], e[0], e[0], e[0]};
            else if constexpr (IPB == 2) {
                const uint32_t hi = __builtin_amdgcn_perm(e[1], e[0], 0x05040100u), lo = __builtin_amdgcn_perm(e[1], e[0], 0x07060302u);
                x = tq_u4{hi, lo, hi, lo};
            } else {
                x = tq_u4{__builtin_amdgcn_perm(e[1], e[0], 0x05040100u), __builtin_amdgcn_perm(e[3], e[2], 0x05040100u),
                          __builtin_amdgcn_perm(e[1], e[0], 0x07060302u), __builtin_amdgcn_perm(e[3], e[2], 0x07060302u)};
            }
            *reinterpret_cast<tq_u4 *>(lds + ((tid >> 3) * ROWS + k) * 256u + (tid & 7u) * 16u) = x;
        }
    }
    static __device__ __forceinline__ uint32_t lane_offset(uint32_t lane) { return (lane & (32u / IPB - 1u)) * 4u * IPB; }
};

// The eight coordinates of step s among a lane's key bytes -> operands of both terms
template <int IPB, int NW>
__device__ __forceinline__ void decode_keys2(const uint32_t (&raw)[NW], int s, const uint8_t *lut, uint32_t slot, tq_u4 &hi, tq_u4 &lo) {
    if constexpr (IPB == 1) {
        uint32_t t[8];
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const uint32_t r = raw[2 * s + d];
            t[4 * d] = lut_entry<0, uint32_t>(lut, r, slot);
            t[4 * d + 1] = lut_entry<1, uint32_t>(lut, r, slot);
            t[4 * d + 2] = lut_entry<2, uint32_t>(lut, r, slot);
            t[4 * d + 3] = lut_entry<3, uint32_t>(lut, r, slot);
        }
        fp16_operands(t, hi, lo);
    } else if constexpr (IPB == 2) {
        const tq_u2 a = lut_entry<0, tq_u2>(lut, raw[s], slot), b = lut_entry<1, tq_u2>(lut, raw[s], slot);
        const tq_u2 c = lut_entry<2, tq_u2>(lut, raw[s], slot), d = lut_entry<3, tq_u2>(lut, raw[s], slot);
        hi = tq_u4{a[0], b[0], c[0], d[0]};
        lo = tq_u4{a[1], b[1], c[1], d[1]};
    } else {
        const uint32_t r = raw[s / 2];
        const tq_u4 a = s % 2 ? lut_entry<2, tq_u4>(lut, r, slot) : lut_entry<0, tq_u4>(lut, r, slot);
        const tq_u4 b = s % 2 ? lut_entry<3, tq_u4>(lut, r, slot) : lut_entry<1, tq_u4>(lut, r, slot);
        hi = tq_u4{a[0], a[1], b[0], b[1]};
        lo = tq_u4{a[2], a[3], b[2], b[3]};
    }
}

// A lane's share of a value vector: coordinates NC n ... NC n + NC - 1, VB bytes (64 wide, four codes a byte: half of one)
template <int IPB, int NC>
struct ValueBytes {
    static constexpr int VB = NC >= IPB ? NC / IPB : 1, W = VB > 4 ? 2 : 1;
    uint32_t raw[W];
    __device__ __forceinline__ void load(const uint8_t *p) {
        if constexpr (VB == 1) raw[0] = *((const TQ_GLOBAL uint8_t *)p);
        else if constexpr (VB == 2) raw[0] = tq_gload2(reinterpret_cast<const uint16_t *>(p));
        else if constexpr (VB == 4) raw[0] = tq_gload4(p);
        else { const tq_u2 v = tq_gload8(p); raw[0] = v[0]; raw[W - 1] = v[1]; }
    }
    __device__ __forceinline__ void fetch(const uint8_t *p) {          // from LDS
        if constexpr (VB == 1) raw[0] = *p;
        else if constexpr (VB == 2) raw[0] = *reinterpret_cast<const uint16_t *>(p);
        else if constexpr (VB == 4) raw[0] = *reinterpret_cast<const uint32_t *>(p);
        else { const tq_u2 v = *reinterpret_cast<const tq_u2 *>(p); raw[0] = v[0]; raw[W - 1] = v[1]; }
    }
    // fp16 pairs; slot: the lane's slot of entry 0 (64 wide, four codes a byte: of its half)
    __device__ __forceinline__ void decode(const uint8_t *lut, uint32_t slot, uint32_t (&out)[NC / 2]) const {
        if constexpr (IPB == 4 && NC == 2) out[0] = lut_entry<0, uint32_t>(lut, raw[0], slot);
        else if constexpr (IPB == 4) {
            const tq_u2 a = lut_entry<0, tq_u2>(lut, raw[0], slot);
            out[0] = a[0]; out[1] = a[1];
            if constexpr (NC == 8) { const tq_u2 b = lut_entry<1, tq_u2>(lut, raw[0], slot); out[2] = b[0]; out[3] = b[1]; }
        } else if constexpr (IPB == 2) {
            out[0] = lut_entry<0, uint32_t>(lut, raw[0], slot);
            if constexpr (NC >= 4) out[1] = lut_entry<1, uint32_t>(lut, raw[0], slot);
            if constexpr (NC == 8) { out[2] = lut_entry<2, uint32_t>(lut, raw[0], slot); out[3] = lut_entry<3, uint32_t>(lut, raw[0], slot); }
        } else {
#pragma unroll
            for (int i = 0; i < NC / 2; i += 2) {
                const uint32_t r = raw[i / 2 < W ? i / 2 : 0];
                out[i] = (uint32_t)lut_entry<0, uint16_t>(lut, r, slot) | ((uint32_t)lut_entry<1, uint16_t>(lut, r, slot) << 16);
                if constexpr (NC > 2) out[i + 1] = (uint32_t)lut_entry<2, uint16_t>(lut, r, slot) | ((uint32_t)lut_entry<3, uint16_t>(lut, r, slot) << 16);
            }
        }
    }
};

// The same from a table of two terms: leading terms and rests
template <int IPB, int NC>
__device__ __forceinline__ void decode_values2(const ValueBytes<IPB, NC> &v, const uint8_t *lut, uint32_t slot, uint32_t odd, uint32_t (&hi)[NC / 2], uint32_t (&lo)[NC / 2]) {
    if constexpr (IPB == 1) {
#pragma unroll
        for (int i = 0; i < NC / 2; i += 2) {
            const uint32_t r = v.raw[i / 2 < ValueBytes<IPB, NC>::W ? i / 2 : 0];
            const uint32_t a = lut_entry<0, uint32_t>(lut, r, slot), b = lut_entry<1, uint32_t>(lut, r, slot);
            hi[i] = __builtin_amdgcn_perm(b, a, 0x05040100u); lo[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            if constexpr (NC > 2) {
                const uint32_t c = lut_entry<2, uint32_t>(lut, r, slot), d = lut_entry<3, uint32_t>(lut, r, slot);
                hi[i + 1] = __builtin_amdgcn_perm(d, c, 0x05040100u); lo[i + 1] = __builtin_amdgcn_perm(d, c, 0x07060302u);
            }
        }
    } else if constexpr (IPB == 2) {
        tq_u2 e[NC / 2];
        e[0] = lut_entry<0, tq_u2>(lut, v.raw[0], slot);
        if constexpr (NC >= 4) e[NC / 2 > 1 ? 1 : 0] = lut_entry<1, tq_u2>(lut, v.raw[0], slot);
        if constexpr (NC == 8) { e[2] = lut_entry<2, tq_u2>(lut, v.raw[0], slot); e[3] = lut_entry<3, tq_u2>(lut, v.raw[0], slot); }
#pragma unroll
        for (int i = 0; i < NC / 2; ++i) { hi[i] = e[i][0]; lo[i] = e[i][1]; }
    } else {
        const tq_u4 a = lut_entry<0, tq_u4>(lut, v.raw[0], slot);
        if constexpr (NC == 2) { hi[0] = odd ? a[1] : a[0]; lo[0] = odd ? a[3] : a[2]; }
        else {
            hi[0] = a[0]; hi[1] = a[1]; lo[0] = a[2]; lo[1] = a[3];
            if constexpr (NC == 8) { const tq_u4 b = lut_entry<1, tq_u4>(lut, v.raw[0], slot); hi[2] = b[0]; hi[3] = b[1]; lo[2] = b[2]; lo[3] = b[3]; }
        }
    }
}

// Packed keys of 32 tokens: a lane's share is half a token, D / 2 coordinates.  issue() asks for them; where the shape is not even, stage() puts the bytes into LDS and take() reads them
// from there (what lies past a vector's end are codes of anything, against queries of zero).
template <int DP, int IPB>
struct KeyRun {
    static constexpr bool EVEN = Shape<DP>::EVEN;
    static constexpr int KB = DP / 2 / IPB, KW = KB / 4, GB = DP / IPB, PIECES = (GB + 7) / 8;      // (words of a run per lane)
    uint32_t raw[KW], piece[EVEN ? 1 : PIECES];
    __device__ __forceinline__ void issue(const uint8_t *run, uint32_t bytes, uint32_t lane) {          // bytes: of a token
        const uint32_t n = lane & 31u, h = lane >> 5;
        if constexpr (!EVEN) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) piece[i] = tq_gload4(run + 4u * min(64u * i + lane, 8u * bytes - 1u));
        } else if constexpr (KB % 16 == 0) {
#pragma unroll
            for (int i = 0; i < KB / 16; ++i) {
                const tq_u4 v = tq_gload16(run + (n * GB + h * KB) + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[4 * i + j] = v[j];
            }
        } else {
            static_assert(KB % 16 == 0 || KB == 8 || !EVEN, "eight bytes");
            const tq_u2 v = tq_gload8(run + (n * GB + h * KB));
            raw[0] = v[0]; raw[KW > 1 ? 1 : 0] = v[1];
        }
    }
    __device__ __forceinline__ void stage(uint8_t *lds, uint32_t lane) const {
        if constexpr (!EVEN) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                if (64 * i + 64 <= 8 * GB || 64u * i + lane < 8u * GB) *reinterpret_cast<uint32_t *>(lds + 4u * (64u * i + lane)) = piece[i];
        }
    }
    __device__ __forceinline__ void take(const uint8_t *lds, uint32_t bytes, uint32_t lane) {
        if constexpr (!EVEN) {
            const uint8_t *p = lds + (lane & 31u) * bytes + (lane >> 5) * KB;
#pragma unroll
            for (int i = 0; i < KW; ++i) raw[i] = *reinterpret_cast<const uint32_t *>(p + 4 * i);
        }
    }
    static constexpr uint32_t BYTES = EVEN ? 0u : 32u * GB;
};

// Eight 16-bit elements from any address
__device__ __forceinline__ tq_u4 load_elements(const uint8_t *p, bool aligned) {
    if (aligned) return tq_gload16(p);
    tq_u4 v;
#pragma unroll
    for (int d = 0; d < 4; ++d)
        v[d] = (uint32_t)tq_gload2(reinterpret_cast<const uint16_t *>(p) + 2 * d) | ((uint32_t)tq_gload2(reinterpret_cast<const uint16_t *>(p) + 2 * d + 1) << 16);
    return v;
}

// Queries of QT tiles into the codec's space, q' = scale * log2(e) * Pi_k q, as fp16 operands in LDS ([tile][term][step][lane], as q_operand_bytes says): wave (tile i, w)
// has coordinates 32 w ... + 31.  Pi as three bf16 terms, or for fp16 queries two fp16 ones (22 bits).  All queries are scaled by the power of two
// that puts their largest coordinate into [2^Q_TOP, 2^(Q_TOP + 1)); finish() answers with what products with them are to be multiplied by.  Queries 2^FAST_APART times smaller
// than the largest, and fp16 reaches no further than 2^14 below that for their smaller coordinates, make each query have a power of its own (`apart`): its products are then to be
// multiplied by its entry of `own` first.  What a row of padding holds would otherwise take the bits of the others.  load() asks for everything, so that other loads
// can be under way before finish() waits.
template <int DP, int QT, int KT, int DT>
struct Rotate {
    static constexpr int TILES = Shape<DP>::TILES, STEPS = DP / 16, CH = DT == TQ_F32 ? 2 : STEPS < 8 ? STEPS : STEPS % 8 ? STEPS / 2 : 8, TERMS = DT == TQ_F16 ? 2 : 3, NT = DT == TQ_F32 ? 3 : 1;
    static_assert(STEPS % CH == 0 && QT * TILES <= FAST_WAVES, "whole chunks, waves that rotate");
    tq_u4 x[CH][NT], p[TERMS][CH];
    const uint8_t *q, *pi;
    uint32_t i, w, m;
    __device__ __forceinline__ void fetch(const TqManyArgs &a, int s0, uint32_t h) {
#pragma unroll
        for (int s = 0; s < CH; ++s)
#pragma unroll
            for (int t = 0; t < TERMS; ++t) p[t][s] = tq_gload16(pi + (size_t)t * TQ_OPERAND_BYTES_FOR(DP) + (size_t)(s0 + s) * 1024u);
        if constexpr (DT == TQ_F32) {
#pragma unroll
            for (int s = 0; s < CH; ++s) {
                tq_u4 t[3];
                load_plain8<TQ_F32>(q, 16u * (s0 + s) + 8u * h, a.D, a.aligned, t);
#pragma unroll
                for (int k = 0; k < NT; ++k) x[s][k] = t[k];
            }
        } else if (a.aligned) {
#pragma unroll
            for (int s = 0; s < CH; ++s) {
                const uint32_t d = 16u * (s0 + s) + 8u * h;
                x[s][0] = tq_gload16(q + 2u * (Shape<DP>::EVEN ? d : min(d, a.D - 8u)));
                if (!Shape<DP>::EVEN && d >= a.D) x[s][0] = tq_u4{0u, 0u, 0u, 0u};
            }
        } else {
#pragma unroll
            for (int s = 0; s < CH; ++s) {
                const uint32_t d = 16u * (s0 + s) + 8u * h;
                x[s][0] = load_elements(q + 2u * (Shape<DP>::EVEN ? d : min(d, a.D - 8u)), false);
                if (!Shape<DP>::EVEN && d >= a.D) x[s][0] = tq_u4{0u, 0u, 0u, 0u};
            }
        }
    }
    __device__ __forceinline__ void load(const TqManyArgs &a, uint32_t row, uint32_t tile0, uint32_t wave, uint32_t lane) {
        i = wave / TILES;
        w = wave % TILES;
        m = (tile0 + i) * 32u + (lane & 31u);
        if (i >= (uint32_t)QT) return;
        q = many_query(a, row, min(m, a.M - 1u), DT == TQ_F32 ? 4u : 2u);
        pi = a.table_k + (DT == TQ_F16 ? TQ_OFF_A_F16 : TQ_OFF_A_BF16(DP)) + ((size_t)w * STEPS * 64u + lane) * 16u;
        fetch(a, 0, lane >> 5);
    }
    __device__ __forceinline__ float finish(const TqManyArgs &a, uint8_t *ops, float (*lds_top)[32], float (*own)[32], bool &apart, uint32_t wave, uint32_t lane) {
        const uint32_t n = lane & 31u, h = lane >> 5;
        float y[16], top = 0.f;
        if (i < (uint32_t)QT) {
            tq_f16v acc = tq_zero16();
#pragma unroll 1
            for (int s0 = 0;;) {
#pragma unroll
                for (int s = 0; s < CH; ++s)
#pragma unroll
                    for (int t = 0; t < TERMS; ++t)
#pragma unroll
                        for (int k = 0; k < NT; ++k)
                            if (t + k < 3) acc = DT == TQ_F16 ? mfma_f16(p[t][s], x[s][k], acc) : mfma_bf16(p[t][s], x[s][k], acc);
                s0 += CH;
                if (s0 >= STEPS) break;
                fetch(a, s0, h);
            }
            const float f = a.scale * (DT == TQ_F16 ? LOG2E / (float)(1 << TQ_F16_PI_SHIFT) : LOG2E);
#pragma unroll
            for (int r = 0; r < 16; ++r) {       // (the table's rows: register r of half h is coordinate 32 w + 16 h + r)
                y[r] = m < a.M ? acc[r] * f : 0.f;
                const float v = fabsf(y[r]);
                top = fmaxf(top, v < __builtin_inff() ? v : 0.f);
            }
            top = halves_max(top);
        }
        if (h == 0u) lds_top[wave][n] = top;
        __syncthreads();
        float of[QT];                            // largest coordinate of this column's query of each tile
        top = 0.f;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            of[t] = 0.f;
#pragma unroll
            for (int k = 0; k < TILES; ++k) of[t] = fmaxf(of[t], lds_top[t * TILES + k][n]);
            top = fmaxf(top, of[t]);
        }
        top = reduce_wave(top, OpMax());
        bool far = false;
#pragma unroll
        for (int t = 0; t < QT; ++t) far = far || (of[t] > 0.f && of[t] * (float)(1 << FAST_APART) <= top);
        apart = __any(far);
        const int up = query_shift(top);
        float f = __uint_as_float((uint32_t)(up + 127) << 23);
        if (apart) {
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const int mine = of[t] > 0.f ? min(query_shift(of[t]), up + 120) : up;        // (so that the entry is a normal number)
                if (i == (uint32_t)t) f = __uint_as_float((uint32_t)(mine + 127) << 23);
                if (wave == (uint32_t)t && h == 0u) own[t][n] = __uint_as_float((uint32_t)(127 + up - mine) << 23);
            }
        }
        if (i < (uint32_t)QT) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                tq_u4 hi, lo;
                fp16_split8(tq_f4{y[8 * j], y[8 * j + 1], y[8 * j + 2], y[8 * j + 3]}, tq_f4{y[8 * j + 4], y[8 * j + 5], y[8 * j + 6], y[8 * j + 7]}, f, hi, lo);
                const uint32_t d = 32u * w + 16u * h + 8u * j, half = d / (DP / 2u), s = (d - half * (DP / 2u)) / 8u;
                uint8_t *o = ops + ((i * KT * STEPS + s) * 64u + half * 32u + n) * 16u;
                *reinterpret_cast<tq_u4 *>(o) = hi;
                if constexpr (KT == 2) *reinterpret_cast<tq_u4 *>(o + STEPS * 1024u) = lo;
            }
        }
        return __uint_as_float((uint32_t)(127 - up - (KT == 2 ? LEVEL_SHIFT : 0)) << 23);
    }
};

// 32 uncompressed tokens of a row (`which`: 0 the window, 1 the drafts; from t0 on) against a tile of queries: raw 16-bit products are exact, weights enter the value
// product as three bf16 terms, or two fp16 ones.  Coordinates of the sums as in the packed loop: row r of acc[c] is coordinate NC r + c.  Infinite and NaN
// values count as zero here (a product would spread them to queries that do not see their token as 0 * inf); `wild` says whether there are any.
// Up to 128 wide all loads of the 32 tokens are under way at once (HELD), at 256 they would not fit into registers and are issued as they are needed.
template <int DP, int DT>
struct PlainTile {
    static constexpr bool BF = DT == TQ_BF16, EVEN = Shape<DP>::EVEN;
    static constexpr int NC = Shape<DP>::NC, STEPS = DP / 16, PT = BF ? 3 : 2;
    static constexpr bool HELD = DP <= 128;
    static constexpr int VT = HELD ? 16 : 8, KH = HELD ? STEPS : 1;       // VT: tokens whose values are held at a time
    static constexpr uint32_t EXPO = BF ? 0x7f807f80u : 0x7c007c00u, ONE = BF ? 0x00800080u : 0x04000400u;
    uint32_t vw[VT][NC / 2];
    tq_u4 kx[KH];
    const uint8_t *k, *v;
    uint32_t which, t0;
    bool wild;

    // elements 16 st + 8 h ... + 7 of a vector, zeros from D on (a multiple of 8)
    static __device__ __forceinline__ tq_u4 half_step(const uint8_t *vec, int st, uint32_t h, uint32_t D, bool aligned) {
        const uint32_t d = 16u * st + 8u * h;
        const tq_u4 v = load_elements(vec + 2u * (EVEN ? d : min(d, D - 8u)), aligned);
        return EVEN || d < D ? v : tq_u4{0u, 0u, 0u, 0u};
    }
    __device__ __forceinline__ void load_values(const TqManyArgs &a, int j0, uint32_t h) {
        const TqManyPlain &seg = a.plain[which];
#pragma unroll
        for (int j = 0; j < VT; ++j) {
            const uint8_t *p = v + (long long)min(t0 + acc_row(j0 + j, h), seg.n - 1u) * seg.v_token * 2;
            if (a.aligned) {
                if constexpr (NC == 2) vw[j][0] = tq_gload4(p);
                else if constexpr (NC == 4) { const tq_u2 x = tq_gload8(p); vw[j][0] = x[0]; vw[j][1] = x[1]; }
                else { const tq_u4 x = tq_gload16(p); vw[j][0] = x[0]; vw[j][1] = x[1]; vw[j][NC / 2 - 2] = x[2]; vw[j][NC / 2 - 1] = x[3]; }
            } else {
#pragma unroll
                for (int c = 0; c < NC / 2; ++c)
                    vw[j][c] = (uint32_t)tq_gload2(reinterpret_cast<const uint16_t *>(p) + 2 * c) | ((uint32_t)tq_gload2(reinterpret_cast<const uint16_t *>(p) + 2 * c + 1) << 16);
            }
        }
    }
    __device__ __forceinline__ void tame_values(const TqManyArgs &a, int j0, uint32_t h) {
        uint32_t over = 0u;
#pragma unroll
        for (int j = 0; j < VT; ++j)
#pragma unroll
            for (int c = 0; c < NC / 2; ++c) {
                if (t0 + acc_row(j0 + j, h) >= a.plain[which].n) vw[j][c] = 0u;
                over |= (vw[j][c] & EXPO) + ONE;         // (an exponent of ones carries into the sign's place)
            }
        if (__any((over & 0x80008000u) != 0u)) {
            wild = true;
#pragma unroll
            for (int j = 0; j < VT; ++j)
#pragma unroll
                for (int c = 0; c < NC / 2; ++c) vw[j][c] &= ~(((((vw[j][c] & EXPO) + ONE) >> 15) & 0x00010001u) * 0xffffu);
        }
    }
    __device__ __forceinline__ void load(const TqManyArgs &a, uint32_t which_, uint32_t t0_, uint32_t row, uint32_t b, uint32_t lane) {
        which = which_;
        t0 = t0_;
        const TqManyPlain &seg = a.plain[which];
        const uint32_t n = lane & 31u, h = lane >> 5, kv = row - b * a.heads;
        k = seg.k + ((long long)b * seg.k_batch + (long long)kv * seg.k_head + (long long)min(t0 + n, seg.n - 1u) * seg.k_token) * 2;
        v = seg.v + ((long long)b * seg.v_batch + (long long)kv * seg.v_head) * 2 + 2u * NC * (EVEN ? n : min(n, a.D / NC - 1u));
        if constexpr (HELD) {
            if (a.aligned) {
#pragma unroll
                for (int st = 0; st < STEPS; ++st) kx[st] = half_step(k, st, h, a.D, true);
            } else {
#pragma unroll 1
                for (int st = 0; st < STEPS; ++st) {
                    const tq_u4 x = half_step(k, st, h, a.D, false);
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) kx[i] = i == st ? x : kx[i];
                }
            }
            load_values(a, 0, h);
            tame_values(a, 0, h);
        }
    }
    __device__ __forceinline__ void attend(const TqManyArgs &a, uint32_t row, uint32_t b, uint32_t tile, uint32_t length, uint32_t lane, float &m_ref, float &l, tq_f16v (&acc)[NC]) {
        const TqManyPlain &seg = a.plain[which];
        const uint32_t n = lane & 31u, h = lane >> 5, m = min(tile * 32u + n, a.M - 1u);
        const uint8_t *q = many_query(a, row, m, 2u);
        tq_f16v s = tq_zero16();
        if (a.aligned) {
            constexpr int CH = HELD ? STEPS : 4;
#pragma unroll 1
            for (int s0 = 0; s0 < STEPS; s0 += CH) {
                tq_u4 x[CH], y[CH];
#pragma unroll
                for (int st = 0; st < CH; ++st) {
                    x[st] = HELD ? kx[HELD ? st : 0] : half_step(k, s0 + st, h, a.D, true);
                    y[st] = half_step(q, s0 + st, h, a.D, true);
                }
#pragma unroll
                for (int st = 0; st < CH; ++st) s = BF ? mfma_bf16(x[st], y[st], s) : mfma_f16(x[st], y[st], s);
            }
        } else {
#pragma unroll 1
            for (int st = 0; st < STEPS; ++st) {
                const tq_u4 x = half_step(k, st, h, a.D, false), y = half_step(q, st, h, a.D, false);
                s = BF ? mfma_bf16(x, y, s) : mfma_f16(x, y, s);
            }
        }
        const uint32_t own = ManyQuery(a, m).t;
        float x[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint32_t t = t0 + acc_row(r, h);
            x[r] = t < seg.n && plain_seen(a, which, b, own, t, length) ? s[r] * (a.scale * LOG2E) : MANY_NONE;
        }
        float top = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
        top = fmaxf(halves_max(top), m_ref);
        const float shrink = __builtin_amdgcn_exp2f(m_ref - top);
        m_ref = top;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[r] = x[r] == MANY_NONE ? 0.f : __builtin_amdgcn_exp2f(x[r] - top);
            sum += x[r];
        }
        l = l * shrink + sum;          // (this lane's half)
        if (__any(shrink != 1.f)) {
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[c] *= shrink;
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            if constexpr (!HELD) {
                load_values(a, 8 * st, h);
                tame_values(a, 8 * st, h);
            }
            tq_u4 p[3];
            float ps[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) ps[j] = x[8 * st + j];
            if constexpr (BF) bf16_terms(ps, p);
            else {
                uint32_t t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = fp16_terms(ps[j]);
                fp16_operands(t, p[0], p[1]);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                tq_u4 o;
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    o[d] = __builtin_amdgcn_perm(vw[(HELD ? 8 * st : 0) + 2 * d + 1][c / 2], vw[(HELD ? 8 * st : 0) + 2 * d][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int t = 0; t < PT; ++t) acc[c] = BF ? mfma_bf16(o, p[t], acc[c]) : mfma_f16(o, p[t], acc[c]);
            }
        }
    }
};

// The same for float32 elements: three bf16 terms of everything, products down to 2^-24 of the largest.
template <int DP>
struct PlainTile<DP, TQ_F32> {
    static constexpr int NC = Shape<DP>::NC, STEPS = DP / 16;
    const uint8_t *k, *v;
    uint32_t which, t0;
    bool wild;
    __device__ __forceinline__ void load(const TqManyArgs &a, uint32_t which_, uint32_t t0_, uint32_t row, uint32_t b, uint32_t lane) {
        which = which_;
        t0 = t0_;
        const TqManyPlain &seg = a.plain[which];
        const uint32_t n = lane & 31u, kv = row - b * a.heads;
        k = seg.k + ((long long)b * seg.k_batch + (long long)kv * seg.k_head + (long long)min(t0 + n, seg.n - 1u) * seg.k_token) * 4;
        v = seg.v + ((long long)b * seg.v_batch + (long long)kv * seg.v_head) * 4 + 4u * NC * min(n, a.D / NC - 1u);
    }
    __device__ __forceinline__ void attend(const TqManyArgs &a, uint32_t row, uint32_t b, uint32_t tile, uint32_t length, uint32_t lane, float &m_ref, float &l, tq_f16v (&acc)[NC]) {
        const TqManyPlain &seg = a.plain[which];
        const uint32_t n = lane & 31u, h = lane >> 5, m = min(tile * 32u + n, a.M - 1u);
        const uint8_t *q = many_query(a, row, m, 4u);
        tq_f16v s = tq_zero16();
#pragma unroll 1
        for (int st = 0; st < STEPS; ++st) {
            tq_u4 kt[3], qt[3];
            load_plain8<TQ_F32>(k, 16u * st + 8u * h, a.D, a.aligned, kt);
            load_plain8<TQ_F32>(q, 16u * st + 8u * h, a.D, a.aligned, qt);
#pragma unroll
            for (int i = 0; i < 3; ++i)
#pragma unroll
                for (int j = 0; j < 3 - i; ++j) s = mfma_bf16(kt[i], qt[j], s);
        }
        const uint32_t own = ManyQuery(a, m).t;
        float x[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint32_t t = t0 + acc_row(r, h);
            x[r] = t < seg.n && plain_seen(a, which, b, own, t, length) ? s[r] * (a.scale * LOG2E) : MANY_NONE;
        }
        float top = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
        top = fmaxf(halves_max(top), m_ref);
        const float shrink = __builtin_amdgcn_exp2f(m_ref - top);
        m_ref = top;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[r] = x[r] == MANY_NONE ? 0.f : __builtin_amdgcn_exp2f(x[r] - top);
            sum += x[r];
        }
        l = l * shrink + sum;
        if (__any(shrink != 1.f)) {
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[c] *= shrink;
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            float ps[8], e[8][NC];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ps[j] = x[8 * st + j];
                const uint32_t t = t0 + acc_row(8 * st + j, h);
                const uint8_t *p = v + (long long)min(t, seg.n - 1u) * seg.v_token * 4;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float value = t < seg.n ? plain_element(p + 4 * c, TQ_F32) : 0.f;
                    const bool fine = fabsf(value) < __builtin_inff();
                    wild = wild || !fine;
                    e[j][c] = fine ? value : 0.f;
                }
            }
            tq_u4 p[3];
            bf16_terms(ps, p);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float own8[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) own8[j] = e[j][c];
                tq_u4 vt[3];
                bf16_terms(own8, vt);
#pragma unroll
                for (int i = 0; i < 3; ++i)
#pragma unroll
                    for (int j = 0; j < 3 - i; ++j) acc[c] = mfma_bf16(vt[i], p[j], acc[c]);
            }
        }
    }
};

// The sums of waves [w0, w0 + COUNT) of a tile of queries into out[32][D + 4] and their largest logits and sums into out_m, out_l[32], all in LDS; every wave of the block
// calls it, those with other w0 for another tile.  unit: what this wave's value sums are multiplied by; m_ref: MANY_NONE where it has seen no token of a
// query; l: this lane's half.  area: [wave][32][64 + 4], two coordinates blocks of 32 at a time.
template <int DP, int COUNT>
__device__ __forceinline__ void join_waves(float *area, float (*lds_m)[32], float (*lds_l)[32], float *out, float *out_m, float *out_l, uint32_t w0, float unit, float m_ref,
                                           float l, const tq_f16v (&acc)[Shape<DP>::NC], uint32_t tid) {
    constexpr int NC = Shape<DP>::NC;
    constexpr uint32_t MROW = 68u, ROW = DP + 4;
    const uint32_t lane = tid & 63u, wave = tq_uniform32(tid >> 6), n = lane & 31u, h = lane >> 5;
    const float both = halves_add(l);
    if (h == 0u) {
        lds_m[wave][n] = m_ref;
        lds_l[wave][n] = both;
    }
    __syncthreads();
    float m = MANY_NONE, sum = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < COUNT; ++w) m = fmaxf(m, lds_m[w0 + w][n]);
#pragma unroll
    for (uint32_t w = 0; w < COUNT; ++w) sum = fmaf(lds_l[w0 + w][n], __builtin_amdgcn_exp2f(lds_m[w0 + w][n] - m), sum);
    if (wave == w0 && h == 0u) {
        out_m[n] = m;
        out_l[n] = sum;
    }
    const float f = unit * __builtin_amdgcn_exp2f(m_ref - m);
    const uint32_t mine = tid - w0 * 64u;       // (a wave sums for its own tile)
#pragma unroll
    for (int c0 = 0; c0 < NC; c0 += 2) {
        if (c0) __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<tq_f4 *>(area + (wave * 32u + n) * MROW + 32 * c + 8 * k + 4 * h) =
                    tq_f4{acc[c0 + c][4 * k] * f, acc[c0 + c][4 * k + 1] * f, acc[c0 + c][4 * k + 2] * f, acc[c0 + c][4 * k + 3] * f};
        __syncthreads();
#pragma unroll
        for (uint32_t pair0 = 0; pair0 < 1024u; pair0 += COUNT * 64u) {        // coordinates NC r + c0, + 1 of query col
            const uint32_t pair = pair0 + mine, col = pair / 32u, r = pair % 32u;
            if (Shape<DP>::LANES < 32 && r >= (uint32_t)Shape<DP>::LANES) continue;
            float x = 0.f, y = 0.f;
#pragma unroll
            for (uint32_t w = 0; w < COUNT; ++w) {
                x += area[((w0 + w) * 32u + col) * MROW + r];
                y += area[((w0 + w) * 32u + col) * MROW + 32u + r];
            }
            out[col * ROW + NC * r + c0] = x;
            out[col * ROW + NC * r + c0 + 1] = y;
        }
    }
}

// joined sums of a tile -> its record
template <int DP>
__device__ __forceinline__ void put_record(float *rec, const float *out, const float *out_m, const float *out_l, uint32_t tid) {
    TQ_GLOBAL float *p = (TQ_GLOBAL float *)rec;
    if (tid < 32u) { p[tid] = out_m[tid]; p[32u + tid] = out_l[tid]; }
    for (uint32_t u = tid; u < 32u * DP / 4u; u += FAST_THREADS) {
        const uint32_t col = u / (DP / 4u), d = (u - col * (DP / 4u)) * 4u;
        *reinterpret_cast<TQ_GLOBAL tq_f4 *>(p + 64u + col * DP + d) = *reinterpret_cast<const tq_f4 *>(out + col * (DP + 4u) + d);
    }
}

// Infinite and NaN values of a row's uncompressed tokens into the joined sums of the queries that see them, whatever their weight (it is not zero).
template <int DP>
__device__ __forceinline__ void add_wild(const TqManyArgs &a, float *out, uint32_t row, uint32_t b, uint32_t tile, uint32_t length, uint32_t tid) {
    const uint32_t kv = row - b * a.heads, elem = a.dtype;
#pragma unroll 1
    for (uint32_t e = tid; e < 32u * a.D; e += FAST_THREADS) {
        const uint32_t col = e / a.D, d = e - col * a.D, m = tile * 32u + col;
        if (m >= a.M) return;
        const uint32_t own = ManyQuery(a, m).t;
        float sum = 0.f;
#pragma unroll 1
        for (uint32_t which = 0; which < 2u; ++which) {
            const TqManyPlain &seg = a.plain[which];
#pragma unroll 1
            for (uint32_t t = 0; t < seg.n; ++t) {
                const float v = plain_element(seg.v + ((long long)b * seg.v_batch + (long long)kv * seg.v_head + (long long)t * seg.v_token + d) * (elem == TQ_F32 ? 4 : 2), elem);
                if (!(fabsf(v) < __builtin_inff()) && plain_seen(a, which, b, own, t, length)) sum += v;
            }
        }
        if (sum != 0.f) out[col * (DP + 4u) + d] += sum;
    }
}

// LDS once the packed tokens are done with: what waves join their sums through, and the joined sums of packed and uncompressed tokens of each tile
template <int DP, int QT>
struct JoinArea {
    static constexpr uint32_t TILE = 32u * (DP + 4u) * 4u, JOIN = FAST_WAVES * 32u * 68u * 4u, PACKED = JOIN, PLAIN = PACKED + QT * TILE, STATS = PLAIN + QT * TILE, BYTES = STATS + 4u * QT * 128u;
    static __device__ __forceinline__ float *sums(uint8_t *lds, uint32_t plain, uint32_t i) { return reinterpret_cast<float *>(lds + (plain ? PLAIN : PACKED) + i * TILE); }
    static __device__ __forceinline__ float *largest(uint8_t *lds, uint32_t plain, uint32_t i) { return reinterpret_cast<float *>(lds + STATS + (2u * (plain * QT + i)) * 128u); }
    static __device__ __forceinline__ float *total(uint8_t *lds, uint32_t plain, uint32_t i) { return reinterpret_cast<float *>(lds + STATS + (2u * (plain * QT + i) + 1u) * 128u); }
};

// A row's uncompressed tokens against the block's tiles of queries, joined sums into LDS.  Two tiles share the waves where four of them hold all tokens (128 of a window,
// 8 x 4096 x 2048: the call 435 us against 463).
template <int DP, int QT, int DT>
__device__ __forceinline__ void plain_phase(const TqManyArgs &a, uint8_t *lds, float (*lds_m)[32], float (*lds_l)[32], float *lds_wild, uint32_t row, uint32_t b, uint32_t tile0, uint32_t tiles,
                                            uint32_t length, uint32_t tid) {
    constexpr int NC = Shape<DP>::NC;
    using J = JoinArea<DP, QT>;
    const uint32_t lane = tid & 63u, wave = tq_uniform32(tid >> 6);
    const uint32_t first = (a.plain[0].n + 31u) / 32u, all = first + (a.plain[1].n + 31u) / 32u;
    const bool share = QT == 2 && tiles == 2u && all <= FAST_WAVES / 2u;
    const uint32_t count = share ? FAST_WAVES / 2u : FAST_WAVES, side = wave / count, w0 = side * count, rounds = share ? 1u : tiles;
#pragma unroll 1
    for (uint32_t i = 0; i < rounds; ++i) {
        const uint32_t mine = share ? side : i;
        float m = MANY_NONE, l = 0.f;
        tq_f16v acc[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c] = tq_zero16();
        bool wild = false;
#pragma unroll 1
        for (uint32_t w = wave - w0; w < all; w += count) {
            PlainTile<DP, DT> t;
            t.wild = false;
            t.load(a, w < first ? 0u : 1u, 32u * (w < first ? w : w - first), row, b, lane);
            t.attend(a, row, b, tile0 + mine, length, lane, m, l, acc);
            wild |= t.wild;
        }
        __syncthreads();             // (what the area held)
        wild = __any(wild);          // (a lane knows of its own coordinates)
        if (lane == 0u) lds_wild[wave] = wild ? 1.f : 0.f;
        float *const area = reinterpret_cast<float *>(lds);
        if (share) join_waves<DP, FAST_WAVES / 2>(area, lds_m, lds_l, J::sums(lds, 1u, mine), J::largest(lds, 1u, mine), J::total(lds, 1u, mine), w0, 1.f, m, l, acc, tid);
        else join_waves<DP, FAST_WAVES>(area, lds_m, lds_l, J::sums(lds, 1u, mine), J::largest(lds, 1u, mine), J::total(lds, 1u, mine), 0u, 1.f, m, l, acc, tid);
        __syncthreads();
        float any = 0.f;
#pragma unroll
        for (int w = 0; w < FAST_WAVES; ++w) any += lds_wild[w];
        if (any != 0.f) {
            if (!share) add_wild<DP>(a, J::sums(lds, 1u, i), row, b, tile0 + i, length, tid);
            else
                for (uint32_t k = 0; k < 2u; ++k) add_wild<DP>(a, J::sums(lds, 1u, k), row, b, tile0 + k, length, tid);
            __syncthreads();
        }
    }
}

// Results of the block's tiles from the joined sums in LDS, where a row's tokens are in one split: packed sums turned back by Pi_v (two fp16 terms each, as the merge
// does), the uncompressed ones added, divided by the sum of weights.
template <int DP, int QT>
__device__ __forceinline__ void finish_block(const TqManyArgs &a, uint8_t *lds, bool plain, uint32_t row, uint32_t tile0, uint32_t tiles, uint32_t tid) {
    constexpr int TILES = Shape<DP>::TILES, STEPS = DP / 16, CH = STEPS < 8 ? STEPS : 8;
    using J = JoinArea<DP, QT>;
    const uint32_t lane = tid & 63u, wave = tq_uniform32(tid >> 6), n = lane & 31u, h = lane >> 5, i = wave / TILES, w = wave % TILES;
    if (i >= tiles) return;
    const float *o = J::sums(lds, 0u, i) + n * (DP + 4u), *p = J::sums(lds, 1u, i) + n * (DP + 4u);
    const float m0 = J::largest(lds, 0u, i)[n], m1 = plain ? J::largest(lds, 1u, i)[n] : MANY_NONE, m = fmaxf(m0, m1);
    const float f0 = m0 == MANY_NONE ? 0.f : __builtin_amdgcn_exp2f(m0 - m), f1 = m1 == MANY_NONE ? 0.f : __builtin_amdgcn_exp2f(m1 - m);
    const float l = J::total(lds, 0u, i)[n] * f0 + (plain ? J::total(lds, 1u, i)[n] * f1 : 0.f), inv = l == 0.f ? 0.f : 1.0f / l;
    const uint32_t q = (tile0 + i) * 32u + n;
    if (a.stat && w == 0u && h == 0u) put_stat(a.stat + ((size_t)row * a.tiles + tile0 + i) * MANY_STATS, n, q < a.M && inv != 0.f, m, l, inv);
    const uint8_t *pi = a.table_v + TQ_OFF_AT_F16(DP) + ((size_t)w * STEPS * 64u + lane) * 16u;
    float largest = 0.f;
#pragma unroll 8
    for (uint32_t d = 0; d < DP / 2u; d += 4u) {
        const tq_f4 v = *reinterpret_cast<const tq_f4 *>(o + h * (DP / 2u) + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) largest = fmaxf(largest, fabsf(v[e]) < __builtin_inff() ? fabsf(v[e]) : 0.f);
    }
    largest = halves_max(largest);
    const int up = largest > 0.f ? max(-100, min(100, Q_TOP - ((int)(__float_as_uint(largest) >> 23) - 127))) : 0;
    const float f = __uint_as_float((uint32_t)(127 + up) << 23);
    tq_f16v acc = tq_zero16();
#pragma unroll 1
    for (int s0 = 0; s0 < STEPS; s0 += CH) {
        tq_u4 ph[CH], pl[CH];
#pragma unroll
        for (int s = 0; s < CH; ++s) { ph[s] = tq_gload16(pi + (size_t)(s0 + s) * 1024u); pl[s] = tq_gload16(pi + TQ_OPERAND_BYTES_FOR(DP) + (size_t)(s0 + s) * 1024u); }
#pragma unroll
        for (int s = 0; s < CH; ++s) {
            const uint32_t j = DP == TQ_HEAD_DIM ? 64u * h + 8u * (s0 + s) : 16u * (s0 + s) + 8u * h;       // (128 wide the table's operands have an order of their own, see tq_table.h)
            tq_f4 x = *reinterpret_cast<const tq_f4 *>(o + j), y = *reinterpret_cast<const tq_f4 *>(o + j + 4u);
            if (!Shape<DP>::EVEN && j >= a.D) x = y = tq_f4{0.f, 0.f, 0.f, 0.f};        // (D a multiple of 8; what lies past it may be anything)
            tq_u4 oh, ol;
            fp16_split8(x, y, f, oh, ol);
            acc = mfma_f16(ph[s], oh, acc);
            acc = mfma_f16(ph[s], ol, acc);
            acc = mfma_f16(pl[s], oh, acc);
        }
    }
    if (q >= a.M) return;
    const float back = __uint_as_float((uint32_t)(127 - up) << 23) * f0;
    const uint32_t d0 = DP == TQ_HEAD_DIM ? 64u * h + 16u * w : 32u * w + 16u * h;
    float out[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) out[r] = inv == 0.f ? 0.f : (acc[r] * back + (plain ? p[d0 + r] * f1 : 0.f)) * inv;
    store_result(a, row, q, d0, out);
}

// Block = (row, QT tiles of 32 queries, split): its waves take runs of 32 tokens in turn, each by itself, and their sums meet in LDS at the end.
//   * scores transposed: A = keys, decoded from the lane's own bytes by table, B = queries; a lane then has 16 tokens of one query;
//   * softmax in base 2 against a reference per query that moves only when a logit exceeds it by 2^FAST_SLACK: no exchange between lanes;
//   * weights times value norms are, as they lie, the B operand of the value product (its contraction runs over the tokens in the order in which a lane
//     has them); A = values, every lane decoding its coordinates' bytes of eight tokens.
// KT = 1: queries and levels as one fp16 value each, for bfloat16: the 2^-12 roundings move logits of some ten by 1e-3, where a bfloat16 result is rounded by up to 4e-3.
// KT = 2: two terms each (three products, 22 bits), for float16, float32 and wherever sums of weights are kept; VT = 2: of weights and value levels as well, for float32.
// Weights and value levels are otherwise one fp16 value each (the reference's own float32 levels are rounded to fp16 by the codec's decompress as well); with KT = 1 a query's
// sum of weights is made of the rounded weights themselves, so that their rounding cancels in part.  KT = 2 for bfloat16 too would take 100 us instead of 76 (16 x 8192 x 64), 643 instead of
// 419 (8 x 4096 x 2048).
// What bounds it: vector instructions and products, which hardly overlap (16 x 8192 x 64: vector 52 % of the cycles, 280 a run of 32 tokens; matrix 24 %, LDS 40 %; 8 x 4096 x 2048: 51, 22
// and 28 %). Waves are not what is missing: twelve with 168 registers took 84 us instead of 78 for the former, sixteen with 128 spill a hundred and took 178. 128 wide, 4 and 2 bits, 8 kv heads, us of this launch: 1 x 2048 tokens x 32 query vectors 12 (start 5, run 2, join 3);
// 1 x 32768 x 256 65 (530 TFLOP/s); 16 x 8192 x 64 79 (440 TFLOP/s, 1.5 TB/s); 32 x 8192 x 4 for sums 87 (2.4 TB/s); with 4 and 4 bits 8 x 4096 x 2048 350 to 480, by card and its clock
// (370 to 500 TFLOP/s), a third of it outside the loop (start, join, uncompressed tokens, way back).
// Query operands stay in registers where they fit beside the sums (QREG): 132 to 134 us against 134 to 138 for the call with 32 x 8192 x 4, with two tiles of 128 wide queries they would spill.
template <int DP, int IPBK, int IPBV, int QT, int KT, int VT>
__global__ __launch_bounds__(FAST_THREADS, FAST_WAVES / 4) void tq_many_fast_kernel(TqManyArgs a) {
    using S = Shape<DP>;
    using Keys = KeyRun<DP, IPBK>;
    constexpr int STEPS = S::STEPS, NC = S::NC, GBV_MAX = DP / IPBV;
    using Values = ValueBytes<IPBV, NC>;
    constexpr int QW = KT * QT * STEPS * 4;                                        // registers of the queries' operands
    constexpr bool QREG = QW + QT * NC * 16 <= 136;
    // a key's norm times the queries' scale from which on logits can pass 2^20: products are at most 2^14 sqrt(D) times the length of the levels, at most 4
    constexpr float LARGE = (float)(1 << 20) / ((float)(1 << 16) * (DP <= 64 ? 8.f : 16.f) * (KT == 2 ? (float)(1 << LEVEL_SHIFT) : 1.f));
    constexpr int LUT_BYTES = 65536, Q_BYTES = KT * QT * STEPS * 1024;
    constexpr bool STAGE = !S::EVEN || GBV_MAX <= 128;
    constexpr int VPIECES = S::EVEN ? (GBV_MAX >= 32 ? GBV_MAX / 32 : 1) : (GBV_MAX + 31) / 32;        // 16 bytes of a run's values, that a lane stages
    constexpr uint32_t WAVE_BYTES = Keys::BYTES + (STAGE ? 32u * GBV_MAX : 0u);
    using J = JoinArea<DP, QT>;
    constexpr uint32_t LOOP_BYTES = LUT_BYTES + Q_BYTES + FAST_WAVES * WAVE_BYTES + (S::EVEN ? 0u : 64u);       // (uneven: lanes past the last coordinate read on)
    constexpr uint32_t AREA = LOOP_BYTES > J::BYTES ? LOOP_BYTES : J::BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[AREA];
    __shared__ __attribute__((aligned(16))) float lds_kn[FAST_WAVES][32];
    __shared__ __attribute__((aligned(16))) std::conditional_t<VT == 2, float, uint16_t> lds_vn[FAST_WAVES][32];
    __shared__ float lds_m[FAST_WAVES][32], lds_l[FAST_WAVES][32], lds_own[QT][32];

    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tq_uniform32(tid >> 6), n = lane & 31u, h = lane >> 5;
    const uint32_t groups = (a.tiles + QT - 1u) / QT;
    const bool packed = blockIdx.x >= a.plain_blocks;
    const uint32_t block = packed ? blockIdx.x - a.plain_blocks : blockIdx.x;
    const uint32_t split = packed ? block % a.splits : 0u, at = packed ? block / a.splits : block, row = at / groups, tile0 = (at - row * groups) * QT, b = row / a.heads;
    const size_t first_tile = (size_t)row * a.tiles + tile0;
    const uint32_t tiles = min((uint32_t)QT, a.tiles - tile0);
    const uint32_t length = many_length(a, b);

    // A row's uncompressed tokens: by the block that has its packed ones, where they are in one split, otherwise by blocks of their own, the first of
    // the launch, so that they are done while the others are at the packed ones.
    if (packed) {
    const uint32_t GBK = S::EVEN ? DP / IPBK : (a.D + IPBK - 1u) / IPBK, GBV = S::EVEN ? DP / IPBV : (a.D + IPBV - 1u) / IPBV;
    const uint32_t seen = min(a.tokens, length);
    const uint32_t chunk = a.lengths ? ((seen + a.splits - 1u) / a.splits + 31u) / 32u * 32u : a.chunk;       // (a short sequence keeps all its blocks busy)
    const uint32_t begin = min(seen, split * chunk), end = min(seen, begin + chunk);
    const size_t slot0 = (size_t)row * a.packed_row_stride;
    const uint8_t *mask = a.mask ? a.mask + (long long)b * a.mask_stride : nullptr;
    const uint32_t v_lane = 4u * h * GBV + (IPBV == 4 && NC == 2 ? n / 2u : n * Values::VB);

    // Loads of a run are issued while the one before it is worked on.  The last run of a row begins 32 tokens before the end: what the one before it
    // had already is hidden, and nothing past the row's tokens is read.
    // Value bytes go through LDS on their way (a lane needs single bytes of sixteen tokens), but at 256 with a byte a code, where they are
    // read from memory as they are needed.
    Keys keys;
    tq_u4 vpiece[VPIECES];
    Values vraw[16];
    uint16_t kn_raw = 0, vn_raw = 0;
    uint8_t *kstage = lds + LUT_BYTES + Q_BYTES + wave * WAVE_BYTES, *vstage = kstage + Keys::BYTES;
    auto issue_keys = [&](uint32_t t) __attribute__((always_inline)) {
        keys.issue(a.k_idx + (slot0 + t) * GBK, GBK, lane);
        kn_raw = tq_gload2(a.k_norms + slot0 + t + n);
        vn_raw = tq_gload2(a.v_norms + slot0 + t + n);
    };
    auto issue_values = [&](uint32_t t) __attribute__((always_inline)) {
        const uint8_t *p = a.v_idx + (slot0 + t) * GBV;
        if constexpr (!STAGE) {
#pragma unroll
            for (int j = 0; j < 16; ++j) vraw[j].load(p + v_lane + (8 * (j / 4) + j % 4) * GBV);
        } else if constexpr (!S::EVEN) {
#pragma unroll
            for (int i = 0; i < VPIECES; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) vpiece[i][k] = tq_gload4(p + 4u * min(256u * i + 64u * k + lane, 8u * GBV - 1u));
        } else if constexpr (GBV_MAX == 16) {
            const tq_u2 v = tq_gload8(p + lane * 8u);
            vpiece[0][0] = v[0]; vpiece[0][1] = v[1];
        } else {
#pragma unroll
            for (int i = 0; i < VPIECES; ++i) vpiece[i] = tq_gload16(p + i * 1024 + lane * 16u);
        }
    };
    auto stage_values = [&]() __attribute__((always_inline)) {
        if constexpr (!S::EVEN) {
#pragma unroll
            for (int i = 0; i < VPIECES; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (256u * i + 64u * k + lane < 8u * GBV_MAX) *reinterpret_cast<uint32_t *>(vstage + 4u * (256u * i + 64u * k + lane)) = vpiece[i][k];
        } else if constexpr (GBV_MAX == 16) *reinterpret_cast<tq_u2 *>(vstage + lane * 8u) = tq_u2{vpiece[0][0], vpiece[0][1]};
        else {
#pragma unroll
            for (int i = 0; i < VPIECES; ++i) *reinterpret_cast<tq_u4 *>(vstage + i * 1024 + lane * 16u) = vpiece[i];
        }
    };
    const uint32_t last = a.tokens - 32u;    // (launched for 32 tokens at least)
    uint32_t t_next = begin + 32u * wave;
    // ---- start: tables, rotation and the first run are asked for before anything is waited for
    uint8_t *ops = lds + LUT_BYTES;
    std::conditional_t<KT == 1, Lut<IPBK>, Lut2<IPBK>> table_k;
    std::conditional_t<VT == 1, Lut<IPBV>, Lut2<IPBV>> table_v;
    if constexpr (KT == 1) table_k.load(a.table_k + TQ_OFF_LUT(DP), tid);
    else table_k.load(a.table_k, a.bits_k, DP, tid);
    if constexpr (VT == 1) table_v.load(a.table_v + TQ_OFF_LUT(DP), tid);
    else table_v.load(a.table_v, a.bits_v, DP, tid);
    float q_scale;
    bool apart;
    auto start = [&](auto dt_tag) __attribute__((always_inline)) {
        Rotate<DP, QT, KT, decltype(dt_tag)::value> r;
        r.load(a, row, tile0, wave, lane);
        if (t_next < end) {
            issue_keys(min(t_next, last));
            issue_values(min(t_next, last));
        }
        __builtin_amdgcn_sched_barrier(0);
        table_k.store(lds, tid);
        table_v.store(lds + 128, tid);
        q_scale = r.finish(a, ops, lds_kn, lds_own, apart, wave, lane);
    };
    if constexpr (VT == 2) start(std::integral_constant<int, TQ_F32>{});
    else if (a.dtype == TQ_BF16) start(std::integral_constant<int, TQ_BF16>{});
    else if constexpr (KT == 2) start(std::integral_constant<int, TQ_F16>{});
    else __builtin_unreachable();            // (KT = 1 is launched for bfloat16 alone)
    __syncthreads();
    uint32_t ops_lane = LUT_BYTES + lane * 16u;
    asm volatile("" : "+v"(ops_lane));        // (one base for all operands: the offsets then fit the instructions)
    tq_u4 q[QREG ? KT * QT * STEPS : 1];
    if constexpr (QREG) {
#pragma unroll
        for (int s = 0; s < KT * QT * STEPS; ++s) q[s] = *reinterpret_cast<const tq_u4 *>(lds + ops_lane + s * 1024);
    }
    auto query = [&](int i, int term, int s) __attribute__((always_inline)) -> tq_u4 {
        if constexpr (QREG) return q[(i * KT + term) * STEPS + s];
        else return *reinterpret_cast<const tq_u4 *>(lds + ops_lane + ((i * KT + term) * STEPS + s) * 1024);
    };
    if (a.weights && split == 0u) {          // (KT = 2: whole operands) for the launch that adds up what keys receive
        for (uint32_t i = tid; i < Q_BYTES / 16u; i += FAST_THREADS) tq_gstore16(a.q_op + first_tile * q_operand_bytes(DP) + i * 16u, *reinterpret_cast<const tq_u4 *>(ops + i * 16u));
        if (tid < 32u) a.q_scale[first_tile * 32u + tid] = apart ? lds_own[0][tid] * q_scale : q_scale;
    }
    const uint32_t slot_k = KT == 1 ? RepLut<IPBK>::lane_offset(lane) : Lut2<IPBK>::lane_offset(lane);
    const uint32_t slot_v = 128u + (VT == 2 ? Lut2<IPBV>::lane_offset(lane) : IPBV == 4 && NC == 2 ? (lane & 30u) / 2u * 8u + 4u * (lane & 1u) : RepLut<IPBV>::lane_offset(lane));

    float m_ref[QT], l[QT];
    tq_f16v acc[QT][NC];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        m_ref[i] = MANY_NONE;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[i][c] = tq_zero16();
    }
    int v_top = -100;                        // 2^v_top: unit of the value norms, their largest binary exponent so far
    while (t_next < end) {
        const uint32_t t_run = t_next, t0 = min(t_run, last), count = min(32u, end - t_run);
        t_next += 32u * FAST_WAVES;
        // (the two waves of a SIMD go first in turn: left to itself the older one runs ahead, and the other then ends alone)
        if (((t_run / (32u * FAST_WAVES)) ^ (wave >> 2)) & 1u) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        const uint32_t t_after = min(t_next < end ? t_next : t_run, last);
        uint32_t hidden = ~((count == 32u ? 0xffffffffu : (1u << count) - 1u) << (t_run - t0));
        if (mask) hidden |= ~(uint32_t)__ballot(mask[t0 + n] != 0);
        // ---- norms: keys' times the queries' scale, values' in the unit of the largest so far
        float norm = (float)__builtin_bit_cast(_Float16, h ? vn_raw : kn_raw);
        if (hidden) norm = (hidden >> n) & 1u ? 0.f : norm;
        const int top = (int)((__float_as_uint(norm) >> 23) & 255u) - 127;
        if (__any(h && top > v_top)) {
            int new_top = h ? top : -100;
#pragma unroll
            for (int i = 32; i; i >>= 1) new_top = max(new_top, __shfl_xor(new_top, i));
            new_top = min(max(new_top, v_top), 16);
            const float f = __uint_as_float((uint32_t)(127 + v_top - new_top) << 23);
            v_top = new_top;
#pragma unroll
            for (int i = 0; i < QT; ++i)
#pragma unroll
                for (int c = 0; c < NC; ++c) acc[i][c] *= f;
        }
        norm *= h ? __uint_as_float((uint32_t)(127 - v_top) << 23) : q_scale;
        // Where logits can be so large that what an unrounded product differs from the (rounded) reference by is no small part of one, up to more than an exponent can be, products
        // are rounded first.
        const bool large = __any(!h && norm >= LARGE);
        if (!h) lds_kn[wave][n] = norm;
        else if constexpr (VT == 2) lds_vn[wave][n] = norm;
        else lds_vn[wave][n] = __builtin_bit_cast(uint16_t, (_Float16)norm);
        keys.stage(kstage, lane);
        if constexpr (STAGE) {
            stage_values();
            issue_values(t_after);
        }
        wave_sync();
        // ---- scores
        keys.take(kstage, GBK, lane);
        tq_f16v s[QT];
#pragma unroll
        for (int i = 0; i < QT; ++i) s[i] = tq_zero16();
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            if constexpr (KT == 1) {
                const tq_u4 k = decode_keys<IPBK, Keys::KW>(keys.raw, st, lds, slot_k);
#pragma unroll
                for (int i = 0; i < QT; ++i) s[i] = mfma_f16(k, query(i, 0, st), s[i]);
            } else {
                tq_u4 hi, lo;
                decode_keys2<IPBK, Keys::KW>(keys.raw, st, lds, slot_k, hi, lo);
#pragma unroll
                for (int i = 0; i < QT; ++i) {
                    const tq_u4 qh = query(i, 0, st), ql = query(i, KT - 1, st);
                    s[i] = mfma_f16(hi, qh, s[i]);
                    s[i] = mfma_f16(hi, ql, s[i]);
                    s[i] = mfma_f16(lo, qh, s[i]);
                }
            }
        }
        issue_keys(t_after);
        // ---- weights
        tq_u4 p[QT][2], p2[VT == 2 ? QT : 1][2];
        float kn[16];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const tq_f4 v = *reinterpret_cast<const tq_f4 *>(&lds_kn[wave][8 * k + 4 * h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) kn[4 * k + j] = v[j];
        }
        uint32_t vn[VT == 2 ? 16 : 8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (VT == 2) {
                const tq_u4 v = *reinterpret_cast<const tq_u4 *>(&lds_vn[wave][8 * k + 4 * h]);
#pragma unroll
                for (int j = 0; j < 4; ++j) vn[4 * k + j] = v[j];
            } else {
                const tq_u2 v = *reinterpret_cast<const tq_u2 *>(&lds_vn[wave][8 * k + 4 * h]);
                vn[2 * k] = v[0]; vn[2 * k + 1] = v[1];
            }
        }
        if (large || apart) {
            float own[QT];
#pragma unroll
            for (int i = 0; i < QT; ++i) own[i] = apart ? lds_own[i][n] : 1.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
#pragma unroll
                for (int i = 0; i < QT; ++i) {
                    float logit = s[i][r] * own[i] * kn[r];
                    asm volatile("" : "+v"(logit));
                    s[i][r] = logit;
                }
                kn[r] = 1.f;
            }
        }
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            float x[16];
            auto logits = [&]() __attribute__((always_inline)) {
                const float bias = (float)FAST_P - m_ref[i];
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = fmaf(s[i][r], kn[r], bias);
                if (hidden) {        // (opaque: in its branch, not ahead of it for every run)
                    uint32_t bits = hidden >> (4u * h);
                    asm volatile("" : "+v"(bits));
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] = (bits >> acc_row(r, 0u)) & 1u ? -__builtin_inff() : x[r];
                }
            };
            logits();
            float most = x[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) most = fmaxf(most, x[r]);
            if (__any(most > (float)(FAST_P + FAST_SLACK))) {
                float now = -__builtin_inff();
                uint32_t bits = hidden >> (4u * h);
                asm volatile("" : "+v"(bits));
#pragma unroll
                for (int r = 0; r < 16; ++r) now = (bits >> acc_row(r, 0u)) & 1u ? now : fmaxf(now, s[i][r] * kn[r]);
                now = fmaxf(halves_max(now), m_ref[i]);
                const float shrink = __builtin_amdgcn_exp2f(m_ref[i] - now);
                m_ref[i] = now;
                l[i] *= shrink;
#pragma unroll
                for (int c = 0; c < NC; ++c) acc[i][c] *= shrink;
                logits();
            }
            if (KT == 2) {
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) { x[r] = __builtin_amdgcn_exp2f(x[r]); sum += x[r]; }
                l[i] += sum;
            }
            if constexpr (VT == 2) {
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    uint32_t t[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[j] = fp16_terms(x[8 * st + j] * __uint_as_float(vn[8 * st + j]));
                    fp16_operands(t, p[i][st], p2[i][st]);
                }
            } else {
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    tq_half2 w;
                    if constexpr (KT == 2) w = tq_half2{(_Float16)x[2 * d], (_Float16)x[2 * d + 1]};
                    else {
                        w = tq_half2{(_Float16)__builtin_amdgcn_exp2f(x[2 * d]), (_Float16)__builtin_amdgcn_exp2f(x[2 * d + 1])};
                        l[i] = __builtin_amdgcn_fdot2(w, tq_half2{(_Float16)1.f, (_Float16)1.f}, l[i], false);
                    }
                    p[i][d / 4][d % 4] = __builtin_bit_cast(uint32_t, w * __builtin_bit_cast(tq_half2, vn[d]));
                }
            }
        }
        // ---- values
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            uint32_t w[8][NC / 2], w2[VT == 2 ? 8 : 1][NC / 2];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                Values v;
                if constexpr (STAGE) v.fetch(vstage + v_lane + (16 * st + 8 * (j / 4) + j % 4) * GBV);
                else v = vraw[8 * st + j];
                if constexpr (VT == 2) decode_values2<IPBV, NC>(v, lds, slot_v, n & 1u, w[j], w2[j]);
                else v.decode(lds, slot_v, w[j]);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                auto operand = [&](const auto &x) __attribute__((always_inline)) {
                    tq_u4 v;
#pragma unroll
                    for (int d = 0; d < 4; ++d) v[d] = __builtin_amdgcn_perm(x[2 * d + 1][c / 2], x[2 * d][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
                    return v;
                };
                const tq_u4 v = operand(w);
#pragma unroll
                for (int i = 0; i < QT; ++i) acc[i][c] = mfma_f16(v, p[i][st], acc[i][c]);
                if constexpr (VT == 2) {
                    const tq_u4 v2 = operand(w2);
#pragma unroll
                    for (int i = 0; i < QT; ++i) {
                        acc[i][c] = mfma_f16(v, p2[i][st], acc[i][c]);
                        acc[i][c] = mfma_f16(v2, p[i][st], acc[i][c]);
                    }
                }
            }
        }
        if constexpr (!STAGE) issue_values(t_after);
        wave_sync();
    }

    __builtin_amdgcn_s_setprio(0);
    // ---- the waves' sums
    const float unit = v_top == -100 ? 0.f : __uint_as_float((uint32_t)(127 + v_top - FAST_P - (VT == 2 ? LEVEL_SHIFT : 0)) << 23);
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        __syncthreads();
        join_waves<DP, FAST_WAVES>(reinterpret_cast<float *>(lds), lds_m, lds_l, J::sums(lds, 0u, i), J::largest(lds, 0u, i), J::total(lds, 0u, i), 0u, unit,
                      m_ref[i], l[i] * (1.0f / (float)(1 << FAST_P)), acc[i], tid);
    }
    __syncthreads();
    }
    const bool whole = a.splits == 1u, plain = (a.plain[0].n | a.plain[1].n) != 0u;
    if (plain && (whole || !packed)) {
        if constexpr (VT == 2) plain_phase<DP, QT, TQ_F32>(a, lds, lds_m, lds_l, lds_kn[0], row, b, tile0, tiles, length, tid);
        else if (a.dtype == TQ_BF16) plain_phase<DP, QT, TQ_BF16>(a, lds, lds_m, lds_l, lds_kn[0], row, b, tile0, tiles, length, tid);
        else if constexpr (KT == 2) plain_phase<DP, QT, TQ_F16>(a, lds, lds_m, lds_l, lds_kn[0], row, b, tile0, tiles, length, tid);
    }
    if (whole) {
        finish_block<DP, QT>(a, lds, plain, row, tile0, tiles, tid);
        return;
    }
    for (uint32_t i = 0; i < tiles; ++i) {
        float *rec = packed ? a.rec + ((first_tile + i) * a.records + split) * record_floats(DP) : a.plain_rec + (first_tile + i) * record_floats(DP);
        put_record<DP>(rec, J::sums(lds, packed ? 0u : 1u, i), J::largest(lds, packed ? 0u : 1u, i), J::total(lds, packed ? 0u : 1u, i), tid);
    }
}

// What the packed tokens receive: weight = 2^(logit - largest) / sum with the statistics of the merge, from the two-term products.  Rows of the product are queries
// here, columns tokens, so that a token's sum is made in its lane; rows in which a tile has no query are left out eight at a time.  Block = part of
// a row's tokens, a wave takes 32 at a time and all tiles of queries in order (the first one's operands lie in LDS, a decode step has no more).
// The first blocks are for the window's tokens: a wave 32 of them.
// 128 wide, 4 bits, 8 kv heads x 4 query vectors (before those had the kernel below): 32768 tokens 11 us, 32 sequences of 8192 59 us (155 MB, 2.6 TB/s): the two-term entries' reads (LDS busy 39 % of the
// time) and the products hardly overlap.  Loads two runs ahead instead of one changed nothing, none ahead took 14 instead of 11 us.
template <int DP, int DT>
__device__ __forceinline__ void window_weights(const TqManyArgs &a, uint32_t item, uint32_t lane) {
    if constexpr (DT == TQ_F32) plain_weights<TQ_F32>(a, item, DP / 16u, lane);
    else {
        using T = PlainTile<DP, DT>;
        constexpr int STEPS = DP / 16, CH = DP <= 128 ? STEPS : 8;
        const TqManyPlain &seg = a.plain[0];
        const uint32_t groups = (seg.n + 31u) / 32u, row = item / groups, t0 = 32u * (item - row * groups), b = row / a.heads, kv = row - b * a.heads;
        const uint32_t n = lane & 31u, h = lane >> 5, length = many_length(a, b), t = t0 + n, tc = min(t, seg.n - 1u);
        const uint8_t *k = seg.k + ((long long)b * seg.k_batch + (long long)kv * seg.k_head + (long long)tc * seg.k_token) * 2;
        const bool seen = t < seg.n && plain_seen(a, 0u, b, 0u, tc, length);
        float w = 0.f;
#pragma unroll 1
        for (uint32_t tile = 0; tile < a.tiles; ++tile) {             // rows of the product: queries, columns: tokens
            const uint8_t *q = many_query(a, row, min(tile * 32u + n, a.M - 1u), 2u);
            const TQ_GLOBAL float *stat = (const TQ_GLOBAL float *)a.stat + ((size_t)row * a.tiles + tile) * MANY_STATS + 4u * h;
            tq_f16v s = tq_zero16();
#pragma unroll 1
            for (int s0 = 0; s0 < STEPS; s0 += CH) {
                tq_u4 x[CH], y[CH];
#pragma unroll
                for (int st = 0; st < CH; ++st) { x[st] = T::half_step(k, s0 + st, h, a.D, a.aligned); y[st] = T::half_step(q, s0 + st, h, a.D, a.aligned); }
#pragma unroll
                for (int st = 0; st < CH; ++st) s = DT == TQ_BF16 ? mfma_bf16(y[st], x[st], s) : mfma_f16(y[st], x[st], s);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const tq_f4 m = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(stat + 8 * g), inv = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(stat + 32 + 8 * g), most = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(stat + 64 + 8 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (inv[r] != 0.f) w = fmaf(__builtin_amdgcn_exp2f(weight_exponent(s[4 * g + r], a.scale * LOG2E, m[r], most[r])), inv[r], w);
            }
        }
        w = halves_add(w);
        if (h == 0u && seen) a.weights[(long long)row * a.w_stride + a.tokens + t] += w;
    }
}

template <int DP, int IPBK>
__global__ __launch_bounds__(FAST_THREADS, FAST_WAVES / 4) void tq_many_weights_kernel(TqManyArgs a, uint32_t blocks) {
    const uint32_t items = a.rows * ((a.plain[0].n + 31u) / 32u), first = (items + FAST_WAVES - 1u) / FAST_WAVES;
    if (blockIdx.x < first) {
        const uint32_t item = blockIdx.x * FAST_WAVES + tq_uniform32(threadIdx.x >> 6);
        if (item >= items) return;
        if (a.dtype == TQ_BF16) window_weights<DP, TQ_BF16>(a, item, threadIdx.x & 63u);
        else if (a.dtype == TQ_F16) window_weights<DP, TQ_F16>(a, item, threadIdx.x & 63u);
        else window_weights<DP, TQ_F32>(a, item, threadIdx.x & 63u);
        return;
    }
    const uint32_t block = blockIdx.x - first;
    using Keys = KeyRun<DP, IPBK>;
    constexpr int STEPS = DP / 16, KW = Keys::KW, LUT_BYTES = 65536;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[LUT_BYTES + 2 * STEPS * 1024 + FAST_WAVES * Keys::BYTES];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tq_uniform32(tid >> 6), n = lane & 31u, h = lane >> 5;
    const uint32_t row = block / blocks, b = row / a.heads;
    const size_t first_tile = (size_t)row * a.tiles;
    const uint32_t seen = min(a.tokens, many_length(a, b));
    {
        Lut2<IPBK> table;
        table.load(a.table_k, a.bits_k, DP, tid);
        table.store(lds, tid);              // (alone, it takes the whole row)
        table.store(lds + 128, tid);
    }
    tq_copy_to_lds(lds + LUT_BYTES, a.q_op + first_tile * q_operand_bytes(DP), 2 * STEPS * 1024, tid, FAST_THREADS);
    const uint32_t slot = (lane & (64u / IPBK - 1u)) * 4u * IPBK;
    __syncthreads();
    const size_t slot0 = (size_t)row * a.packed_row_stride;
    const uint32_t GBK = Shape<DP>::EVEN ? DP / IPBK : (a.D + IPBK - 1u) / IPBK;
    uint8_t *kstage = lds + LUT_BYTES + 2 * STEPS * 1024 + wave * Keys::BYTES;
    const uint32_t last = a.tokens - 32u, step = 32u * FAST_WAVES * blocks;
    // (loads of a run are issued while the one before it is worked on)
    Keys keys;
    uint16_t norm_raw = 0;
    float before_raw = 0.f;
    float *const sums = a.weights + (long long)row * a.w_stride;
    auto issue = [&](uint32_t t) __attribute__((always_inline)) {
        keys.issue(a.k_idx + (slot0 + t) * GBK, GBK, lane);
        norm_raw = tq_gload2(a.k_norms + slot0 + t + n);
        before_raw = *((const TQ_GLOBAL float *)sums + t + n);
    };
    uint32_t t_next = 32u * ((block - row * blocks) * FAST_WAVES + wave);
    if (t_next < seen) issue(min(t_next, last));
    uint32_t first_of_two = wave >> 2;
    while (t_next < seen) {
        const uint32_t t_run = t_next, t0 = min(t_run, last), t = t0 + n;
        t_next += step;
        first_of_two ^= 1u;                 // (as in the kernel above)
        if (first_of_two) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        const float norm = (float)__builtin_bit_cast(_Float16, norm_raw), before = before_raw;
        const bool counts = t >= t_run && t < seen && (!a.mask || a.mask[(long long)b * a.mask_stride + t]);
        float w = 0.f;
        keys.stage(kstage, lane);
        wave_sync();
        keys.take(kstage, GBK, lane);
        uint32_t kraw[KW];
#pragma unroll
        for (int i = 0; i < KW; ++i) kraw[i] = keys.raw[i];
        if (t_next < seen) issue(min(t_next, last));
        auto add = [&](const tq_f16v &s, uint32_t tile, uint32_t queries) __attribute__((always_inline)) {
            const TQ_GLOBAL float *stat = (const TQ_GLOBAL float *)a.stat + (first_tile + tile) * MANY_STATS + 4u * h, *scale = (const TQ_GLOBAL float *)a.q_scale + (first_tile + tile) * 32u + 4u * h;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (8u * g >= queries) break;
                const tq_f4 m = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(stat + 8 * g), inv = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(stat + 32 + 8 * g), most = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(stat + 64 + 8 * g);
                const tq_f4 qs = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(scale + 8 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r) w = fmaf(__builtin_amdgcn_exp2f(weight_exponent(s[4 * g + r], norm * qs[r], m[r], most[r])), inv[r], w);
            }
        };
        {
            tq_f16v s = tq_zero16();
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                tq_u4 hi, lo;
                decode_keys2<IPBK, KW>(kraw, st, lds, slot, hi, lo);
                const tq_u4 qh = *reinterpret_cast<const tq_u4 *>(lds + LUT_BYTES + st * 1024 + lane * 16u), ql = *reinterpret_cast<const tq_u4 *>(lds + LUT_BYTES + (STEPS + st) * 1024 + lane * 16u);
                s = mfma_f16(qh, hi, s);
                s = mfma_f16(ql, hi, s);
                s = mfma_f16(qh, lo, s);
            }
            add(s, 0u, a.M);
        }
#pragma unroll 1
        for (uint32_t tile = 1; tile < a.tiles; ++tile) {
            const uint8_t *ops = a.q_op + (first_tile + tile) * q_operand_bytes(DP) + lane * 16u;
            tq_f16v s = tq_zero16();
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                tq_u4 hi, lo;
                decode_keys2<IPBK, KW>(kraw, st, lds, slot, hi, lo);
                const tq_u4 qh = tq_gload16(ops + st * 1024), ql = tq_gload16(ops + (STEPS + st) * 1024);
                s = mfma_f16(qh, hi, s);
                s = mfma_f16(ql, hi, s);
                s = mfma_f16(qh, lo, s);
            }
            add(s, tile, a.M - 32u * tile);
        }
        w = halves_add(w);
        if (h == 0u && counts) *((TQ_GLOBAL float *)sums + t) = before + w;
        wave_sync();
    }
}

// The same for at most 16 query vectors a row (a decode step has no more): products of 16 x 16 with twice the contraction, so that half as many of their columns are empty, and
// the queries' operands stay in registers.  Lane (n = lane % 16, kg = lane / 16) has coordinates kg * DP / 4 ... of query n and of tokens n and 16 + n of a run; the sums of a token
// over the queries 4 kg ... + 3 lie in its four lanes.  Two blocks a compute unit, 256 wide (registers) one.
// 128 wide, 4 bits, 8 kv heads x 4 query vectors: 32768 tokens 9.7 us (11.5 by the kernel above), 32 sequences of 8192 41 us (59), 155 MB at 3.8 TB/s.
template <int DP, int IPBK>
__global__ __launch_bounds__(FAST_THREADS, FAST_WAVES / (DP == 256 ? 4 : 2)) void tq_many_few_weights_kernel(TqManyArgs a, uint32_t blocks) {
    const uint32_t items = a.rows * ((a.plain[0].n + 31u) / 32u), first = (items + FAST_WAVES - 1u) / FAST_WAVES;
    if (blockIdx.x < first) {
        const uint32_t item = blockIdx.x * FAST_WAVES + tq_uniform32(threadIdx.x >> 6);
        if (item >= items) return;
        if (a.dtype == TQ_BF16) window_weights<DP, TQ_BF16>(a, item, threadIdx.x & 63u);
        else window_weights<DP, TQ_F16>(a, item, threadIdx.x & 63u);
        return;
    }
    constexpr int STEPS = DP / 32, KW = DP / 16 / IPBK;                // steps of eight coordinates of a lane, words of its packed bytes a token
    constexpr uint32_t GB = DP / IPBK;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[65536];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tq_uniform32(tid >> 6), n = lane & 15u, kg = lane >> 4;
    const uint32_t block = blockIdx.x - first, row = block / blocks, b = row / a.heads;
    const uint32_t seen = min(a.tokens, many_length(a, b));
    {
        Lut2<IPBK> table;
        table.load(a.table_k, a.bits_k, DP, tid);
        table.store(lds, tid);
        table.store(lds + 128, tid);
    }
    tq_u4 q[2][STEPS];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
            q[t][s] = tq_gload16(a.q_op + (size_t)row * q_operand_bytes(DP) + ((t * (DP / 16) + (kg & 1u) * STEPS + s) * 64u + (kg >> 1) * 32u + n) * 16u);
    const TQ_GLOBAL float *stat = (const TQ_GLOBAL float *)a.stat + (size_t)row * MANY_STATS + 4u * kg;
    tq_f4 m = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(stat), inv = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(stat + 32);
    const tq_f4 most = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(stat + 64);
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (4u * kg + r >= a.M) { m[r] = -MANY_NONE; inv[r] = 0.f; }
    const tq_f4 q_scale = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>((const TQ_GLOBAL float *)a.q_scale + (size_t)row * 32u + 4u * kg);
    const uint32_t slot = (lane & (64u / IPBK - 1u)) * 4u * IPBK;
    __syncthreads();
    const size_t slot0 = (size_t)row * a.packed_row_stride;
    const uint32_t last = a.tokens - 32u, step = 32u * FAST_WAVES * blocks;
    float *const sums = a.weights + (long long)row * a.w_stride;
    uint32_t raw[2][KW];
    uint16_t norm_raw[2] = {0, 0};
    float before_raw = 0.f;
    auto issue = [&](uint32_t t) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint8_t *p = a.k_idx + (slot0 + t + 16u * i + n) * GB + kg * (GB / 4u);
            if constexpr (KW == 1) raw[i][0] = tq_gload4(p);
            else if constexpr (KW == 2) { const tq_u2 v = tq_gload8(p); raw[i][0] = v[0]; raw[i][KW > 1 ? 1 : 0] = v[1]; }
            else {
#pragma unroll
                for (int k = 0; k < KW / 4; ++k) {
                    const tq_u4 v = tq_gload16(p + 16 * k);
#pragma unroll
                    for (int j = 0; j < 4; ++j) raw[i][4 * k + j] = v[j];
                }
            }
            norm_raw[i] = tq_gload2(a.k_norms + slot0 + t + 16u * i + n);
        }
        before_raw = *((const TQ_GLOBAL float *)sums + t + (lane & 31u));
    };
    uint32_t t_next = 32u * ((block - row * blocks) * FAST_WAVES + wave);
    if (t_next < seen) issue(min(t_next, last));
    while (t_next < seen) {
        const uint32_t t_run = t_next, t0 = min(t_run, last), t = t0 + (lane & 31u);
        t_next += step;
        const bool counts = lane < 32u && t >= t_run && t < seen && (!a.mask || a.mask[(long long)b * a.mask_stride + t]);
        const float before = before_raw, kn[2] = {(float)__builtin_bit_cast(_Float16, norm_raw[0]), (float)__builtin_bit_cast(_Float16, norm_raw[1])};
        uint32_t now[2][KW];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int k = 0; k < KW; ++k) now[i][k] = raw[i][k];
        if (t_next < seen) issue(min(t_next, last));
        float w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            tq_f4v s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                tq_u4 hi, lo;
                decode_keys2<IPBK, KW>(now[i], st, lds, slot, hi, lo);
                s = mfma16_f16(q[0][st], hi, s);
                s = mfma16_f16(q[1][st], hi, s);
                s = mfma16_f16(q[0][st], lo, s);
            }
            w[i] = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) w[i] = fmaf(__builtin_amdgcn_exp2f(weight_exponent(s[r], kn[i] * q_scale[r], m[r], most[r])), inv[r], w[i]);
            w[i] = reduce_rows(w[i], OpAdd());
        }
        if (counts) *((TQ_GLOBAL float *)sums + t) = before + (lane & 16u ? w[1] : w[0]);
    }
}

template <int DP, int IPBK>
int launch_many_weights(dim3 grid, hipStream_t s, const TqManyArgs &a, uint32_t blocks) {
    if constexpr (Shape<DP>::EVEN) {
        if (many_few(a, DP)) {
            hipLaunchKernelGGL((tq_many_few_weights_kernel<DP, IPBK>), grid, dim3(FAST_THREADS), 0, s, a, blocks);
            return 0;
        }
    }
    hipLaunchKernelGGL((tq_many_weights_kernel<DP, IPBK>), grid, dim3(FAST_THREADS), 0, s, a, blocks);
    return 0;
}

// ipb: codes per byte
template <int DP, int IPBK, int IPBV>
int launch_many_fast(dim3 grid, hipStream_t s, const TqManyArgs &a, int qt, int kt, int vt) {
    if (vt == 2) hipLaunchKernelGGL((tq_many_fast_kernel<DP, IPBK, IPBV, 1, 2, 2>), grid, dim3(FAST_THREADS), 0, s, a);
    else if (kt == 2) hipLaunchKernelGGL((tq_many_fast_kernel<DP, IPBK, IPBV, 1, 2, 1>), grid, dim3(FAST_THREADS), 0, s, a);
    else if (DP == 256 || qt == 1) hipLaunchKernelGGL((tq_many_fast_kernel<DP, IPBK, IPBV, 1, 1, 1>), grid, dim3(FAST_THREADS), 0, s, a);
    else if constexpr (DP != 256) hipLaunchKernelGGL((tq_many_fast_kernel<DP, IPBK, IPBV, 2, 1, 1>), grid, dim3(FAST_THREADS), 0, s, a);
    return 0;
}
template <int DP, int IPBK>
int launch_many_fast(int ipbv, dim3 grid, hipStream_t s, const TqManyArgs &a, int qt, int kt, int vt) {
    if (ipbv == 4) return launch_many_fast<DP, IPBK, 4>(grid, s, a, qt, kt, vt);
    if (ipbv == 2) return launch_many_fast<DP, IPBK, 2>(grid, s, a, qt, kt, vt);
    return launch_many_fast<DP, IPBK, 1>(grid, s, a, qt, kt, vt);
}

}  // namespace
