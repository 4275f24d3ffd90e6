// Attention of tiles of queries over packed tokens at head dimensions 64, 128 and 256, codes of one, two or four to a byte (tq_many.hip).
// One source file per head dimension instantiates it.
#pragma once
#include "tq_many.h"
#include "tq_lut.h"

namespace {

constexpr int FAST_WAVES = 8;                // one block per compute unit, two waves per SIMD, which share the tables
constexpr int FAST_THREADS = 64 * FAST_WAVES;
static_assert(FAST_THREADS == LUT_THREADS, "threads that stage the tables");
constexpr int FAST_SLACK = 8;                // a column's reference moves when a logit exceeds it by more than this
constexpr int FAST_P = 14 - FAST_SLACK;      // weights enter the products times 2^FAST_P, at most 2^14; value norms below 2 in their unit
constexpr float FAST_START = -1.0e30f;

// The keys' table with two fp16 terms a level: an entry is the byte's leading terms, then the rests; spread over the banks as Lut does.
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

// Block = (row, QT tiles of 32 queries, split): its waves take runs of 32 tokens in turn, each by itself, and their sums meet in LDS at the end.
//   * scores transposed: A = keys, decoded from the lane's own bytes by table, B = queries; a lane then has 16 tokens of one query;
//   * softmax in base 2 against a reference per query that moves only when a logit exceeds it by 2^FAST_SLACK: no exchange between lanes;
//   * weights times value norms are, as they lie, the B operand of the value product (its contraction runs over the tokens in the order in which a lane
//     has them); A = values, every lane reading its coordinates' bytes of the eight tokens straight from memory.
// KT = 1: queries and levels as one fp16 value each, for bfloat16: the 2^-12 roundings move logits of some ten by 1e-3, where a bfloat16 result is rounded by up to 4e-3.
// KT = 2: two terms each (three products, 22 bits), for float16 and wherever sums of weights are kept.  Weights and value levels are one fp16 value each (the
// reference's own float32 levels are rounded to fp16 by the codec's decompress as well); with KT = 1 a query's sum of weights is made of the rounded weights
// themselves, so that their rounding cancels in part.
template <int D, int IPBK, int IPBV, int QT, int KT>
__global__ __launch_bounds__(FAST_THREADS, FAST_WAVES / 4) void tq_many_fast_kernel(TqManyArgs a) {
    constexpr int STEPS = D / 16, NC = D / 32, KB = D / 2 / IPBK, KW = KB / 4, GBK = D / IPBK, GBV = D / IPBV;
    using Values = ValueBytes<IPBV, NC>;
    constexpr int QW = KT * QT * STEPS * 4;                                        // registers of the queries' operands
    constexpr bool QREG = QW + QT * NC * 16 <= 136;
    constexpr int TC = NC < 4 ? NC : 4, MROW = 32 * TC + 4;                        // sums of a wave on their way through LDS, 32 TC coordinates at a time
    constexpr int LUT_BYTES = 65536, Q_BYTES = QREG ? 0 : KT * QT * STEPS * 1024, MERGE_BYTES = FAST_WAVES * 32 * MROW * 4;
    constexpr int AREA = LUT_BYTES + Q_BYTES > MERGE_BYTES ? LUT_BYTES + Q_BYTES : MERGE_BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[AREA];
    __shared__ __attribute__((aligned(16))) float lds_kn[FAST_WAVES][32];
    __shared__ __attribute__((aligned(16))) uint16_t lds_vn[FAST_WAVES][32];
    __shared__ float lds_m[FAST_WAVES][32 * QT], lds_l[FAST_WAVES][32 * QT];

    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tq_uniform32(tid >> 6), n = lane & 31u, h = lane >> 5;
    const uint32_t groups = (a.tiles + QT - 1u) / QT;
    const uint32_t split = blockIdx.x % a.splits, at = blockIdx.x / a.splits, row = at / groups, tile0 = (at - row * groups) * QT, b = row / a.heads;
    const size_t first_tile = (size_t)row * a.tiles + tile0;
    const bool both = QT == 1 || tile0 + 1u < a.tiles;
    const uint8_t *q_op = a.q_op + first_tile * q_operand_bytes(D);

    if constexpr (KT == 1) {
        Lut<IPBK> table;
        table.load(a.table_k + TQ_OFF_LUT(D), tid);
        table.store(lds, tid);
    } else {
        Lut2<IPBK> table;
        table.load(a.table_k, a.bits_k, D, tid);
        table.store(lds, tid);
    }
    {
        Lut<IPBV> table;
        table.load(a.table_v + TQ_OFF_LUT(D), tid);
        table.store(lds + 128, tid);
    }
    tq_u4 q[QREG ? KT * QT * STEPS : 1];
    // operands of a tile: [term][step][lane]; one term is all that KT = 1 reads
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        const uint8_t *src = q_op + (i && both ? q_operand_bytes(D) : 0u);
        if constexpr (QREG) {
#pragma unroll
            for (int s = 0; s < KT * STEPS; ++s) q[i * KT * STEPS + s] = tq_gload16(src + (size_t)s * 1024u + lane * 16u);
        } else {
            tq_copy_to_lds(lds + LUT_BYTES + i * KT * STEPS * 1024, src, KT * STEPS * 1024, tid, FAST_THREADS);
        }
    }
    auto query = [&](int i, int term, int s) __attribute__((always_inline)) -> tq_u4 {
        if constexpr (QREG) return q[(i * KT + term) * STEPS + s];
        else return *reinterpret_cast<const tq_u4 *>(lds + LUT_BYTES + ((i * KT + term) * STEPS + s) * 1024 + lane * 16u);
    };
    // (the levels of KT = 1 come without 2^LEVEL_SHIFT)
    const float q_scale = a.q_scale[first_tile] * (KT == 1 ? (float)(1 << LEVEL_SHIFT) : 1.f);
    const uint32_t slot_k = KT == 1 ? RepLut<IPBK>::lane_offset(lane) : Lut2<IPBK>::lane_offset(lane);
    const uint32_t slot_v = 128u + (IPBV == 4 && NC == 2 ? (lane & 30u) / 2u * 8u + 4u * (lane & 1u) : RepLut<IPBV>::lane_offset(lane));
    __syncthreads();

    const uint32_t seen = min(a.tokens, many_length(a, b));
    const uint32_t chunk = a.lengths ? ((seen + a.splits - 1u) / a.splits + 31u) / 32u * 32u : a.chunk;       // (a short sequence keeps all its blocks busy)
    const uint32_t begin = min(seen, split * chunk), end = min(seen, begin + chunk);
    const size_t slot0 = (size_t)row * a.packed_row_stride;
    const uint8_t *mask = a.mask ? a.mask + (long long)b * a.mask_stride : nullptr;
    const uint8_t *k_lane = a.k_idx + slot0 * GBK + n * GBK + h * KB;
    const uint8_t *v_lane = a.v_idx + slot0 * GBV + 4u * h * GBV + (IPBV == 4 && NC == 2 ? n / 2u : n * Values::VB);
    const uint16_t *n_lane = (h ? a.v_norms : a.k_norms) + slot0 + n;

    float m_ref[QT], l[QT];
    tq_f16v acc[QT][NC];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        m_ref[i] = FAST_START;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[i][c] = tq_zero16();
    }
    int v_top = -100;                        // 2^v_top: unit of the value norms, their largest binary exponent so far

    // Loads of a run are issued while the one before it is worked on.  The last run of a row begins 32 tokens before the end: what the one before it
    // had already is hidden, and nothing past the row's tokens is read.
    uint32_t kraw[KW];
    Values vraw[16];
    uint16_t norm_raw = 0;
    auto issue_keys = [&](uint32_t t) __attribute__((always_inline)) {
        const uint8_t *p = k_lane + (size_t)t * GBK;
        if constexpr (KB % 16 == 0) {
#pragma unroll
            for (int i = 0; i < KB / 16; ++i) {
                const tq_u4 v = tq_gload16(p + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) kraw[4 * i + j] = v[j];
            }
        } else {
            static_assert(KB == 8, "eight bytes");
            const tq_u2 v = tq_gload8(p);
            kraw[0] = v[0]; kraw[1] = v[1];
        }
        norm_raw = tq_gload2(n_lane + t);
    };
    auto issue_values = [&](uint32_t t) __attribute__((always_inline)) {
        const uint8_t *p = v_lane + (size_t)t * GBV;
#pragma unroll
        for (int j = 0; j < 16; ++j) vraw[j].load(p + (8 * (j / 4) + j % 4) * GBV);
    };
    const uint32_t last = a.tokens - 32u;    // (launched for 32 tokens at least)
    uint32_t t_next = begin + 32u * wave;
    if (t_next < end) {
        issue_keys(min(t_next, last));
        issue_values(min(t_next, last));
    }
    while (t_next < end) {
        const uint32_t t_run = t_next, t0 = min(t_run, last), count = min(32u, end - t_run);
        t_next += 32u * FAST_WAVES;
        const uint32_t t_after = min(t_next < end ? t_next : t_run, last);
        uint32_t hidden = ~((count == 32u ? 0xffffffffu : (1u << count) - 1u) << (t_run - t0));
        if (mask) hidden |= ~(uint32_t)__ballot(mask[t0 + n] != 0);
        // ---- norms: keys' times the queries' scale, values' in the unit of the largest so far
        float norm = (float)__builtin_bit_cast(_Float16, norm_raw);
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
        if (h) lds_vn[wave][n] = __builtin_bit_cast(uint16_t, (_Float16)norm);
        else lds_kn[wave][n] = norm;
        wave_sync();
        // ---- scores
        tq_f16v s[QT];
#pragma unroll
        for (int i = 0; i < QT; ++i) s[i] = tq_zero16();
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            if constexpr (KT == 1) {
                const tq_u4 k = decode_keys<IPBK, KW>(kraw, st, lds, slot_k);
#pragma unroll
                for (int i = 0; i < QT; ++i) s[i] = mfma_f16(k, query(i, 0, st), s[i]);
            } else {
                tq_u4 hi, lo;
                decode_keys2<IPBK, KW>(kraw, st, lds, slot_k, hi, lo);
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
        tq_u4 p[QT][2];
        float kn[16];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const tq_f4 v = *reinterpret_cast<const tq_f4 *>(&lds_kn[wave][8 * k + 4 * h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) kn[4 * k + j] = v[j];
        }
        uint32_t vn[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const tq_u2 v = *reinterpret_cast<const tq_u2 *>(&lds_vn[wave][8 * k + 4 * h]);
            vn[2 * k] = v[0]; vn[2 * k + 1] = v[1];
        }
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            float x[16];
            auto logits = [&]() __attribute__((always_inline)) {
                const float bias = (float)FAST_P - m_ref[i];
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = fmaf(s[i][r], kn[r], bias);
                if (hidden) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] = (hidden >> acc_row(r, h)) & 1u ? -__builtin_inff() : x[r];
                }
            };
            logits();
            float most = x[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) most = fmaxf(most, x[r]);
            if (__any(most > (float)(FAST_P + FAST_SLACK))) {
                float now = -__builtin_inff();
#pragma unroll
                for (int r = 0; r < 16; ++r) now = (hidden >> acc_row(r, h)) & 1u ? now : fmaxf(now, s[i][r] * kn[r]);
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
        // ---- values
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            uint32_t w[8][NC / 2];
#pragma unroll
            for (int j = 0; j < 8; ++j) vraw[8 * st + j].decode(lds, slot_v, w[j]);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                tq_u4 v;
#pragma unroll
                for (int d = 0; d < 4; ++d) v[d] = __builtin_amdgcn_perm(w[2 * d + 1][c / 2], w[2 * d][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int i = 0; i < QT; ++i) acc[i][c] = mfma_f16(v, p[i][st], acc[i][c]);
            }
        }
        issue_values(t_after);
        wave_sync();
    }

    // ---- the waves' sums, and the block's record of each tile
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        l[i] = halves_add(l[i]) * (1.0f / (float)(1 << FAST_P));
        if (h == 0u) {
            lds_m[wave][32 * i + n] = m_ref[i] == FAST_START ? MANY_NONE : m_ref[i];
            lds_l[wave][32 * i + n] = l[i];
        }
    }
    __syncthreads();
    float *area = reinterpret_cast<float *>(lds);
    const float unit = v_top == -100 ? 0.f : __uint_as_float((uint32_t)(127 + v_top - FAST_P) << 23);
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        float m = MANY_NONE;
#pragma unroll
        for (int w = 0; w < FAST_WAVES; ++w) m = fmaxf(m, lds_m[w][32 * i + n]);
        const bool write = i == 0 || both;
        float *rec = a.rec + ((first_tile + i) * a.records + split) * record_floats(D);
        if (tid < 32u && write) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < FAST_WAVES; ++w) sum = fmaf(lds_l[w][32 * i + n], __builtin_amdgcn_exp2f(lds_m[w][32 * i + n] - m), sum);
            rec[n] = m;
            rec[32u + n] = sum;
        }
        const float f = unit * __builtin_amdgcn_exp2f(lds_m[wave][32 * i + n] - m);
#pragma unroll
        for (int c0 = 0; c0 < NC; c0 += TC) {
            if (i || c0) __syncthreads();
#pragma unroll
            for (int c = 0; c < TC; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<tq_f4 *>(area + (wave * 32u + n) * MROW + 32 * c + 8 * k + 4 * h) =
                        tq_f4{acc[i][c0 + c][4 * k] * f, acc[i][c0 + c][4 * k + 1] * f, acc[i][c0 + c][4 * k + 2] * f, acc[i][c0 + c][4 * k + 3] * f};
            __syncthreads();
            if (write) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t pair = tid + e * FAST_THREADS, col = pair / 32u, r = pair % 32u;       // coordinates NC r + c0 ... of query col
                    float sum[TC];
#pragma unroll
                    for (int c = 0; c < TC; ++c) sum[c] = 0.f;
#pragma unroll
                    for (int w = 0; w < FAST_WAVES; ++w)
#pragma unroll
                        for (int c = 0; c < TC; ++c) sum[c] += area[(w * 32 + col) * MROW + 32 * c + r];
                    TQ_GLOBAL float *dst = (TQ_GLOBAL float *)rec + 64u + col * D + NC * r + c0;
                    if constexpr (TC == 4) *reinterpret_cast<TQ_GLOBAL tq_f4 *>(dst) = tq_f4{sum[0], sum[1], sum[2], sum[3]};
                    else { dst[0] = sum[0]; dst[1] = sum[1]; }
                }
            }
        }
    }
}

// ipb: codes per byte
template <int D, int IPBK, int IPBV>
int launch_many_fast(dim3 grid, hipStream_t s, const TqManyArgs &a, int qt, int kt) {
    if (kt == 2) hipLaunchKernelGGL((tq_many_fast_kernel<D, IPBK, IPBV, 1, 2>), grid, dim3(FAST_THREADS), 0, s, a);
    else if (D == 256 || qt == 1) hipLaunchKernelGGL((tq_many_fast_kernel<D, IPBK, IPBV, 1, 1>), grid, dim3(FAST_THREADS), 0, s, a);
    else if constexpr (D != 256) hipLaunchKernelGGL((tq_many_fast_kernel<D, IPBK, IPBV, 2, 1>), grid, dim3(FAST_THREADS), 0, s, a);
    return 0;
}
template <int D, int IPBK>
int launch_many_fast(int ipbv, dim3 grid, hipStream_t s, const TqManyArgs &a, int qt, int kt) {
    if (ipbv == 4) return launch_many_fast<D, IPBK, 4>(grid, s, a, qt, kt);
    if (ipbv == 2) return launch_many_fast<D, IPBK, 2>(grid, s, a, qt, kt);
    return launch_many_fast<D, IPBK, 1>(grid, s, a, qt, kt);
}

}  // namespace
