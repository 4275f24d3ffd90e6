// The kernel behind tq_paged_attend for head dimensions 64, 65 to 96, 128 and 256, codes of one, two or four to a byte (tq_paged.hip).
// One source file per padded head dimension instantiates it.
#pragma once
#include "tq_many_fast.h"
#include "tq_paged.h"

namespace {

// What a block knows of its sequence
struct PagedRow {
    const int32_t *pages, *plain_pages;
    uint32_t fresh, total, packed, kv;
};

// Base-2 logits after the cap: C tanh(z / C) = C - 2 C / (1 + 2^(2 z / cap)), C = cap log2 e.  The difference leaves some 2^-22 C of a logit (so that caps of 16-bit elements end at 1024); where products
// are as exact as float32 (EXACT) small ones come from the series.  (Five instructions, two of them at a quarter of the rate; with series and selection for all, a chunk of 512 tokens over 32768
// took 637 us instead of 374 without a cap.)
struct Cap {
    float rate, c;
    __device__ __forceinline__ explicit Cap(const TqPagedArgs &a) : rate(a.cap != 0.f ? 2.f / a.cap : 0.f), c(a.cap * LOG2E) {}
    template <bool EXACT>
    __device__ __forceinline__ float one(float z) const {
        const float large = fmaf(-2.f * c, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * rate)), c);
        if constexpr (!EXACT) return large;
        else {
            const float y = z * (0.34657359027997265f * rate), y2 = y * y;          // (z / c: half a log 2)
            const float small = z * fmaf(y2, fmaf(y2, fmaf(y2, fmaf(y2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
            return fabsf(y) < 0.3f ? small : large;
        }
    }
    template <bool EXACT, typename X>
    __device__ __forceinline__ void all(X &x, int n) const {
#pragma unroll
        for (int j = 0; j < n; ++j) x[j] = one<EXACT>(x[j]);
    }
};

// Tokens t0 ... t0 + 31 that a query at `pos` does not see, as bits
__device__ __forceinline__ uint32_t unseen_bits(uint32_t t0, uint32_t pos, uint32_t window) {
    uint32_t bits = 0u;
    if (t0 + 31u > pos) bits = t0 > pos ? 0xffffffffu : ~0u << (pos - t0) << 1;
    if (window && pos >= window) {
        const uint32_t first = pos - window + 1u;
        if (first > t0) bits |= first - t0 >= 32u ? 0xffffffffu : (1u << (first - t0)) - 1u;
    }
    return bits;
}

// Infinite and NaN values of plain tokens [from, to) into the joined sums of the queries that see them, whatever their weight (it is not zero).
template <int DP>
__device__ __forceinline__ void paged_wild(const TqPagedArgs &a, const PagedRow &r, float *out, uint32_t tile, uint32_t from, uint32_t to, uint32_t tid) {
    const uint32_t es = a.dtype == TQ_F32 ? 4u : 2u, M = r.fresh * a.group;
#pragma unroll 1
    for (uint32_t e = tid; e < 32u * a.D; e += FAST_THREADS) {
        const uint32_t col = e / a.D, d = e - col * a.D, m = tile * 32u + col;
        if (m >= M) return;
        const uint32_t pos = r.total - r.fresh + m / a.group;
        float sum = 0.f;
#pragma unroll 1
        for (uint32_t t = from; t < to; ++t) {
            const uint8_t *page = a.plain + (long long)r.plain_pages[t >> a.shift] * a.plain_stride + a.plain_v;
            const float v = plain_element(page + (((r.kv << a.shift) + (t & ((1u << a.shift) - 1u))) * a.D + d) * es, a.dtype);
            const uint32_t at = r.packed + t;
            if (!(fabsf(v) < __builtin_inff()) && at <= pos && (!a.window || at + a.window > pos)) sum += v;
        }
        if (sum != 0.f) out[col * (DP + 4u) + d] += sum;
    }
}

// A block's plain tokens against its tiles of queries, sums into LDS.  Eight runs of 32 tokens at a time: a wave has the scores of one run, for all tiles; the waves agree on the largest logit
// of every query, put their weights into LDS as operands, and then a wave has 32 coordinates of the value sums (of every second run, or fourth, where there are fewer than eight such
// slices), so that what they hold need not be joined.  (Against a run a wave with all coordinates, joined at the end: 29000 cycles instead of 55000 for the 320 plain tokens of a block of 64
// bfloat16 query vectors 128 wide, four chunks of 256 tokens over 8191: 138 us instead of 157 for the call.)
// Raw 16-bit products are exact; weights are two terms (bfloat16: 16 bits, half a step of 2^-17 where a result has 2^-9; fp16: 22 bits); float32 elements are three bf16 terms of everything, products down
// to 2^-24 of the largest.  Infinite and NaN values count as zero in the products (they would spread to queries that do not see their token as 0 * inf) and are added after.
template <int DP, int QT, int DT>
__device__ __forceinline__ void paged_plain_phase(const TqPagedArgs &a, const TqManyArgs &v, const PagedRow &r, uint8_t *lds, float *lds_wild, uint32_t tile0, uint32_t tiles, uint32_t from,
                                                  uint32_t to, uint32_t tid) {
    constexpr bool F32 = DT == TQ_F32, BF = DT == TQ_BF16, EVEN = Shape<DP>::EVEN;
    constexpr int STEPS = DP / 16, SLICES = DP / 32, GROUPS = FAST_WAVES / SLICES, PT = F32 ? 3 : 2;
    constexpr int RG = FAST_WAVES / GROUPS, VH = RG < 4 ? RG : 4;          // runs of a group, those whose values are under way at once
    constexpr int CH = F32 ? 1 : EVEN ? 4 : STEPS;                         // steps of a score product that are staged at a time
    constexpr uint32_t ES = F32 ? 4u : 2u, EXPO = BF ? 0x7f807f80u : 0x7c007c00u, ONE = BF ? 0x00800080u : 0x04000400u, ROW = DP + 4u;
    using J = JoinArea<DP, QT>;
    constexpr uint32_t PIECES = 2 * CH, TURN = PIECES % 8u ? 0u : 7u;        // sixteen bytes each of a staged vector; they lie in an order that is turned by the vector's number, so that lanes' reads spread over the banks
    constexpr uint32_t OPERANDS = 2u * QT * PT * 1024u, STAGED = F32 ? 0u : 32u * 16u * PIECES, RUN_BYTES = OPERANDS > STAGED ? OPERANDS : STAGED, STATS = FAST_WAVES * RUN_BYTES;
    static_assert(STATS + FAST_WAVES * QT * 128u <= J::PACKED && (GROUPS - 1u) * QT * 32u * ROW * 4u <= STATS, "beside the packed tokens' sums");
    asm volatile("" : "+v"(tid));    // (what lanes make of their number is made here, not ahead of the loop over packed tokens, which has no register left)
    const uint32_t lane = tid & 63u, wave = tq_uniform32(tid >> 6), n = lane & 31u, h = lane >> 5, runs = (to - from + 31u) / 32u, slice = wave % SLICES, g = wave / SLICES;
    const bool adds = g < (uint32_t)GROUPS;          // (96 wide: two waves have no slice)
    float *const stats = reinterpret_cast<float *>(lds + STATS) + n;       // [wave][tile][32]
    uint8_t *const weights = lds + lane * 16u;       // [run][step][tile][term] operands; before that a wave's keys
    uint8_t *const staged = lds + wave * RUN_BYTES, *const queries = reinterpret_cast<uint8_t *>(J::sums(lds, 1u, 0u));        // [step of CH][tile][32][pieces]
    const Cap cap(a);
    const uint8_t *q[QT];
    uint32_t pos[QT];
    float slope[QT], m_ref[QT], l[QT];
    tq_f16v acc[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        const uint32_t m = min((tile0 + i) * 32u + n, v.M - 1u), token = m / a.group;
        q[i] = many_query(v, 0u, m, ES);
        pos[i] = r.total - r.fresh + token;
        slope[i] = a.slopes ? a.slopes[r.kv * a.group + (m - token * a.group)] * LOG2E : 0.f;
        m_ref[i] = MANY_NONE;
        l[i] = 0.f;
        acc[i] = tq_zero16();
    }
    // pages of the eight runs from r0 on, a lane's each: asked for ahead of the runs before
    auto lookup = [&](uint32_t r0) { return r.plain_pages[min(from + 32u * (r0 + (lane & 7u)), to - 1u) >> a.shift]; };
    int pages = lookup(0u);
    auto first_of = [&](uint32_t r0, uint32_t own) {         // of the head's keys: the first token of the run that is `own`'th of the eight
        const uint32_t t0 = from + 32u * (r0 + own);
        return a.plain + (long long)__builtin_amdgcn_readlane(pages, (int)own) * a.plain_stride + (size_t)((r.kv << a.shift) + (t0 & ((1u << a.shift) - 1u))) * ((EVEN ? (uint32_t)DP : a.D) * ES);
    };
    if constexpr (!F32) {
        // queries into LDS, whole vectors by neighbouring lanes (as operands straight from memory every load touched a line a query)
        auto copy = [&](bool aligned) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t at = tid; at < QT * 32u * (DP / 8u); at += FAST_THREADS) {
                const uint32_t vec = at / (DP / 8u), piece = at % (DP / 8u);
                const tq_u4 x = load_elements(many_query(v, 0u, min(tile0 * 32u + vec, v.M - 1u), ES) + 16u * (EVEN ? piece : min(piece, a.D / 8u - 1u)), aligned);
                *reinterpret_cast<tq_u4 *>(queries + ((piece / PIECES * QT * 32u + vec) * PIECES + ((piece % PIECES) ^ (vec & TURN))) * 16u) = EVEN || 8u * piece < a.D ? x : tq_u4{0u, 0u, 0u, 0u};
            }
        };
        if (v.aligned) copy(true);
        else copy(false);
        __syncthreads();
    }
    uint32_t raw[VH][16];                            // values of coordinate 32 slice + n
    const uint32_t vec_bytes = (EVEN ? (uint32_t)DP : a.D) * ES, v_at = (EVEN ? 32u * slice + n : min(32u * slice + n, a.D - 1u)) * ES + 4u * h * vec_bytes;
    auto load_values = [&](uint32_t r0, int k0) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < VH; ++k) {
            const uint32_t own = g + (uint32_t)((k0 + k) * GROUPS);
            if (!adds || r0 + own >= runs) continue;
            const uint8_t *p = first_of(r0, own) + a.plain_v;
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const uint32_t lane_at = v_at + 16u * st * vec_bytes;        // (whole vectors up to 16 fit the instruction)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint8_t *e = p + lane_at + acc_row(j, 0u) * vec_bytes;
                    if constexpr (F32) raw[k][8 * st + j] = tq_gload4(e);
                    else raw[k][8 * st + j] = tq_gload2(reinterpret_cast<const uint16_t *>(e));
                }
            }
        }
    };
    bool wild = false;
#pragma unroll 1
    for (uint32_t r0 = 0; r0 < runs; r0 += FAST_WAVES) {
        const uint32_t run = r0 + wave, t0 = from + 32u * run;
        const bool some = run < runs;
        float x[QT][16];
        const int pages_after = lookup(r0 + FAST_WAVES);
        if (some) {
            const uint8_t *k = first_of(r0, wave) + (F32 ? n * vec_bytes : 0u);
            tq_u4 keys[F32 ? 1 : STEPS];
            if constexpr (!F32) {
#pragma unroll
                for (int s0 = 0; s0 < STEPS; s0 += CH)
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        if constexpr (EVEN) keys[s0 + i] = tq_gload16(k + (lane / PIECES * vec_bytes + 16u * (lane % PIECES)) + (i * (64u / PIECES) * vec_bytes + 16u * (s0 / CH * PIECES)));
                        else {
                            const uint32_t at = i * 64u + lane, vec = at / PIECES, piece = at % PIECES;
                            const tq_u4 x = tq_gload16(k + vec * vec_bytes + 16u * min(piece, a.D / 8u - 1u));
                            keys[s0 + i] = 8u * piece < a.D ? x : tq_u4{0u, 0u, 0u, 0u};
                        }
                    }
                load_values(r0, 0);
            }
            tq_f16v s[QT];
#pragma unroll
            for (int i = 0; i < QT; ++i) s[i] = tq_zero16();
#pragma unroll(F32 ? 1 : 4)
            for (int s0 = 0; s0 < STEPS; s0 += CH) {
                if constexpr (F32) {
                    tq_u4 kt[3];
                    load_plain8<TQ_F32>(k, 16u * s0 + 8u * h, a.D, true, kt);
#pragma unroll
                    for (int i = 0; i < QT; ++i) {
                        tq_u4 qt[3];
                        load_plain8<TQ_F32>(q[i], 16u * s0 + 8u * h, a.D, v.aligned, qt);
#pragma unroll
                        for (int x0 = 0; x0 < 3; ++x0)
#pragma unroll
                            for (int x1 = 0; x1 < 3 - x0; ++x1) s[i] = mfma_bf16(kt[x0], qt[x1], s[i]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < CH; ++k) {
                        const uint32_t at = k * 64u + lane, vec = at / PIECES, piece = at % PIECES;
                        *reinterpret_cast<tq_u4 *>(staged + (vec * PIECES + (piece ^ (vec & TURN))) * 16u) = keys[s0 + k];
                    }
                    wave_sync();
#pragma unroll
                    for (int st = 0; st < CH; ++st) {
                        const uint32_t piece = (2u * st + h) ^ (n & TURN);
                        const tq_u4 y = *reinterpret_cast<const tq_u4 *>(staged + (n * PIECES + piece) * 16u);
#pragma unroll
                        for (int i = 0; i < QT; ++i) {
                            const tq_u4 z = *reinterpret_cast<const tq_u4 *>(queries + ((s0 / CH * QT * 32 + 32 * i + n) * PIECES + piece) * 16u);
                            s[i] = BF ? mfma_bf16(y, z, s[i]) : mfma_f16(y, z, s[i]);
                        }
                    }
                    wave_sync();
                }
            }
            if (F32) load_values(r0, 0);
            const uint32_t at = r.packed + t0, valid = min(32u, to - t0);
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                const uint32_t gone = (unseen_bits(at, pos[i], a.window) | (valid < 32u ? ~0u << valid : 0u)) >> (4u * h);
#pragma unroll
                for (int j = 0; j < 16; ++j) x[i][j] = s[i][j] * (a.scale * LOG2E);
                if (a.cap != 0.f) cap.template all<F32>(x[i], 16);
                if (a.slopes) {
                    const float first = (float)((int)(at + 4u * h) - (int)pos[i]);
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[i][j] = fmaf(slope[i], first + (float)acc_row(j, 0u), x[i][j]);
                }
                if (__any(gone != 0u)) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[i][j] = (gone >> acc_row(j, 0u)) & 1u ? MANY_NONE : x[i][j];
                }
                float top = x[i][0];
#pragma unroll
                for (int j = 1; j < 16; ++j) top = fmaxf(top, x[i][j]);
                top = halves_max(fmaxf(top, MANY_NONE));
                if (h == 0u) stats[(wave * QT + i) * 32u] = top;
            }
        } else {
            load_values(r0, 0);
#pragma unroll
            for (int i = 0; i < QT; ++i)
                if (h == 0u) stats[(wave * QT + i) * 32u] = MANY_NONE;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            float now = m_ref[i];
#pragma unroll
            for (int w = 0; w < FAST_WAVES; ++w) now = fmaxf(now, stats[(w * QT + i) * 32]);
            const float shrink = __builtin_amdgcn_exp2f(m_ref[i] - now);
            m_ref[i] = now;
            l[i] *= shrink;              // (this lane's tokens)
            acc[i] *= shrink;
            if (!some) continue;
            const float least = now == MANY_NONE ? 0.f : now;        // (no token seen so far: weights of zero)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                x[i][j] = __builtin_amdgcn_exp2f(x[i][j] - least);
                l[i] += x[i][j];
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                tq_u4 p[3];
                float ps[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) ps[j] = x[i][8 * st + j];
                if constexpr (BF || F32) bf16_terms(ps, p);
                else fp16_split8(tq_f4{ps[0], ps[1], ps[2], ps[3]}, tq_f4{ps[4], ps[5], ps[6], ps[7]}, 1.f, p[0], p[1]);
#pragma unroll
                for (int t = 0; t < PT; ++t) *reinterpret_cast<tq_u4 *>(weights + (((wave * 2u + st) * QT + i) * PT + t) * 1024u) = p[t];
            }
        }
        __syncthreads();
        if (adds) {
#pragma unroll
        for (int k0 = 0; k0 < RG; k0 += VH) {
            if (k0) load_values(r0, k0);
#pragma unroll
            for (int k = 0; k < VH; ++k) {
                const uint32_t own = g + (uint32_t)((k0 + k) * GROUPS), left = to - min(to, from + 32u * (r0 + own));       // of the eight; its tokens and those behind them
                if (!left) continue;
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    tq_u4 o[3];
                    if (left < 32u) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) raw[k][8 * st + j] = acc_row(8 * st + j, h) < left ? raw[k][8 * st + j] : 0u;
                    }
                    if constexpr (F32) {
                        float e[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float value = __uint_as_float(raw[k][8 * st + j]);
                            const bool fine = fabsf(value) < __builtin_inff();
                            wild = wild || !fine;
                            e[j] = fine ? value : 0.f;
                        }
                        bf16_terms(e, o);
                    } else {
                        uint32_t over = 0u;
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            o[0][d] = raw[k][8 * st + 2 * d] | raw[k][8 * st + 2 * d + 1] << 16;
                            over |= (o[0][d] & EXPO) + ONE;          // (an exponent of ones carries into the sign's place)
                        }
                        if (__any((over & 0x80008000u) != 0u)) {
                            wild = true;
#pragma unroll
                            for (int d = 0; d < 4; ++d) o[0][d] &= ~(((((o[0][d] & EXPO) + ONE) >> 15) & 0x00010001u) * 0xffffu);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < QT; ++i) {
                        tq_u4 p[PT];
#pragma unroll
                        for (int t = 0; t < PT; ++t) p[t] = *reinterpret_cast<const tq_u4 *>(weights + (((own * 2u + st) * QT + i) * PT + t) * 1024u);
#pragma unroll
                        for (int t = 0; t < PT; ++t) {
                            if constexpr (F32) {
#pragma unroll
                                for (int x0 = 0; x0 < 3 - t; ++x0) acc[i] = mfma_bf16(o[x0], p[t], acc[i]);
                            } else acc[i] = BF ? mfma_bf16(o[0], p[t], acc[i]) : mfma_f16(o[0], p[t], acc[i]);
                        }
                    }
                }
            }
        }
        }
        pages = pages_after;
        __syncthreads();             // (weights and stats have been read)
    }
    wild = __any(wild);
    if (lane == 0u) lds_wild[wave] = wild ? 1.f : 0.f;
    float *const others = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        const float both = halves_add(l[i]);
        if (h == 0u) stats[(wave * QT + i) * 32u] = both;
        if (GROUPS > 1 && adds && g) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<tq_f4 *>(others + (((g - 1u) * QT + i) * 32u + n) * ROW + 32u * slice + 8u * k + 4u * h) = tq_f4{acc[i][4 * k], acc[i][4 * k + 1], acc[i][4 * k + 2], acc[i][4 * k + 3]};
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        if (g == 0u) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                tq_f4 sum = tq_f4{acc[i][4 * k], acc[i][4 * k + 1], acc[i][4 * k + 2], acc[i][4 * k + 3]};
#pragma unroll
                for (int o = 0; o < GROUPS - 1; ++o) sum += *reinterpret_cast<const tq_f4 *>(others + ((o * QT + i) * 32u + n) * ROW + 32u * slice + 8u * k + 4u * h);
                *reinterpret_cast<tq_f4 *>(J::sums(lds, 1u, i) + n * ROW + 32u * slice + 8u * k + 4u * h) = sum;
            }
        }
        if (wave == (uint32_t)i && h == 0u) {
            float total = 0.f;
#pragma unroll
            for (int w = 0; w < FAST_WAVES; ++w) total += stats[(w * QT + i) * 32];
            J::largest(lds, 1u, i)[n] = m_ref[i];
            J::total(lds, 1u, i)[n] = total;
        }
    }
    __syncthreads();
    float any = 0.f;
#pragma unroll
    for (int w = 0; w < FAST_WAVES; ++w) any += lds_wild[w];
    if (any != 0.f) {
#pragma unroll 1
        for (uint32_t i = 0; i < tiles; ++i) paged_wild<DP>(a, r, J::sums(lds, 1u, i), tile0 + i, from, to, tid);
        __syncthreads();
    }
}

// Coordinates d0 ... d0 + 15 of query vector m's result
__device__ __forceinline__ void paged_store(const TqPagedArgs &a, uint32_t q_first, uint32_t kv, uint32_t m, uint32_t d0, const float (&o)[16]) {
    const uint32_t token = m / a.group;
    const size_t first = ((size_t)(q_first + token) * (a.heads * a.group) + kv * a.group + (m - token * a.group)) * a.D + d0;
    if (d0 >= a.D) return;
    if (a.dtype != TQ_F32 && !(a.D & 15u) && !((uintptr_t)a.out & 15u)) {
        uint32_t w[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            if (a.dtype == TQ_F16) w[d] = __builtin_bit_cast(uint32_t, tq_half2{(_Float16)o[2 * d], (_Float16)o[2 * d + 1]});
            else w[d] = __builtin_bit_cast(uint32_t, tq_bf2{(__bf16)o[2 * d], (__bf16)o[2 * d + 1]});
        }
        tq_gstore16(a.out + first * 2u, tq_u4{w[0], w[1], w[2], w[3]});
        tq_gstore16(a.out + first * 2u + 16u, tq_u4{w[4], w[5], w[6], w[7]});
        return;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        if (d0 + r >= a.D) continue;
        if (a.dtype == TQ_F32) {
            reinterpret_cast<TQ_GLOBAL float *>((TQ_GLOBAL uint8_t *)a.out)[first + r] = o[r];
        } else {
            uint16_t e;
            if (a.dtype == TQ_F16) e = __builtin_bit_cast(uint16_t, (_Float16)o[r]);
            else e = __builtin_bit_cast(uint16_t, (__bf16)o[r]);
            reinterpret_cast<TQ_GLOBAL uint16_t *>((TQ_GLOBAL uint8_t *)a.out)[first + r] = e;
        }
    }
}

// Joined sums of a column as they lie in LDS: packed tokens' (value space of the codec; null: none) and plain ones', their largest logits and sums of weights
struct JoinedColumn {
    const float *packed, *plain;
    float m0, l0, m1, l1;
};

// A wave's 32 coordinates of 32 columns' results: packed sums turned back by Pi_v (two fp16 terms each), the plain ones added; divided by the sum of weights into the result of query vector q, or as they are into
// column `col` of the record.  `some`: whether the lane's column is one.
template <int DP>
__device__ __forceinline__ void paged_finish(const TqPagedArgs &a, const JoinedColumn &j, uint32_t kv, uint32_t q_first, TQ_GLOBAL float *rec, uint32_t q, uint32_t col, bool some,
                                             uint32_t w, uint32_t lane) {
    constexpr int STEPS = DP / 16, CH = STEPS < 8 ? STEPS : 8;
    const uint32_t h = lane >> 5;
    const bool packed = j.packed != nullptr, plain = j.plain != nullptr;
    const float m = fmaxf(j.m0, j.m1);
    // (no largest logit: no token seen, or logits that are all NaN, which the sum of weights tells)
    const float f0 = j.m0 != MANY_NONE ? __builtin_amdgcn_exp2f(j.m0 - m) : j.l0 == 0.f ? 0.f : __builtin_nanf("");
    const float f1 = j.m1 != MANY_NONE ? __builtin_amdgcn_exp2f(j.m1 - m) : j.l1 == 0.f ? 0.f : __builtin_nanf("");
    const float l = j.l0 * f0 + j.l1 * f1, inv = 1.0f / l;         // (of a result a query's own token is part: a sum of zero is that of logits which are all -infinity, and 0 / 0 what comes of it)
    tq_f16v acc = tq_zero16();
    float back = 0.f;
    if (packed) {
        const float *o = j.packed;
        const uint8_t *pi = a.table_v + TQ_OFF_AT_F16(DP) + ((size_t)w * STEPS * 64u + lane) * 16u;
        float largest = 0.f;
#pragma unroll 8
        for (uint32_t d = 0; d < DP / 2u; d += 4u) {
            const tq_f4 x = *reinterpret_cast<const tq_f4 *>(o + h * (DP / 2u) + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) largest = fmaxf(largest, fabsf(x[e]) < __builtin_inff() ? fabsf(x[e]) : 0.f);
        }
        largest = halves_max(largest);
        const int up = largest > 0.f ? max(-100, min(100, Q_TOP - ((int)(__float_as_uint(largest) >> 23) - 127))) : 0;
        const float f = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll 1
        for (int s0 = 0; s0 < STEPS; s0 += CH) {
            tq_u4 ph[CH], pl[CH];
#pragma unroll
            for (int s = 0; s < CH; ++s) { ph[s] = tq_gload16(pi + (size_t)(s0 + s) * 1024u); pl[s] = tq_gload16(pi + TQ_OPERAND_BYTES_FOR(DP) + (size_t)(s0 + s) * 1024u); }
#pragma unroll
            for (int s = 0; s < CH; ++s) {
                const uint32_t i = DP == TQ_HEAD_DIM ? 64u * h + 8u * (s0 + s) : 16u * (s0 + s) + 8u * h;       // (128 wide the table's operands have an order of their own, see tq_table.h)
                tq_f4 x = *reinterpret_cast<const tq_f4 *>(o + i), y = *reinterpret_cast<const tq_f4 *>(o + i + 4u);
                if (!Shape<DP>::EVEN && i >= a.D) x = y = tq_f4{0.f, 0.f, 0.f, 0.f};        // (D a multiple of 8; what lies past it may be anything)
                tq_u4 oh, ol;
                fp16_split8(x, y, f, oh, ol);
                acc = mfma_f16(ph[s], oh, acc);
                acc = mfma_f16(ph[s], ol, acc);
                acc = mfma_f16(pl[s], oh, acc);
            }
        }
        back = __uint_as_float((uint32_t)(127 - up) << 23) * f0;
    }
    if (!some) return;
    const uint32_t d0 = DP == TQ_HEAD_DIM ? 64u * h + 16u * w : 32u * w + 16u * h;
    float out[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) out[r] = (packed ? acc[r] * back : 0.f) + (plain ? j.plain[d0 + r] * f1 : 0.f);
    if (!rec) {
#pragma unroll
        for (int r = 0; r < 16; ++r) out[r] *= inv;
        paged_store(a, q_first, kv, q, d0, out);
        return;
    }
    if (w == 0u && h == 0u) { rec[col] = m; rec[a.cols + col] = l; }
#pragma unroll
    for (int r = 0; r < 16; r += 4) *reinterpret_cast<TQ_GLOBAL tq_f4 *>(rec + 2u * a.cols + col * DP + d0 + r) = tq_f4{out[r], out[r + 1], out[r + 2], out[r + 3]};
}

// Block = (item of the plan, kv head): QT tiles of 32 queries of a sequence against a share of what they see, packed tokens first, then plain ones.  The loop over packed tokens is the one of
// tq_many_fast_kernel (where its numbers of terms are explained), with runs of 32 tokens found through the sequence's pages: a run never crosses a page, whose number is fetched two
// runs ahead.  Causality concerns plain tokens only (the step's own are never packed), a sliding window either kind, as bits per query in the runs that its edge crosses.
template <int DP, int IPBK, int IPBV, int QT, int KT, int VT>
__global__ __launch_bounds__(FAST_THREADS, FAST_WAVES / 4) void tq_paged_kernel(TqPagedArgs a) {
    using S = Shape<DP>;
    using Keys = KeyRun<DP, IPBK>;
    constexpr int STEPS = S::STEPS, NC = S::NC, GBV_MAX = DP / IPBV;
    using Values = ValueBytes<IPBV, NC>;
    constexpr int QW = KT * QT * STEPS * 4;
    constexpr bool QREG = QW + QT * NC * 16 <= 136;
    constexpr float LARGE = (float)(1 << 20) / ((float)(1 << 16) * (DP <= 64 ? 8.f : 16.f) * (KT == 2 ? (float)(1 << LEVEL_SHIFT) : 1.f));
    constexpr int LUT_BYTES = 65536, Q_BYTES = KT * QT * STEPS * 1024;
    constexpr bool STAGE = !S::EVEN || GBV_MAX <= 128;
    constexpr int VPIECES = S::EVEN ? (GBV_MAX >= 32 ? GBV_MAX / 32 : 1) : (GBV_MAX + 31) / 32;
    constexpr uint32_t WAVE_BYTES = Keys::BYTES + (STAGE ? 32u * GBV_MAX : 0u);
    using J = JoinArea<DP, QT>;
    constexpr uint32_t LOOP_BYTES = LUT_BYTES + Q_BYTES + FAST_WAVES * WAVE_BYTES + (S::EVEN ? 0u : 64u);
    constexpr uint32_t AREA = LOOP_BYTES > J::BYTES ? LOOP_BYTES : J::BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[AREA];
    __shared__ __attribute__((aligned(16))) float lds_kn[FAST_WAVES][32];
    __shared__ __attribute__((aligned(16))) std::conditional_t<VT == 2, float, uint16_t> lds_vn[FAST_WAVES][32];
    __shared__ float lds_m[FAST_WAVES][32], lds_l[FAST_WAVES][32], lds_own[QT][32];

    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tq_uniform32(tid >> 6), n = lane & 31u, h = lane >> 5;
    const uint32_t item = blockIdx.x / a.heads;
    const int32_t *it = a.items + (size_t)item * PAGED_ITEM;
    if (it[0] < 0) return;                   // (a plan that is over)
    const int32_t *sq = a.seqs + (size_t)it[0] * PAGED_SEQ;
    const uint32_t tile0 = (uint32_t)it[1], begin = (uint32_t)it[2], end = (uint32_t)it[3], plain_from = (uint32_t)it[4], plain_to = (uint32_t)it[5];
    const int record = it[6];
    PagedRow row;
    row.fresh = (uint32_t)sq[1]; row.total = (uint32_t)sq[2]; row.packed = (uint32_t)sq[3];
    row.pages = a.tables + sq[4]; row.plain_pages = a.tables + sq[5];
    row.kv = blockIdx.x - item * a.heads;
    const uint32_t q_first = (uint32_t)sq[0];
    // the sequence's queries as the rotation takes them: "heads" are its tokens here
    TqManyArgs v;
    v.q = a.q + ((long long)q_first * a.q_token + (long long)(row.kv * a.group) * a.q_head) * (a.dtype == TQ_F32 ? 4 : 2);
    v.q_batch = 0; v.q_head = a.q_token; v.q_token = a.q_head;
    v.heads = 1u; v.group = 0u; v.queries = a.group; v.M = row.fresh * a.group; v.D = a.D; v.dtype = a.dtype; v.scale = a.scale; v.aligned = a.aligned; v.table_k = a.table_k;
    const uint32_t tiles = min((uint32_t)QT, (v.M + 31u) / 32u - tile0);

    if (end > begin) {
        const uint32_t GBK = S::EVEN ? DP / IPBK : (a.D + IPBK - 1u) / IPBK, GBV = S::EVEN ? DP / IPBV : (a.D + IPBV - 1u) / IPBV;
        const uint32_t v_lane = 4u * h * GBV + (IPBV == 4 && NC == 2 ? n / 2u : n * Values::VB);
        Keys keys;
        tq_u4 vpiece[VPIECES];
        Values vraw[16];
        uint16_t kn_raw = 0, vn_raw = 0;
        uint8_t *kstage = lds + LUT_BYTES + Q_BYTES + wave * WAVE_BYTES, *vstage = kstage + Keys::BYTES;
        const uint32_t place_mask = (1u << a.shift) - 1u, last = (end - 1u) & ~31u;
        auto page_of = [&](uint32_t t) { return (int)tq_uniform32((uint32_t)row.pages[min(t, last) >> a.shift]); };
        auto place_of = [&](uint32_t t) { return (row.kv << a.shift) + (min(t, last) & place_mask); };       // of the layer's part of a page
        auto issue_keys = [&](int page, uint32_t place) __attribute__((always_inline)) {
            const uint8_t *p = a.pool + (long long)page * a.page_stride;
            keys.issue(p + (size_t)place * GBK, GBK, lane);
            kn_raw = tq_gload2(reinterpret_cast<const uint16_t *>(p + a.k_norms) + place + n);
            vn_raw = tq_gload2(reinterpret_cast<const uint16_t *>(p + a.v_norms) + place + n);
        };
        auto issue_values = [&](int page, uint32_t place) __attribute__((always_inline)) {
            const uint8_t *p = a.pool + (long long)page * a.page_stride + a.v_idx + (size_t)place * GBV;
            if constexpr (!STAGE) {
#pragma unroll
                for (int j = 0; j < 16; ++j) vraw[j].load(p + v_lane + (8 * (j / 4) + j % 4) * GBV);
            } else if constexpr (!S::EVEN) {
#pragma unroll
                for (int i = 0; i < VPIECES; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) vpiece[i][k] = tq_gload4(p + 4u * min(256u * i + 64u * k + lane, 8u * GBV - 1u));
            } else if constexpr (GBV_MAX == 16) {
                const tq_u2 x = tq_gload8(p + lane * 8u);
                vpiece[0][0] = x[0]; vpiece[0][1] = x[1];
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
        constexpr uint32_t STRIDE = 32u * FAST_WAVES;
        uint32_t t_next = begin + 32u * wave;
        int page = page_of(t_next), page_next = page_of(t_next + STRIDE);
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
            r.load(v, 0u, tile0, wave, lane);
            if (t_next < end) {
                issue_keys(page, place_of(t_next));
                issue_values(page, place_of(t_next));
            }
            __builtin_amdgcn_sched_barrier(0);
            table_k.store(lds, tid);
            table_v.store(lds + 128, tid);
            q_scale = r.finish(v, ops, lds_kn, lds_own, apart, wave, lane);
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
        const uint32_t slot_k = KT == 1 ? RepLut<IPBK>::lane_offset(lane) : Lut2<IPBK>::lane_offset(lane);
        const uint32_t slot_v = 128u + (VT == 2 ? Lut2<IPBV>::lane_offset(lane) : IPBV == 4 && NC == 2 ? (lane & 30u) / 2u * 8u + 4u * (lane & 1u) : RepLut<IPBV>::lane_offset(lane));

        float m_ref[QT], l[QT], slope[QT];
        uint32_t pos[QT];
        tq_f16v acc[QT][NC];
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            const uint32_t m = min((tile0 + i) * 32u + n, v.M - 1u), token = m / a.group;
            pos[i] = row.total - row.fresh + token;
            slope[i] = a.slopes ? a.slopes[row.kv * a.group + (m - token * a.group)] * LOG2E : 0.f;
            m_ref[i] = MANY_NONE;
            l[i] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[i][c] = tq_zero16();
        }
        const bool shaped = a.cap != 0.f || a.slopes;
        const Cap cap(a);
        // runs that begin before this are not seen whole by the last query of the block
        const uint32_t last_pos = row.total - row.fresh + min((tile0 + QT) * 32u - 1u, v.M - 1u) / a.group;
        const uint32_t whole_from = a.window && last_pos >= a.window ? last_pos - a.window + 1u : 0u;
        int v_top = -100;                        // 2^v_top: unit of the value norms, their largest binary exponent so far
        while (t_next < end) {
            const uint32_t t0 = t_next, count = min(32u, end - t0);
            t_next += STRIDE;
            // (the two waves of a SIMD go first in turn: left to itself the older one runs ahead, and the other then ends alone)
            if (((t0 / STRIDE) ^ (wave >> 2)) & 1u) __builtin_amdgcn_s_setprio(1);
            else __builtin_amdgcn_s_setprio(0);
            const uint32_t place_after = place_of(t_next);
            const int page_after = page_next;
            page_next = page_of(t_next + STRIDE);
            const uint32_t hidden = count == 32u ? 0u : ~0u << count;
            const bool cut = t0 < whole_from;
            // ---- norms: keys' times the queries' scale, values' in the unit of the largest so far
            float norm = (float)__builtin_bit_cast(_Float16, h ? vn_raw : kn_raw);
            if (hidden) norm = (hidden >> n) & 1u ? 0.f : norm;
            if (cut) {
                // Where not all queries see a token, an infinite norm of its values times a weight of 0 would make NaN of those that do not: it is zero there, and the keys' norm NaN, which
                // makes NaN of the logits of those that do.  (Logits are masked by selection.  Masking products or norms by tile: 5 to 10 registers more are spilled in the loop.)
                const uint32_t wild = (uint32_t)(__ballot(!(norm < __builtin_inff())) >> 32);
                if ((wild >> n) & 1u) norm = h ? 0.f : __builtin_nanf("");
            }
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
                issue_values(page_after, place_after);
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
            issue_keys(page_after, place_after);
            // ---- weights
            tq_u4 p[QT][2], p2[VT == 2 ? QT : 1][2];
            float kn[16];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const tq_f4 x = *reinterpret_cast<const tq_f4 *>(&lds_kn[wave][8 * k + 4 * h]);
#pragma unroll
                for (int j = 0; j < 4; ++j) kn[4 * k + j] = x[j];
            }
            uint32_t vn[VT == 2 ? 16 : 8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (VT == 2) {
                    const tq_u4 x = *reinterpret_cast<const tq_u4 *>(&lds_vn[wave][8 * k + 4 * h]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) vn[4 * k + j] = x[j];
                } else {
                    const tq_u2 x = *reinterpret_cast<const tq_u2 *>(&lds_vn[wave][8 * k + 4 * h]);
                    vn[2 * k] = x[0]; vn[2 * k + 1] = x[1];
                }
            }
            if (large || apart || shaped) {
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
                if (a.cap != 0.f) {
#pragma unroll
                    for (int i = 0; i < QT; ++i) cap.template all<VT == 2>(s[i], 16);
                }
                if (a.slopes) {
#pragma unroll
                    for (int i = 0; i < QT; ++i) {
                        const float first = (float)((int)(t0 + 4u * h) - (int)pos[i]);
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[i][r] = fmaf(slope[i], first + (float)acc_row(r, 0u), s[i][r]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                float x[16];
                uint32_t gone = hidden;
                if (cut) gone |= unseen_bits(t0, pos[i], a.window);
                auto logits = [&]() __attribute__((always_inline)) {
                    const float bias = (float)FAST_P - m_ref[i];
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] = fmaf(s[i][r], kn[r], bias);
                    if (hidden || cut) {        // (opaque: in its branch, not ahead of it for every run)
                        uint32_t bits = gone >> (4u * h);
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
                    uint32_t bits = gone >> (4u * h);
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
                    Values x;
                    if constexpr (STAGE) x.fetch(vstage + v_lane + (16 * st + 8 * (j / 4) + j % 4) * GBV);
                    else x = vraw[8 * st + j];
                    if constexpr (VT == 2) decode_values2<IPBV, NC>(x, lds, slot_v, n & 1u, w[j], w2[j]);
                    else x.decode(lds, slot_v, w[j]);
                }
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    auto operand = [&](const auto &y) __attribute__((always_inline)) {
                        tq_u4 o;
#pragma unroll
                        for (int d = 0; d < 4; ++d) o[d] = __builtin_amdgcn_perm(y[2 * d + 1][c / 2], y[2 * d][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
                        return o;
                    };
                    const tq_u4 o = operand(w);
#pragma unroll
                    for (int i = 0; i < QT; ++i) acc[i][c] = mfma_f16(o, p[i][st], acc[i][c]);
                    if constexpr (VT == 2) {
                        const tq_u4 o2 = operand(w2);
#pragma unroll
                        for (int i = 0; i < QT; ++i) {
                            acc[i][c] = mfma_f16(o, p2[i][st], acc[i][c]);
                            acc[i][c] = mfma_f16(o2, p[i][st], acc[i][c]);
                        }
                    }
                }
            }
            if constexpr (!STAGE) issue_values(page_after, place_after);
            wave_sync();
        }
        __builtin_amdgcn_s_setprio(0);
        // ---- the waves' sums
        const float unit = v_top == -100 ? 0.f : __uint_as_float((uint32_t)(127 + v_top - FAST_P - (VT == 2 ? LEVEL_SHIFT : 0)) << 23);
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            __syncthreads();
            join_waves<DP, FAST_WAVES>(reinterpret_cast<float *>(lds), lds_m, lds_l, J::sums(lds, 0u, i), J::largest(lds, 0u, i), J::total(lds, 0u, i), 0u, unit, m_ref[i],
                                       l[i] * (1.0f / (float)(1 << FAST_P)), acc[i], tid);
        }
        __syncthreads();
    }
    const bool plain = plain_to > plain_from;
    if (plain) {
        if constexpr (VT == 2) paged_plain_phase<DP, QT, TQ_F32>(a, v, row, lds, lds_kn[0], tile0, tiles, plain_from, plain_to, tid);
        else if (a.dtype == TQ_BF16) paged_plain_phase<DP, QT, TQ_BF16>(a, v, row, lds, lds_kn[0], tile0, tiles, plain_from, plain_to, tid);
        else if constexpr (KT == 2) paged_plain_phase<DP, QT, TQ_F16>(a, v, row, lds, lds_kn[0], tile0, tiles, plain_from, plain_to, tid);
    }
    const uint32_t i = wave / S::TILES;
    if (i >= tiles) return;
    const bool packed = end > begin;
    JoinedColumn j;
    j.packed = packed ? J::sums(lds, 0u, i) + n * (DP + 4u) : nullptr;
    j.plain = plain ? J::sums(lds, 1u, i) + n * (DP + 4u) : nullptr;
    j.m0 = packed ? J::largest(lds, 0u, i)[n] : MANY_NONE; j.l0 = packed ? J::total(lds, 0u, i)[n] : 0.f;
    j.m1 = plain ? J::largest(lds, 1u, i)[n] : MANY_NONE; j.l1 = plain ? J::total(lds, 1u, i)[n] : 0.f;
    const uint32_t q = (tile0 + i) * 32u + n;
    TQ_GLOBAL float *rec = record < 0 ? nullptr : (TQ_GLOBAL float *)a.rec + (((size_t)record + row.kv) * a.qt + i) * paged_record(a.cols, DP);
    paged_finish<DP>(a, j, row.kv, q_first, rec, q, n, record < 0 ? q < v.M : n < a.cols, wave % S::TILES, lane);
}

template <int DP, int IPBK, int IPBV>
int launch_paged(dim3 grid, hipStream_t s, const TqPagedArgs &a, int qt, int kt, int vt) {
    if (vt == 2) hipLaunchKernelGGL((tq_paged_kernel<DP, IPBK, IPBV, 1, 2, 2>), grid, dim3(FAST_THREADS), 0, s, a);
    else if (DP == 96 || DP == 256 || qt == 1) {
        if (kt == 2) hipLaunchKernelGGL((tq_paged_kernel<DP, IPBK, IPBV, 1, 2, 1>), grid, dim3(FAST_THREADS), 0, s, a);
        else hipLaunchKernelGGL((tq_paged_kernel<DP, IPBK, IPBV, 1, 1, 1>), grid, dim3(FAST_THREADS), 0, s, a);
    } else if constexpr (DP == 64 || DP == 128) {
        if (kt == 2) hipLaunchKernelGGL((tq_paged_kernel<DP, IPBK, IPBV, 2, 2, 1>), grid, dim3(FAST_THREADS), 0, s, a);
        else hipLaunchKernelGGL((tq_paged_kernel<DP, IPBK, IPBV, 2, 1, 1>), grid, dim3(FAST_THREADS), 0, s, a);
    }
    return 0;
}
template <int DP>
int launch_paged(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, int qt, int kt, int vt) {
    if (ipbk == 4) return ipbv == 4 ? launch_paged<DP, 4, 4>(grid, s, a, qt, kt, vt) : ipbv == 2 ? launch_paged<DP, 4, 2>(grid, s, a, qt, kt, vt) : launch_paged<DP, 4, 1>(grid, s, a, qt, kt, vt);
    if (ipbk == 2) return ipbv == 4 ? launch_paged<DP, 2, 4>(grid, s, a, qt, kt, vt) : ipbv == 2 ? launch_paged<DP, 2, 2>(grid, s, a, qt, kt, vt) : launch_paged<DP, 2, 1>(grid, s, a, qt, kt, vt);
    return ipbv == 4 ? launch_paged<DP, 1, 4>(grid, s, a, qt, kt, vt) : ipbv == 2 ? launch_paged<DP, 1, 2>(grid, s, a, qt, kt, vt) : launch_paged<DP, 1, 1>(grid, s, a, qt, kt, vt);
}

}  // namespace
