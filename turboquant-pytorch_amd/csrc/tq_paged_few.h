// The kernel behind tq_paged_attend for sequences with few query vectors a kv head (a token or two of each: decoding), 16-bit elements, head dimensions 64, 96, 128 and 256.
// One source file per head dimension instantiates it.
#pragma once
#include "tq_decode_kernel.h"
#include "tq_paged_kernel.h"

namespace {

// 32 uncompressed tokens of a page against up to 16 query vectors: scores as raw 16-bit products, softmax, weights in three bf16 terms (fp16: two of fp16) times the raw values.  Infinite
// and NaN values count as zero here (`wild` says whether there are any, see paged_wild).
template <int D, bool BF>
struct FewPlain {
    static constexpr int SK = D / 32, NC = D / 16, PT = BF ? 3 : 2;
    static constexpr bool HELD = D <= 128;
    static constexpr int VW = HELD ? NC / 2 : 4;         // words of a lane's coordinates that are held at a time
    static constexpr uint32_t EXPO = BF ? 0x7f807f80u : 0x7c007c00u, ONE = BF ? 0x00800080u : 0x04000400u;
    static constexpr int KH = HELD ? SK : 1, CH = HELD ? SK : 2;      // 256 wide keys do not fit beside the sums: two steps at a time
    tq_u4 k[KH][2];
    uint32_t v[8][VW];
    const uint8_t *kw, *vw;
    uint32_t valid;
    static __device__ __forceinline__ uint32_t token(int j, uint32_t q4) { return 16u * (j / 4) + 4u * q4 + (uint32_t)(j % 4); }
    // N coordinates from c0 on, into words w0 ...
    template <int N> __device__ __forceinline__ void load_columns(uint32_t lane, int c0, int w0) {
        const uint32_t first = value_coord<D>(lane & 15u, c0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint8_t *src = vw + token(j, lane >> 4) * (2u * D) + 2u * first;
            if constexpr (N == 8) { const tq_u4 x = tq_gload16(src); v[j][w0] = x[0]; v[j][w0 + 1] = x[1]; v[j][w0 + (VW > 2 ? 2 : 0)] = x[2]; v[j][w0 + (VW > 3 ? 3 : 0)] = x[3]; }
            else if constexpr (N == 4) { const tq_u2 x = tq_gload8(src); v[j][w0] = x[0]; v[j][w0 + 1] = x[1]; }
            else v[j][w0] = tq_gload4(src);
        }
    }
    // keys, values: of the head's first of the 32 tokens (the page holds all of them; those from `valid` on are not used)
    __device__ __forceinline__ void load(const uint8_t *keys, const uint8_t *values, uint32_t valid_, uint32_t lane) {
        valid = valid_;
        kw = keys + (lane & 15u) * (2u * D) + 16u * (lane >> 4);
        vw = values;
        if constexpr (HELD) {
#pragma unroll
            for (int s = 0; s < SK; ++s)
#pragma unroll
                for (int b = 0; b < 2; ++b) k[s][b] = tq_gload16(kw + b * (32u * D) + 64 * s);
        }
        if constexpr (D == 64 || D == 128) load_columns<NC>(lane, 0, 0);
        else if constexpr (D == 96) { load_columns<4>(lane, 0, 0); load_columns<2>(lane, 4, 2); }
    }
    // q: this lane's column's vector, from element 8 q4 on
    __device__ __forceinline__ void scores(const uint8_t *q, float (&x)[8]) const {
        tq_f4v sc[2] = {tq_f4v{0.f, 0.f, 0.f, 0.f}, tq_f4v{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
        for (int s0 = 0; s0 < SK; s0 += CH) {
            tq_u4 y[CH], z[CH][2];
#pragma unroll
            for (int s = 0; s < CH; ++s) {
                y[s] = tq_gload16(q + 64 * (s0 + s));
#pragma unroll
                for (int b = 0; b < 2; ++b) z[s][b] = HELD ? k[HELD ? s : 0][b] : tq_gload16(kw + b * (32u * D) + 64 * (s0 + s));
            }
#pragma unroll
            for (int s = 0; s < CH; ++s)
#pragma unroll
                for (int b = 0; b < 2; ++b) sc[b] = BF ? mfma16_bf16(z[s][b], y[s], sc[b]) : mfma16_f16(z[s][b], y[s], sc[b]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = sc[j / 4][j % 4];
    }
    __device__ __forceinline__ void tame(uint32_t lane, bool &wild) {
        uint32_t over = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int c = 0; c < VW; ++c) {
                if (token(j, lane >> 4) >= valid) v[j][c] = 0u;
                over |= (v[j][c] & EXPO) + ONE;          // (an exponent of ones carries into the sign's place)
            }
        if (__any((over & 0x80008000u) != 0u)) {
            wild = true;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < VW; ++c) v[j][c] &= ~(((((v[j][c] & EXPO) + ONE) >> 15) & 0x00010001u) * 0xffffu);
        }
    }
    // acc[c]: register r = column 4 q4 + r, coordinate value_coord(n16, c)
    __device__ __forceinline__ void values(const float (&p)[8], uint32_t lane, bool &wild, tq_f4v (&acc)[NC]) {
        tq_u4 pa[3];
        if constexpr (BF) bf16_terms(p, pa);
        else {
            uint32_t t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = fp16_terms(p[j]);
            fp16_operands(t, pa[0], pa[1]);
        }
        auto column = [&](int c, int w) __attribute__((always_inline)) {
            tq_u4 bt;
#pragma unroll
            for (int d = 0; d < 4; ++d) bt[d] = __builtin_amdgcn_perm(v[2 * d + 1][w], v[2 * d][w], (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int t = 0; t < PT; ++t) acc[c] = BF ? mfma16_bf16(pa[t], bt, acc[c]) : mfma16_f16(pa[t], bt, acc[c]);
        };
        if constexpr (HELD) {
            tame(lane, wild);
#pragma unroll
            for (int c = 0; c < NC; ++c) column(c, c / 2);
        } else {
#pragma unroll
            for (int c0 = 0; c0 < NC; c0 += 8) {
                load_columns<8>(lane, c0, 0);
                tame(lane, wild);
#pragma unroll
                for (int c = 0; c < 8; ++c) column(c0 + c, c / 2);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
};

// Bound by reading (64 x 16384 tokens x 8 heads of 128, 4- and 2-bit codes: 839 MB in 186 us, 4.5 TB/s; 32 x 16384 x 8 of 256: 198 us), in short rows by an item's start and end (128 x 2048: 79 us, and 86 with a way back for every item by itself), where one
// block a compute unit has nothing to overlap them with.
// A block takes items of the plan in turn, each a share of what the queries of a (sequence, kv head) see; the tables stay in LDS.  Up to 16 / C query vectors are the columns of 16 x 16 x 32 products, C times over, so that C blocks of 16 tokens share a softmax: every block's
// scores are made for all columns, a lane keeps those of its own column's block, and the weights of the others are zeros in its column of the value product (as in tq_decode_kernel, whose
// loop this is, with runs found through the sequence's pages: a run lies within a page, whose number is fetched a run ahead).  QT: fp16 terms of a rotated query, one for bfloat16 (two then, and two of the levels, for float16: with one the result of half a unit's
// rounding, 2.1e-4, came out at 6e-4.  Weights, their products with norms and value levels keep one: 3.0e-4; second ones would be two more value products and tables of two words).
// Base-2 logits are rounded before the reference is taken off, so that the largest ones stay exact against it however large they are.
template <int D, int IPBK, int IPBV, int C, bool BF>
__global__ __launch_bounds__(DTHREADS, DW / 4) void tq_paged_few_kernel(TqPagedArgs a) {
    constexpr int QT = BF ? 1 : 2;
    constexpr int QREG = D == 256 && (IPBK == 1 || IPBV == 1) ? 1 : QT;
    constexpr int PART = D + 2, TILES = D / 32, SK = D / 32, NC = D / 16, KB = D / 4 / IPBK, NWK = (KB + 3) / 4, GBV = D / IPBV;
    constexpr int RUN = decode_run(D, IPBK, IPBV), SUB = RUN / 32, HEADS = 16 / C, UNIT = C == 4 ? 64 : 32, SPL = C == 1 ? 8 : 4;
    static_assert(UNIT <= RUN, "a round of softmax lies within a run");
    constexpr int VPB = GBV % 16 ? 8 : 16, VBYTES = RUN * GBV, VPIECES = VBYTES / VPB, NVP = (VPIECES + 63) / 64;
    constexpr float SLACK = 8.f;
    constexpr int P_SHIFT = 14 - 8;
    constexpr int HR = D == 256 && C == 1 ? 4 : HEADS < 8 ? HEADS : 8;            // columns a round of the join
    constexpr int QROW = D + 4;
    // LDS: tables; values of each wave, rotated queries; the waves' sums of packed tokens and of plain ones, and the joined ones.  Where that is more than there is, the waves' sums lie over values and
    // queries, take turns, and cost barriers.
    constexpr uint32_t V_AT = 65536u, Q_AT = V_AT + DW * VBYTES, LOOP_END = Q_AT + 16u * QROW * 4u, JOIN = DW * HR * PART * 4u;
    constexpr bool SIDE = HR >= HEADS && LOOP_END + 2u * JOIN + 2u * 16u * QROW * 4u + 4u * 16u * 4u + DW * RUN * 6u + (QT > QREG ? (QT - QREG) * SK * 1024u : 0u) + 1280u <= 163840u;
    constexpr uint32_t COLS = SIDE ? 16u : HEADS, SUMS = COLS * QROW * 4u, STATS = 4u * COLS * 4u;          // columns that joined sums are held of
    constexpr uint32_t JOIN_AT = SIDE ? LOOP_END : V_AT, SUMS_AT = JOIN_AT + (SIDE ? 2u : 1u) * JOIN, STATS_AT = SUMS_AT + 2u * SUMS, JOIN_END = STATS_AT + STATS;
    constexpr uint32_t AREA = LOOP_END > JOIN_END ? LOOP_END : JOIN_END;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[AREA];
    __shared__ __attribute__((aligned(16))) float lds_kn[DW][RUN];
    __shared__ __attribute__((aligned(16))) uint16_t lds_vn[DW][RUN];      // value norms / 2^ev_ref
    __shared__ __attribute__((aligned(16))) tq_u4 lds_q[QT > QREG ? (QT - QREG) * SK : 1][TQ_WAVE];
    __shared__ __attribute__((aligned(16))) float lds_corr[DW][16];
    __shared__ uint32_t lds_trips[DW];
    __shared__ float lds_wild[DW];
    __shared__ uint32_t lds_item[C][4];              // of the items whose sums are held: first query token, kv head, query vectors, record

    {
        const uint32_t tid = threadIdx.x;
        std::conditional_t<BF, Lut<IPBK>, Lut2<IPBK>> table_k;
        Lut<IPBV> table_v;
        if constexpr (BF) table_k.load(a.table_k + TQ_OFF_LUT(D), tid);
        else table_k.load(a.table_k, a.bits_k, D, tid);
        table_v.load(a.table_v + TQ_OFF_LUT(D), tid);
        table_k.store(lds, tid);
        table_v.store(lds + 128, tid);
        if (tid < (uint32_t)DW) lds_trips[tid] = 0u;
    }
    const int32_t first_item = a.blocks[blockIdx.x], end_item = a.blocks[blockIdx.x + 1];
    uint32_t trips = 0u;
    bool turned = false;                     // whether any of the items whose sums are held has packed tokens
#pragma unroll 1
    for (int32_t index = first_item; index < end_item; ++index) {
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));        // (what lanes make of their number is made anew for every item: kept from one to the next it took a hundred registers that there are not)
    const uint32_t lane = tid & 63u, wave = tq_uniform32(tid >> 6), n16 = lane & 15u, q4 = lane >> 4, head = n16 % HEADS, cls = n16 / HEADS;
    const bool shaped = a.cap != 0.f || a.slopes;
    const Cap cap(a);
    const int32_t *it = a.items + (size_t)index * PAGED_ITEM;
    const int32_t *sq = a.seqs + (size_t)it[0] * PAGED_SEQ;
    const uint32_t t_begin = (uint32_t)it[2], t_end = (uint32_t)it[3], plain_from = (uint32_t)it[4], plain_to = (uint32_t)it[5];
    const int record = it[6];
    PagedRow row;
    row.fresh = (uint32_t)sq[1]; row.total = (uint32_t)sq[2]; row.packed = (uint32_t)sq[3];
    row.pages = a.tables + sq[4]; row.plain_pages = a.tables + sq[5];
    row.kv = (uint32_t)it[7];
    const uint32_t q_first = (uint32_t)sq[0], M = row.fresh * a.group;
    const uint8_t *queries = a.q + ((long long)q_first * a.q_token + (long long)(row.kv * a.group) * a.q_head) * 2;
    const bool live = head < M;
    const uint32_t vector = min(head, M - 1u), token = vector / a.group, pos = row.total - row.fresh + token;        // of this lane's column
    const float slope = a.slopes ? a.slopes[row.kv * a.group + (vector - token * a.group)] * LOG2E : 0.f;
    // [packed, plain][COLS][QROW]; [largest, total of packed, of plain][COLS]: HEADS columns an item, of as many items as there is a way back for at a time (SIDE)
    const uint32_t slot = SIDE ? (uint32_t)((index - first_item) % C) : 0u;
    float *const sums = reinterpret_cast<float *>(lds + SUMS_AT) + slot * (HEADS * QROW), *const stats = reinterpret_cast<float *>(lds + STATS_AT) + slot * HEADS;

    // The waves' sums meet in LDS, HR columns from h0 on (which: 0 packed, 1 plain).  put(): unit: what this wave's value sums are multiplied by, l: all lanes' of a column
    auto put = [&](uint32_t which, uint32_t h0, float m_ref, float l, float unit, const tq_f4v (&acc)[NC]) __attribute__((always_inline)) {
        float *const mine = reinterpret_cast<float *>(lds + JOIN_AT + (SIDE ? which * JOIN : 0u)) + wave * (HR * PART);
        if (q4 == 0u && n16 < (uint32_t)HEADS && n16 >= h0 && n16 < h0 + HR) {
            mine[(n16 - h0) * PART] = m_ref;
            mine[(n16 - h0) * PART + 1u] = l;
        }
        if (C == 1 || which) {
            if (4u * q4 >= h0 && 4u * q4 < min(h0 + HR, (uint32_t)HEADS)) {
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mine[(4u * q4 + r - h0) * PART + 2u + value_coord<D>(n16, c)] = acc[c][r] * unit;
            }
        } else {
            // The blocks of tokens lie in lanes 32 apart (C = 4: and 16 apart): two registers exchange halves and are added, which leaves the sum of one in each half (then quarters).
            static_assert(C == 1 || HR >= HEADS, "one round");
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float half[NC / 2];
#pragma unroll
                for (int c = 0; c < NC; c += 2) half[c / 2] = fold<32>(acc[c][r], acc[c + 1][r]);
                if constexpr (C == 2) {
#pragma unroll
                    for (int c = 0; c < NC; c += 2) mine[(4u * (q4 & 1u) + r) * PART + 2u + value_coord<D>(n16, c + (int)(q4 >> 1))] = half[c / 2] * unit;
                } else {
#pragma unroll
                    for (int c = 0; c < NC; c += 4) {
                        const bool pair = c + 2 < NC;     // (96: the last two columns stand alone, both quarters hold them)
                        const float sum = fold<16>(half[c / 2], half[pair ? c / 2 + 1 : c / 2]);
                        mine[r * PART + 2u + value_coord<D>(n16, c + (int)((pair ? 2u * (q4 & 1u) : 0u) + (q4 >> 1)))] = sum * unit;
                    }
                }
            }
        }
    };
    // of the first `waves` (none: zeros)
    auto combine = [&](uint32_t which, uint32_t h0, uint32_t waves) __attribute__((always_inline)) {
        const float *all = reinterpret_cast<const float *>(lds + JOIN_AT + (SIDE ? which * JOIN : 0u));
        for (uint32_t i = tid; i < min((uint32_t)HR, M - h0) * D; i += DTHREADS) {
            const uint32_t col = i / D, d = i - col * D;
            float m = MANY_NONE, sum = 0.f, total = 0.f;
#pragma unroll
            for (uint32_t w = 0; w < DW; ++w) m = w < waves ? fmaxf(m, all[(w * HR + col) * PART]) : m;
#pragma unroll
            for (uint32_t w = 0; w < DW; ++w) {
                if (w >= waves) continue;
                const float own = all[(w * HR + col) * PART], lw = all[(w * HR + col) * PART + 1u];
                const float f = own != MANY_NONE ? __builtin_amdgcn_exp2f(own - m) : lw == 0.f ? 0.f : __builtin_nanf("");
                sum = fmaf(all[(w * HR + col) * PART + 2u + d], f, sum);
                total = fmaf(lw, f, total);
            }
            sums[which * (SUMS / 4u) + (h0 + col) * QROW + d] = sum;
            if (d == 0u) {
                stats[(2u * which) * COLS + h0 + col] = m;
                stats[(2u * which + 1u) * COLS + h0 + col] = total;
            }
        }
    };
    // where there is no room for both sides
    auto join = [&](uint32_t which, float m_ref, float l, float unit, const tq_f4v (&acc)[NC]) __attribute__((always_inline)) {
        for (uint32_t h0 = 0; h0 < (uint32_t)HEADS && h0 < M; h0 += HR) {
            __syncthreads();         // (values, queries, and the round before)
            put(which, h0, m_ref, l, unit, acc);
            __syncthreads();
            combine(which, h0, DW);
        }
    };
    // Queries into the codec's space, of as many items as the columns hold (SIDE: what lies there has been read before the barrier that stood last; else the sums have been written over it)
    if (!SIDE || (index - first_item) % C == 0) {
        if (!SIDE) __syncthreads();
        if (wave < (uint32_t)TILES) {
            const int32_t *mine = a.items + (size_t)min(index + (int32_t)cls, end_item - 1) * PAGED_ITEM, *of = a.seqs + (size_t)mine[0] * PAGED_SEQ;
            const uint32_t m = min(head, (uint32_t)of[1] * a.group - 1u), t = m / a.group;
            Rotation<D, BF> r;
            r.qsrc = a.q + ((long long)((uint32_t)of[0] + t) * a.q_token + (long long)((uint32_t)mine[7] * a.group + (m - t * a.group)) * a.q_head) * 2 + 16u * q4;
            r.asrc = a.table_k + (BF ? TQ_OFF_A_BF16(D) : TQ_OFF_A_F16) + ((size_t)wave * (D / 16 * 64u) + q4 * 32u + n16) * 16u;
            r.fetch(0);
            r.finish(reinterpret_cast<float *>(lds + Q_AT), QROW, a.scale, wave, lane);
        }
        __syncthreads();
    }
    const uint32_t q_row = slot * HEADS + head;

    if (t_end > t_begin) {
        const uint32_t lo = a.window && pos >= a.window ? pos - a.window + 1u : 0u;              // first token that this lane's column sees
        const uint32_t last_pos = row.total - 1u, whole_from = a.window && last_pos >= a.window ? last_pos - a.window + 1u : 0u;
        uint8_t *vcodes = lds + V_AT + wave * VBYTES;
        // Runs of a wave: in every whole round of the block one of RUN tokens; what is left of the block's tokens is dealt out evenly, in blocks of 16, 32 or 64 tokens (which lie within a
        // page), so that no wave works on a whole run alone at the end.
        const uint32_t rounds = (t_end - t_begin) / (RUN * DW), rest0 = t_begin + rounds * (RUN * DW), rest = t_end - rest0;
        const uint32_t share = rest > 32u * DW ? 64u : rest > 16u * DW ? 32u : 16u;
        const uint32_t tail0 = min(t_end, rest0 + wave * share), n_tail = min(t_end, tail0 + share) - tail0;
        auto run_start = [&](uint32_t i) { return i < rounds ? t_begin + (i * DW + wave) * RUN : tail0; };
        auto run_tokens = [&](uint32_t i) { return i < rounds ? (uint32_t)RUN : i == rounds ? n_tail : 0u; };
        const uint32_t place_mask = (1u << a.shift) - 1u;
        // where a run lies: its page and its place there (a run that there is not: the block's first token, which is)
        struct Where { int page; uint32_t place; };
        auto where = [&](uint32_t i) {
            const uint32_t t = run_tokens(i) ? run_start(i) : t_begin;
            return Where{(int)tq_uniform32((uint32_t)row.pages[t >> a.shift]), (row.kv << a.shift) + (t & place_mask)};
        };
        uint32_t kraw[SUB][2][NWK];
        tq_u4 vpiece[NVP];
        uint16_t kn_raw, vn_raw;
        // n_tok >= 1: what lies past the last token is read as that token.  (One form for whole and partial runs, see tq_decode_kernel.)
        auto issue_keys = [&](Where w, uint32_t n_tok) __attribute__((always_inline)) {
            const uint8_t *base = a.pool + (long long)w.page * a.page_stride + (size_t)w.place * (4 * KB);
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint32_t tl = 32u * u + 16u * b + n16;
                    const uint8_t *src = base + min(tl, n_tok - 1u) * (4 * KB) + q4 * KB;
                    if constexpr (KB % 16 == 0) {
#pragma unroll
                        for (int p = 0; p < KB / 16; ++p) {
                            const tq_u4 v = tq_gload16(src + 16 * p);
#pragma unroll
                            for (int i = 0; i < 4; ++i) kraw[u][b][4 * p + i] = v[i];
                        }
                    } else if constexpr (KB % 8 == 0) {
#pragma unroll
                        for (int p = 0; p < KB / 8; ++p) {
                            const tq_u2 v = tq_gload8(src + 8 * p);
                            kraw[u][b][2 * p] = v[0]; kraw[u][b][2 * p + 1] = v[1];
                        }
                    } else if constexpr (KB % 4 == 0) {
#pragma unroll
                        for (int p = 0; p < KB / 4; ++p) kraw[u][b][p] = tq_gload4(src + 4 * p);
                    } else {
                        static_assert(KB % 2 == 0, "key bytes of a lane");
                        uint32_t h[KB / 2];
#pragma unroll
                        for (int p = 0; p < KB / 2; ++p) h[p] = tq_gload2(reinterpret_cast<const uint16_t *>(src) + p);
#pragma unroll
                        for (int p = 0; p < NWK; ++p) kraw[u][b][p] = h[2 * p] | (2 * p + 1 < KB / 2 ? h[2 * p + 1 < KB / 2 ? 2 * p + 1 : 0] << 16 : 0u);
                    }
                }
        };
        auto issue_values = [&](Where w, uint32_t n_tok) __attribute__((always_inline)) {
            const uint8_t *base = a.pool + (long long)w.page * a.page_stride, *vsrc = base + a.v_idx + (size_t)w.place * GBV;
#pragma unroll
            for (int p = 0; p < NVP; ++p) {
                const uint32_t piece = min(p * 64u + lane, min((uint32_t)VPIECES, n_tok * (GBV / VPB)) - 1u);
                if constexpr (VPB == 16) vpiece[p] = tq_gload16(vsrc + piece * 16u);
                else { const tq_u2 v = tq_gload8(vsrc + piece * 8u); vpiece[p][0] = v[0]; vpiece[p][1] = v[1]; }
            }
            const uint32_t own = w.place + min(lane, n_tok - 1u);
            kn_raw = tq_gload2(reinterpret_cast<const uint16_t *>(base + a.k_norms) + own);
            vn_raw = tq_gload2(reinterpret_cast<const uint16_t *>(base + a.v_norms) + own);
        };
        // ---- start: the first run's loads
        Where now = where(0u), next = where(1u);
        issue_keys(now, max(run_tokens(0u), 1u));
        issue_values(now, max(run_tokens(0u), 1u));
        __builtin_amdgcn_sched_barrier(0);

        // ---- B operand of the score product: fp16 of q * 2^(10 - e), e = binary exponent of the column's largest magnitude
        tq_u4 qb[QREG][SK];
        float c1;                // base-2 logit = accumulator * key norm * c1
        {
            const float *q = reinterpret_cast<const float *>(lds + Q_AT) + q_row * QROW + (D / 4) * q4;
            float x[D / 4];
#pragma unroll
            for (int i = 0; i < D / 4; i += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(q + i);
                x[i] = f.x; x[i + 1] = f.y; x[i + 2] = f.z; x[i + 3] = f.w;
            }
            float big = 0.f;
#pragma unroll
            for (int i = 0; i < D / 4; ++i) big = fmaxf(big, fabsf(x[i]));
            big = reduce_rows(big, OpMax());
            int e = 0;
            if (big > 0.f && big < __builtin_inff()) (void)frexpf(big, &e);
            e = e < -100 ? -100 : e;
            const float up = ldexpf(1.f, TQ_F16_PI_SHIFT - e);
            c1 = live ? ldexpf(LOG2E, e - TQ_F16_PI_SHIFT - (BF ? 0 : LEVEL_SHIFT)) : 0.f;
#pragma unroll
            for (int s = 0; s < SK; ++s) {
                tq_half8 term[QT];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float y = live ? x[8 * s + i] * up : 0.f;
#pragma unroll
                    for (int k = 0; k < QT; ++k) {
                        term[k][i] = (_Float16)y;
                        y -= (float)term[k][i];
                    }
                }
#pragma unroll
                for (int k = 0; k < QREG; ++k) qb[k][s] = __builtin_bit_cast(tq_u4, term[k]);
#pragma unroll
                for (int k = QREG; k < QT; ++k) lds_q[(k - QREG) * SK + s][lane] = __builtin_bit_cast(tq_u4, term[k]);     // (the same in every wave, and each writes it)
            }
        }
        const uint32_t slot_k = BF ? RepLut<IPBK>::lane_offset(lane) : Lut2<IPBK>::lane_offset(lane), slot_v = 128u + RepLut<IPBV>::lane_offset(lane);
        tq_f4v acc[NC];          // register r = column 4 q4 + r, c = coordinate value_coord(n16, c)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c] = tq_f4v{0.f, 0.f, 0.f, 0.f};
        float m_ref = MANY_NONE, l_run = 0.f;
        int ev_ref = -100;       // largest binary exponent of a value norm this wave has seen; the sums are in units of 2^ev_ref

        // one run of staged tokens from t0 on; FULL: all of them exist and every column sees them
        auto run = [&](auto full_tag, uint32_t t0, uint32_t n_tok, Where after, uint32_t n_after) __attribute__((always_inline)) {
            constexpr bool FULL = decltype(full_tag)::value;
            tq_f4v sc[SUB][2];   // register r of block b = token 32 u + 16 b + 4 q4 + r
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                sc[u][0] = sc[u][1] = tq_f4v{0.f, 0.f, 0.f, 0.f};
                if (!FULL && 32u * u >= n_tok) continue;       // uniform
                auto step = [&](int b, int s, const tq_u4 (&q)[QT]) __attribute__((always_inline)) {
                    if constexpr (BF) sc[u][b] = mfma16_f16(decode_keys<IPBK, NWK>(kraw[u][b], s, lds, slot_k), q[0], sc[u][b]);
                    else {
                        tq_u4 hi, lo;
                        decode_keys2<IPBK, NWK>(kraw[u][b], s, lds, slot_k, hi, lo);
                        sc[u][b] = mfma16_f16(hi, q[0], sc[u][b]);
                        sc[u][b] = mfma16_f16(hi, q[QT - 1], sc[u][b]);
                        sc[u][b] = mfma16_f16(lo, q[0], sc[u][b]);
                    }
                };
                auto terms = [&](int s, tq_u4 (&q)[QT]) __attribute__((always_inline)) {
#pragma unroll
                    for (int k = 0; k < QT; ++k) q[k] = k < QREG ? qb[k < QREG ? k : 0][s] : lds_q[(k - QREG) * SK + s][lane];
                };
                tq_u4 q[QT];
                if constexpr (QREG == QT) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int s = 0; s < SK; ++s) { terms(s, q); step(b, s, q); }
                } else {         // a term from LDS serves both blocks
#pragma unroll
                    for (int s = 0; s < SK; ++s) {
                        terms(s, q);
                        step(0, s, q);
                        step(1, s, q);
                        if (s % 2 == 1) __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            issue_keys(after, n_after);
#pragma unroll
            for (int u = 0; u < RUN / UNIT; ++u) {
                if (!FULL && (uint32_t)(UNIT * u) >= n_tok) break;  // uniform
                // tokens of this lane: tok .. tok + 3 (C = 1: and tok + 16 .. tok + 19)
                const uint32_t tok = (uint32_t)(UNIT * u) + 16u * cls + 4u * q4;
                float z[SPL];
#pragma unroll
                for (int b = 0; b < SPL / 4; ++b) {
                    tq_f4v own = sc[(UNIT / 32) * u][b];
                    if constexpr (C > 1) {
#pragma unroll
                        for (int k = 1; k < C; ++k) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) own[r] = cls == (uint32_t)k ? sc[(UNIT / 32) * u + k / 2][k % 2][r] : own[r];
                        }
                    }
                    const float4 k4 = *reinterpret_cast<const float4 *>(&lds_kn[wave][tok + 16u * b]);
                    z[4 * b + 0] = own[0] * k4.x * c1; z[4 * b + 1] = own[1] * k4.y * c1;
                    z[4 * b + 2] = own[2] * k4.z * c1; z[4 * b + 3] = own[3] * k4.w * c1;
                }
#pragma unroll
                for (int j = 0; j < SPL; ++j) asm volatile("" : "+v"(z[j]));        // (rounded here, not fused with what is taken off)
                if (shaped) {
                    if (a.cap != 0.f) {
                        cap.template all<false>(z, SPL);
                    }
                    const float first = (float)((int)(t0 + tok) - (int)pos);
#pragma unroll
                    for (int j = 0; j < SPL; ++j) z[j] = fmaf(slope, first + (float)(16 * (j / 4) + j % 4), z[j]);
                }
                auto gone = [&](int j) { const uint32_t i = tok + 16u * (j / 4) + (j % 4); return i >= n_tok || t0 + i < lo; };
                if constexpr (!FULL) {
#pragma unroll
                    for (int j = 0; j < SPL; ++j)
                        if (gone(j)) z[j] = MANY_NONE;
                }
                float zmax = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
                if constexpr (SPL == 8) zmax = fmaxf(zmax, fmaxf(fmaxf(z[SPL - 4], z[SPL - 3]), fmaxf(z[SPL - 2], z[SPL - 1])));
                if (__any(zmax > m_ref + SLACK)) {     // (rare after the first tiles) move the column's reference, rescale its sums
                    float zm = zmax;
#pragma unroll
                    for (int d = HEADS; d < 64; d <<= 1) zm = fmaxf(zm, __shfl_xor(zm, d));
                    const float m_new = fmaxf(m_ref, zm);
                    const float corr = __builtin_amdgcn_exp2f(m_ref - m_new);
                    l_run *= corr;
                    m_ref = m_new;
                    if (q4 == 0u) lds_corr[wave][n16] = corr;
                    asm volatile("" ::: "memory");
                    __builtin_amdgcn_wave_barrier();
                    const float4 c4 = *reinterpret_cast<const float4 *>(&lds_corr[wave][4u * q4]);
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        acc[c][0] *= c4.x; acc[c][1] *= c4.y; acc[c][2] *= c4.z; acc[c][3] *= c4.w;
                    }
                }
                const float bias = (float)P_SHIFT - m_ref;
                float ps[SPL];
                float lsum = 0.f;
#pragma unroll
                for (int j = 0; j < SPL; ++j) {
                    ps[j] = __builtin_amdgcn_exp2f(z[j] + bias);     // p * 2^P_SHIFT, p <= 2^8
                    if constexpr (!FULL) {   // (where nothing has been seen yet the reference is no larger than what stands for hidden tokens)
                        if (gone(j)) ps[j] = 0.f;
                    }
                    lsum += ps[j];
                }
                l_run += lsum;
                // ---- weights p_j |v_j| / 2^ev_ref of the lane's own tokens, in pairs
                uint32_t w[SPL / 2];
#pragma unroll
                for (int b = 0; b < SPL / 4; ++b) {
                    const tq_u2 nrm = *reinterpret_cast<const tq_u2 *>(&lds_vn[wave][tok + 16u * b]);
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        const tq_half2 two = tq_half2{(_Float16)ps[4 * b + 2 * d], (_Float16)ps[4 * b + 2 * d + 1]} * __builtin_bit_cast(tq_half2, (uint32_t)nrm[d]);
                        w[2 * b + d] = __builtin_bit_cast(uint32_t, two);
                    }
                }
#pragma unroll
                for (int tile = 0; tile < UNIT / 32; ++tile) {
                    if (!FULL && (uint32_t)(UNIT * u + 32 * tile) >= n_tok) break;  // uniform
                    // slice j of lane (., q4) = token tok_a + j (j < 4), tok_b + j - 4; a column holds the weights of its own block of tokens
                    const uint32_t tok_a = (uint32_t)(UNIT * u + 32 * tile) + 4u * q4, tok_b = tok_a + 16u;
                    tq_u4 pa;
#pragma unroll
                    for (int d = 0; d < 4; ++d) pa[d] = C == 1 ? w[d % (SPL / 2)] : (cls == (uint32_t)(2 * tile + d / 2) ? w[d % 2] : 0u);
                    auto columns = [&](auto n_tag, int c0) __attribute__((always_inline)) {
                        constexpr int N = decltype(n_tag)::value;
                        uint32_t dec[8][N / 2];      // per token: N coordinates of the lane as fp16
                        const uint32_t first = value_coord<D>(n16, c0);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            decode_values<IPBV, N>(vcodes + ((j < 4 ? tok_a : tok_b) + (uint32_t)(j % 4)) * GBV, first, lds, slot_v, dec[j]);
#pragma unroll
                        for (int c = 0; c < N; ++c) {
                            tq_u4 bt;
#pragma unroll
                            for (int d = 0; d < 4; ++d) bt[d] = __builtin_amdgcn_perm(dec[2 * d + 1][c / 2], dec[2 * d][c / 2], (c & 1) ? 0x07060302u : 0x05040100u);
                            acc[c0 + c] = mfma16_f16(pa, bt, acc[c0 + c]);
                        }
                    };
                    if constexpr (D == 64) columns(std::integral_constant<int, 4>{}, 0);
                    else if constexpr (D == 96) { columns(std::integral_constant<int, 4>{}, 0); columns(std::integral_constant<int, 2>{}, 4); }
                    else if constexpr (D == 128) columns(std::integral_constant<int, 8>{}, 0);
                    else { columns(std::integral_constant<int, 8>{}, 0); __builtin_amdgcn_sched_barrier(0); columns(std::integral_constant<int, 8>{}, 8); }
                }
            }
        };
        // one trip: stage the run that has been loaded, start the loads of the next one, compute.  The two waves of a SIMD are kept level (see tq_decode_kernel).
        auto trip = [&](auto full_tag, uint32_t i) __attribute__((always_inline)) {
            ++trips;
            volatile __attribute__((address_space(3))) uint32_t *begun = (__attribute__((address_space(3))) uint32_t *)lds_trips;
            if (lane == 0u) begun[wave] = trips;
            if (trips > tq_uniform32(begun[wave ^ 4u])) __builtin_amdgcn_s_setprio(0); else __builtin_amdgcn_s_setprio(1);
            constexpr bool FULL = decltype(full_tag)::value;
            const uint32_t n_tok = run_tokens(i), t0 = run_start(i);
#pragma unroll
            for (int p = 0; p < NVP; ++p) {
                const uint32_t piece = p * 64u + lane;
                if (VPIECES % 64 == 0 || piece < VPIECES) {
                    if constexpr (VPB == 16) *reinterpret_cast<tq_u4 *>(vcodes + piece * 16u) = vpiece[p];
                    else *reinterpret_cast<tq_u2 *>(vcodes + piece * 8u) = tq_u2{vpiece[p][0], vpiece[p][1]};
                }
            }
            {
                // Where not all columns need see a token, an infinite norm of its values times a weight of 0 would make NaN of those that do not: it is zero there, and the keys' norm NaN (see
                // tq_paged_kernel)
                const bool wild = !FULL && (vn_raw & 0x7c00u) == 0x7c00u;
                const _Float16 kh = __builtin_bit_cast(_Float16, wild ? (uint16_t)0x7e00u : kn_raw);
                if (RUN == 64 || lane < (uint32_t)RUN) lds_kn[wave][lane] = (float)kh;     // one token per lane
                // does a value norm of this run exceed the reference exponent?  (a vote; a handful of times per wave)
                const uint16_t vn = lane < n_tok && !wild ? vn_raw : (uint16_t)0;   // tokens past the end weigh nothing
                uint32_t e = ((uint32_t)vn >> 10) & 31u;
                if (__any((int)max(e, 1u) - 15 > ev_ref)) {
                    e = max(e, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)e, 0x111, 0xf, 0xf, true));
                    e = max(e, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)e, 0x112, 0xf, 0xf, true));
                    e = max(e, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)e, 0x114, 0xf, 0xf, true));
                    e = max(e, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)e, 0x118, 0xf, 0xf, true));
                    const uint32_t emax = max(max((uint32_t)__builtin_amdgcn_readlane((int)e, 15), (uint32_t)__builtin_amdgcn_readlane((int)e, 31)),
                                              max((uint32_t)__builtin_amdgcn_readlane((int)e, 47), (uint32_t)__builtin_amdgcn_readlane((int)e, 63)));
                    const int ev = (int)max(emax, 1u) - 15;
                    const float f = ldexpf(1.f, ev_ref - ev);
#pragma unroll
                    for (int c = 0; c < NC; ++c) acc[c] *= f;
                    ev_ref = ev;
                }
                const float vs = ldexpf((float)__builtin_bit_cast(_Float16, vn), -ev_ref);
                if (RUN == 64 || lane < (uint32_t)RUN) lds_vn[wave][lane] = __builtin_bit_cast(uint16_t, (_Float16)vs);
            }
            const uint32_t n_after = max(run_tokens(i + 1u), 1u);
            const Where after = next;
            next = where(i + 2u);
            issue_values(after, n_after);
            asm volatile("" ::: "memory");    // staged with one access width, read back with others (LDS serves a wave in order)
            __builtin_amdgcn_wave_barrier();
            run(full_tag, t0, n_tok, after, n_after);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_wave_barrier();
        };
        {
            // Whole runs in a loop of their own; those that the window's edge crosses and the partial one (a wave has one at most) by the careful form.
            uint32_t i = 0u;
#pragma unroll 1
            while (run_tokens(i) && run_start(i) < whole_from) trip(std::false_type{}, i++);
#pragma unroll 1
            while (run_tokens(i) == (uint32_t)RUN) trip(std::true_type{}, i++);
            if (run_tokens(i)) trip(std::false_type{}, i);
            if (lane == 0u) *(volatile __attribute__((address_space(3))) uint32_t *)&lds_trips[wave] = 0xffffffffu;
            __builtin_amdgcn_s_setprio(0);
        }
        float l_all = l_run;
#pragma unroll
        for (int d = HEADS; d < 64; d <<= 1) l_all += __shfl_xor(l_all, d);
        l_all *= 1.0f / (float)(1 << P_SHIFT);
        const float unit = ldexpf(1.f, ev_ref - P_SHIFT);
        if constexpr (SIDE) put(0u, 0u, m_ref, l_all, unit, acc);
        else join(0u, m_ref, l_all, unit, acc);
    }
    const bool packed = t_end > t_begin, plain = plain_to > plain_from;
    if (plain) {
        // ---- uncompressed tokens: a wave takes 32 at a time, columns as they are (not C times over)
        const uint32_t runs = (plain_to - plain_from + 31u) / 32u, col = min(n16, M - 1u), ct = col / a.group, cpos = row.total - row.fresh + ct;
        const float cslope = a.slopes ? a.slopes[row.kv * a.group + (col - ct * a.group)] * LOG2E : 0.f;
        const uint8_t *cq = queries + ((long long)ct * a.q_token + (long long)(col - ct * a.group) * a.q_head) * 2;
        tq_f4v acc[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c] = tq_f4v{0.f, 0.f, 0.f, 0.f};
        float m_ref = MANY_NONE, l = 0.f;
        bool wild = false;
#pragma unroll 1
        for (uint32_t w = DW - 1u - wave; w < runs; w += DW) {
            const uint32_t t0 = plain_from + 32u * w;
            const uint8_t *page = a.plain + (long long)(int)tq_uniform32((uint32_t)row.plain_pages[t0 >> a.shift]) * a.plain_stride + (size_t)((row.kv << a.shift) + (t0 & ((1u << a.shift) - 1u))) * (2u * D);
            FewPlain<D, BF> t;
            t.load(page, page + a.plain_v, min(32u, plain_to - t0), lane);
            float x[8];
            t.scores(cq + 16u * q4, x);
            const uint32_t at = row.packed + t0, gone = unseen_bits(at, cpos, a.window);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= a.scale * LOG2E;
            if (a.cap != 0.f) {
                cap.template all<false>(x, 8);
            }
            float top = m_ref;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t i = FewPlain<D, BF>::token(j, q4);
                x[j] = fmaf(cslope, (float)((int)(at + i) - (int)cpos), x[j]);
                x[j] = i < t.valid && !((gone >> i) & 1u) ? x[j] : MANY_NONE;
                top = fmaxf(top, x[j]);
            }
            top = reduce_rows(top, OpMax());
            const float shrink = __builtin_amdgcn_exp2f(m_ref - top);
            m_ref = top;
            l *= shrink;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = x[j] == MANY_NONE ? 0.f : __builtin_amdgcn_exp2f(x[j] - top);
                l += x[j];               // (this lane's tokens)
            }
            if (w >= DW) {             // (sums so far: a lane has those of columns 4 q4 ...)
                float4 c4;
#pragma unroll
                for (int r = 0; r < 4; ++r) (&c4.x)[r] = __shfl(shrink, (int)(4u * q4 + r));
#pragma unroll
                for (int c = 0; c < NC; ++c) { acc[c][0] *= c4.x; acc[c][1] *= c4.y; acc[c][2] *= c4.z; acc[c][3] *= c4.w; }
            }
            t.values(x, lane, wild, acc);
        }
        l = reduce_rows(l, OpAdd());
        wild = __any(wild);
        if (lane == 0u) lds_wild[wave] = wild ? 1.f : 0.f;
        if constexpr (SIDE) put(1u, 0u, m_ref, l, 1.f, acc);
        else join(1u, m_ref, l, 1.f, acc);
    }
    __syncthreads();
    turned = packed || (slot && turned);
    if constexpr (SIDE) {
        combine(0u, 0u, packed ? DW : 0u);
        combine(1u, 0u, plain ? DW : 0u);
    } else {
        for (uint32_t h0 = 0; h0 < (uint32_t)HEADS && h0 < M; h0 += HR) {
            if (!packed) combine(0u, h0, 0u);
            if (!plain) combine(1u, h0, 0u);
        }
    }
    if (tid == 0u) {
        lds_item[slot][0] = q_first; lds_item[slot][1] = row.kv; lds_item[slot][2] = M; lds_item[slot][3] = (uint32_t)record;
    }
    if (plain) {
        float any = 0.f;
#pragma unroll
        for (int w = 0; w < DW; ++w) any += lds_wild[w];
        if (any != 0.f) {
            __syncthreads();
            paged_wild<D>(a, row, sums + SUMS / 4u, 0u, plain_from, plain_to, tid);
        }
    }
    __syncthreads();
    // The way back, of up to C items at a time (9000 cycles of four waves, whose operands come from memory)
    if (wave < (uint32_t)TILES && (!SIDE || slot == C - 1u || index + 1 == end_item)) {
        // (32 columns to an instruction: the sixteen twice)
        const uint32_t col = lane % COLS, its = col / HEADS, vec = col % HEADS;
        const float *const s0 = sums - slot * (HEADS * QROW) + col * QROW, *const t0 = stats - slot * HEADS + col;
        const JoinedColumn j{turned ? s0 : nullptr, s0 + SUMS / 4u, t0[0], t0[COLS], t0[2u * COLS], t0[3u * COLS]};
        const bool some = (lane & 31u) < COLS && its <= slot && vec < lds_item[its][2];
        const int to = (int)lds_item[its][3];
        TQ_GLOBAL float *rec = to < 0 ? nullptr : (TQ_GLOBAL float *)a.rec + (size_t)to * a.qt * paged_record(a.cols, D);
        paged_finish<D>(a, j, lds_item[its][1], lds_item[its][0], rec, vec, vec, some, wave, lane);
    }
    }
}

template <int D, int IPBK, int IPBV>
int launch_paged_few(dim3 grid, hipStream_t s, const TqPagedArgs &a, uint32_t vectors) {
    constexpr int C = decode_run(D, IPBK, IPBV) == 64 ? 4 : 2;
    const dim3 t(DTHREADS);
    if (a.dtype == TQ_BF16) {
        if (vectors <= 16u / C) hipLaunchKernelGGL((tq_paged_few_kernel<D, IPBK, IPBV, C, true>), grid, t, 0, s, a);
        else hipLaunchKernelGGL((tq_paged_few_kernel<D, IPBK, IPBV, 1, true>), grid, t, 0, s, a);
    } else {
        if (vectors <= 16u / C) hipLaunchKernelGGL((tq_paged_few_kernel<D, IPBK, IPBV, C, false>), grid, t, 0, s, a);
        else hipLaunchKernelGGL((tq_paged_few_kernel<D, IPBK, IPBV, 1, false>), grid, t, 0, s, a);
    }
    return 0;
}
template <int D>
int launch_paged_few(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, uint32_t vectors) {
    if (ipbk == 4) return ipbv == 4 ? launch_paged_few<D, 4, 4>(grid, s, a, vectors) : ipbv == 2 ? launch_paged_few<D, 4, 2>(grid, s, a, vectors) : launch_paged_few<D, 4, 1>(grid, s, a, vectors);
    if (ipbk == 2) return ipbv == 4 ? launch_paged_few<D, 2, 4>(grid, s, a, vectors) : ipbv == 2 ? launch_paged_few<D, 2, 2>(grid, s, a, vectors) : launch_paged_few<D, 2, 1>(grid, s, a, vectors);
    return ipbv == 4 ? launch_paged_few<D, 1, 4>(grid, s, a, vectors) : ipbv == 2 ? launch_paged_few<D, 1, 2>(grid, s, a, vectors) : launch_paged_few<D, 1, 1>(grid, s, a, vectors);
}

}  // namespace
