// The kernel behind tq_paged_attend for sequences with few query vectors a kv head (a token or two of each: decoding), 16-bit elements, head dimensions 64, 96, 128 and 256.
// One source file per head dimension instantiates it.
#pragma once
#include "tq_decode_kernel.h"
#include "tq_paged_kernel.h"

namespace {

// Block = (item of the plan, kv head).  Up to 16 / C query vectors are the columns of 16 x 16 x 32 products, C times over, so that C blocks of 16 tokens share a softmax: every block's
// scores are made for all columns, a lane keeps those of its own column's block, and the weights of the others are zeros in its column of the value product (as in tq_decode_kernel, whose
// loop this is, with runs found through the sequence's pages: a run lies within a page, whose number is fetched a run ahead).  QT: fp16 terms of a rotated query, one for bfloat16.
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
    constexpr int HR = HEADS < 8 ? HEADS : 8;            // columns a round of the join
    constexpr int QROW = D + 4;
    using J = JoinArea<D, 1>;
    static_assert(DW * HR * PART * 4 <= (int)J::PACKED, "the waves' sums and the joined ones side by side");
    constexpr uint32_t Q_AT = 65536u + DW * VBYTES, LOOP_BYTES = Q_AT + 16u * QROW * 4u, AREA = LOOP_BYTES > J::BYTES ? LOOP_BYTES : J::BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[AREA];           // tables, values of each wave, rotated queries; later the waves' sums and the joined ones
    __shared__ __attribute__((aligned(16))) float lds_kn[DW][RUN];
    __shared__ __attribute__((aligned(16))) uint16_t lds_vn[DW][RUN];      // value norms / 2^ev_ref
    __shared__ __attribute__((aligned(16))) tq_u4 lds_q[QT > QREG ? (QT - QREG) * SK : 1][TQ_WAVE];
    __shared__ __attribute__((aligned(16))) float lds_corr[DW][16];
    __shared__ float lds_m[FAST_WAVES][32], lds_l[FAST_WAVES][32];
    __shared__ uint32_t lds_trips[DW];

    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tq_uniform32(tid >> 6), n16 = lane & 15u, q4 = lane >> 4;
    const uint32_t item = blockIdx.x / a.heads;
    const int32_t *it = a.items + (size_t)item * PAGED_ITEM;
    const int32_t *sq = a.seqs + (size_t)it[0] * PAGED_SEQ;
    const uint32_t t_begin = (uint32_t)it[2], t_end = (uint32_t)it[3], plain_from = (uint32_t)it[4], plain_to = (uint32_t)it[5];
    const int record = it[6];
    PagedRow row;
    row.fresh = (uint32_t)sq[1]; row.total = (uint32_t)sq[2]; row.packed = (uint32_t)sq[3];
    row.pages = a.tables + sq[4]; row.plain_pages = a.tables + sq[5];
    row.kv = blockIdx.x - item * a.heads;
    const uint32_t q_first = (uint32_t)sq[0], M = row.fresh * a.group;
    const uint8_t *queries = a.q + ((long long)q_first * a.q_token + (long long)(row.kv * a.group) * a.q_head) * 2;
    const uint32_t head = n16 % HEADS, cls = n16 / HEADS;
    const bool live = head < M;

    if (t_end > t_begin) {
        const uint32_t token = min(head, M - 1u) / a.group, pos = row.total - row.fresh + token;
        const float slope = a.slopes ? a.slopes[row.kv * a.group + (min(head, M - 1u) - token * a.group)] * LOG2E : 0.f;
        const uint32_t lo = a.window && pos >= a.window ? pos - a.window + 1u : 0u;              // first token that this lane's column sees
        const uint32_t last_pos = row.total - 1u, whole_from = a.window && last_pos >= a.window ? last_pos - a.window + 1u : 0u;
        const bool shaped = a.cap != 0.f || a.slopes;
        uint8_t *vcodes = lds + 65536 + wave * VBYTES;
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
        // ---- start: tables, then the operands of the query rotation (the first waves), then the first run
        if (tid < (uint32_t)DW) lds_trips[tid] = 0u;
        Lut<IPBK> table_k;
        Lut<IPBV> table_v;
        table_k.load(a.table_k + TQ_OFF_LUT(D), tid);
        table_v.load(a.table_v + TQ_OFF_LUT(D), tid);
        Where now = where(0u), next = where(1u);
        __builtin_amdgcn_sched_barrier(0);
        auto first_run = [&]() __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
            issue_keys(now, max(run_tokens(0u), 1u));
            issue_values(now, max(run_tokens(0u), 1u));
            __builtin_amdgcn_sched_barrier(0);
            table_k.store(lds, tid);
            table_v.store(lds + 128, tid);
        };
        if (wave < (uint32_t)TILES) {
            Rotation<D, BF> r;
            const uint32_t m = n16 < M ? n16 : 0u, t = m / a.group;
            r.qsrc = queries + ((long long)t * a.q_token + (long long)(m - t * a.group) * a.q_head) * 2 + 16u * q4;
            r.asrc = a.table_k + (BF ? TQ_OFF_A_BF16(D) : TQ_OFF_A_F16) + ((size_t)wave * (D / 16 * 64u) + q4 * 32u + n16) * 16u;
            r.fetch(0);
            first_run();
            r.finish(reinterpret_cast<float *>(lds + Q_AT), QROW, a.scale, wave, lane);
        } else first_run();
        __syncthreads();

        // ---- B operand of the score product: fp16 of q * 2^(10 - e), e = binary exponent of the column's largest magnitude
        tq_u4 qb[QREG][SK];
        float c1;                // base-2 logit = accumulator * key norm * c1
        {
            const float *q = reinterpret_cast<const float *>(lds + Q_AT) + head * QROW + (D / 4) * q4;
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
            c1 = live ? ldexpf(LOG2E, e - TQ_F16_PI_SHIFT) : 0.f;
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
        const uint32_t slot_k = RepLut<IPBK>::lane_offset(lane), slot_v = 128u + RepLut<IPBV>::lane_offset(lane);
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
                    const tq_u4 kd = decode_keys<IPBK, NWK>(kraw[u][b], s, lds, slot_k);
#pragma unroll
                    for (int k = 0; k < QT; ++k) sc[u][b] = mfma16_f16(kd, q[k], sc[u][b]);
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
#pragma unroll
                    for (int j = 0; j < SPL; ++j) z[j] = shape_logit(a, z[j], slope, (float)((int)(t0 + tok + 16u * (j / 4) + (j % 4)) - (int)pos));
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
        uint32_t trips = 0u;
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
                const _Float16 kh = __builtin_bit_cast(_Float16, kn_raw);
                if (RUN == 64 || lane < (uint32_t)RUN) lds_kn[wave][lane] = (float)kh;     // one token per lane
                // does a value norm of this run exceed the reference exponent?  (a vote; a handful of times per wave)
                const uint16_t vn = lane < n_tok ? vn_raw : (uint16_t)0;   // tokens past the end weigh nothing
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
            for (;;) {
#pragma unroll 1
                while (run_tokens(i) == (uint32_t)RUN && run_start(i) >= whole_from) trip(std::true_type{}, i++);
                if (!run_tokens(i)) break;
                trip(std::false_type{}, i++);
            }
            if (lane == 0u) *(volatile __attribute__((address_space(3))) uint32_t *)&lds_trips[wave] = 0xffffffffu;
            __builtin_amdgcn_s_setprio(0);
        }
        // ---- the waves' sums of HR columns at a time meet in LDS
        float l_all = l_run;
#pragma unroll
        for (int d = HEADS; d < 64; d <<= 1) l_all += __shfl_xor(l_all, d);
        l_all *= 1.0f / (float)(1 << P_SHIFT);
        const float unit = ldexpf(1.f, ev_ref - P_SHIFT);
        float *const mine = reinterpret_cast<float *>(lds) + wave * (HR * PART);
        for (uint32_t h0 = 0; h0 < (uint32_t)HEADS && h0 < M; h0 += HR) {
            __syncthreads();         // (tables, values, and the round before)
            if (q4 == 0u && cls == 0u && n16 >= h0 && n16 < h0 + HR) {
                mine[(n16 - h0) * PART] = m_ref;
                mine[(n16 - h0) * PART + 1u] = l_all;
            }
            if constexpr (C == 1) {
                if (4u * q4 >= h0 && 4u * q4 < h0 + HR) {
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int r = 0; r < 4; ++r) mine[(4u * q4 + r - h0) * PART + 2u + value_coord<D>(n16, c)] = acc[c][r] * unit;
                }
            } else {
                // The blocks of tokens lie in lanes 32 apart (C = 4: and 16 apart): two registers exchange halves and are added, which leaves the sum of one in each half (then quarters).
                static_assert(HR >= HEADS, "one round");
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
            __syncthreads();
            const float *all = reinterpret_cast<const float *>(lds);
            for (uint32_t i = tid; i < HR * D; i += DTHREADS) {
                const uint32_t col = i / D, d = i - col * D;
                float m = MANY_NONE, sum = 0.f, total = 0.f;
#pragma unroll
                for (int w = 0; w < DW; ++w) m = fmaxf(m, all[(w * HR + col) * PART]);
#pragma unroll
                for (int w = 0; w < DW; ++w) {
                    const float own = all[(w * HR + col) * PART], l = all[(w * HR + col) * PART + 1u];
                    const float f = own != MANY_NONE ? __builtin_amdgcn_exp2f(own - m) : l == 0.f ? 0.f : __builtin_nanf("");
                    sum = fmaf(all[(w * HR + col) * PART + 2u + d], f, sum);
                    total = fmaf(l, f, total);
                }
                J::sums(lds, 0u, 0u)[(h0 + col) * (D + 4u) + d] = sum;
                if (d == 0u) {
                    J::largest(lds, 0u, 0u)[h0 + col] = m;
                    J::total(lds, 0u, 0u)[h0 + col] = total;
                }
            }
        }
        __syncthreads();
    }
    const bool plain = plain_to > plain_from;
    if (plain) {
        TqManyArgs v;            // (queries as the plain tokens' products take them: "heads" are the sequence's tokens)
        v.q = queries;
        v.q_batch = 0; v.q_head = a.q_token; v.q_token = a.q_head;
        v.heads = 1u; v.queries = a.group; v.M = M; v.D = a.D; v.aligned = 1u;
        paged_plain_phase<D, 1, BF ? TQ_BF16 : TQ_F16>(a, v, row, lds, lds_m, lds_l, &lds_corr[0][0], 0u, 1u, plain_from, plain_to, tid);
    }
    paged_finish<D, 1>(a, lds, t_end > t_begin, plain, row, q_first, record, 0u, 1u, tid);
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
