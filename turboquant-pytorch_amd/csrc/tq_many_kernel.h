// Kernels of tq_many.hip that are the same for every code width: query rotation, uncompressed tokens, merge, and the attention
// over packed tokens for any head dimension.  DP: the head dimension as the next multiple of 32.
#pragma once
#include "tq_many.h"

namespace {

// ---- queries into the codec's space -----------------------------------------------------------------------------------------
// Block (row, two tiles, one where a row has no more): a tile's wave w has coordinates 32 w ... + 31 of 32 queries, q' = scale * log2(e) * Pi_k q from the operands of the key codec's
// table (Pi as three bf16 terms) and the queries' own bf16 terms, all products down to 2^-24 of the largest.  Every query is then scaled by
// the power of two that puts its largest coordinate into [2^Q_TOP, 2^(Q_TOP + 1)), so that none is too large or too small for the two fp16
// terms it is stored as, whatever the others are.
template <int DT>
__global__ __launch_bounds__(1024) void tq_many_prepare_kernel(TqManyArgs a, uint32_t waves) {
    __shared__ float lds_top[16][32];
    const uint32_t lane = threadIdx.x & 63u, every = tq_uniform32(threadIdx.x >> 6), side = every / waves, wave = every - side * waves;
    const uint32_t pairs = (a.tiles + 1u) / 2u, row = blockIdx.x / pairs, tile = 2u * (blockIdx.x - row * pairs) + side;
    const uint32_t DP = 32u * waves, steps = 2u * waves;
    const uint32_t n = lane & 31u, hk = lane >> 5, m = tile * 32u + n;
    constexpr int NT = plain_terms<DT>();
    const uint8_t *q = many_query(a, row, min(m, a.M - 1u), DT == TQ_F32 ? 4u : 2u);
    const uint8_t *pi = a.table_k + TQ_OFF_A_BF16(a.D) + ((size_t)wave * steps * 64u + lane) * 16u;
    const size_t term = TQ_OPERAND_BYTES_FOR(a.D);
    tq_f16v acc = tq_zero16();
    for (uint32_t s = 0; s < steps; ++s) {
        tq_u4 x[3];
        load_plain8<DT>(q, 16u * s + 8u * hk, a.D, a.aligned, x);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const tq_u4 p = tq_gload16(pi + i * term + (size_t)s * 1024u);
#pragma unroll
            for (int j = 0; j < NT; ++j)
                if (i + j < 3) acc = mfma_bf16(p, x[j], acc);
        }
    }
    float y[16], top = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {           // (the table's rows: register r of half h is coordinate 32 w + 16 h + r)
        y[r] = m < a.M ? acc[r] * (a.scale * LOG2E) : 0.f;
        const float v = fabsf(y[r]);
        top = fmaxf(top, v < __builtin_inff() ? v : 0.f);
    }
    top = halves_max(top);
    if (hk == 0u) lds_top[every][n] = top;
    __syncthreads();
    for (uint32_t w = 0; w < waves; ++w) top = fmaxf(top, lds_top[side * waves + w][n]);
    if (tile >= a.tiles) return;
    const size_t at = (size_t)row * a.tiles + tile;
    const int up = query_shift(top);
    const float f = __uint_as_float((uint32_t)(up + 127) << 23);
    if (wave == 0u && hk == 0u) a.q_scale[at * 32u + n] = __uint_as_float((uint32_t)(127 - up - LEVEL_SHIFT) << 23);
    uint8_t *dst = a.q_op + at * q_operand_bytes(DP);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint32_t t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = fp16_terms(y[8 * j + i] * f);
        tq_u4 hi, lo;
        fp16_operands(t, hi, lo);
        const uint32_t d = 32u * wave + 16u * hk + 8u * j, half = d / (DP / 2u), s = (d - half * (DP / 2u)) / 8u;
        uint8_t *p = dst + ((size_t)s * 64u + half * 32u + n) * 16u;
        tq_gstore16(p, hi);
        tq_gstore16(p + (size_t)steps * 1024u, lo);
    }
}

// ---- softmax of a tile of 32 tokens x 32 queries, columns = queries -----------------------------------------------------------------
// x: base-2 logits, MANY_NONE where a token is not seen.  Afterwards x holds the weights 2^(x - m) (zero where not seen); returns the factor
// by which the column's earlier sums shrink.
__device__ __forceinline__ float softmax_tile(float (&x)[16], float &m, float &l) {
    float top = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
    top = fmaxf(halves_max(top), m);
    const float shrink = __builtin_amdgcn_exp2f(m - top);
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        x[r] = x[r] == MANY_NONE ? 0.f : __builtin_amdgcn_exp2f(x[r] - top);
        sum += x[r];
    }
    m = top;
    l = l * shrink + halves_add(sum);
    return shrink;
}

// a record: column n of the wave's sums, coordinates 32 i + acc_row(r, h) in acc[i][r]
template <int DP>
__device__ __forceinline__ void put_sums(float *rec, uint32_t lane, float m, float l, const tq_f16v (&acc)[DP / 32], float f) {
    TQ_GLOBAL float *p = (TQ_GLOBAL float *)rec;
    const uint32_t n = lane & 31u, h = lane >> 5;
    if (h == 0u) { p[n] = m; p[32u + n] = l; }
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            *reinterpret_cast<TQ_GLOBAL tq_f4 *>(p + 64u + n * DP + 32u * i + 8u * k + 4u * h) =
                tq_f4{acc[i][4 * k] * f, acc[i][4 * k + 1] * f, acc[i][4 * k + 2] * f, acc[i][4 * k + 3] * f};
}

// ---- uncompressed tokens ---------------------------------------------------------------------------------------------------------
// Block (row, tile), waves take 32 tokens at a time of the window, then of the drafted tokens.  Products in bf16 terms of the elements
// and of the weights, down to 2^-24 of the largest: exact for 16-bit logits up to their summation.
template <int DP, int DT>
__global__ __launch_bounds__(64 * PLAIN_WAVES) void tq_many_plain_kernel(TqManyArgs a) {
    constexpr uint32_t ES = DT == TQ_F32 ? 4u : 2u;
    constexpr int NT = plain_terms<DT>();
    __shared__ float lds_p[PLAIN_WAVES][32][33];
    const uint32_t row = blockIdx.x / a.tiles, tile = blockIdx.x - row * a.tiles, b = row / a.heads, kv = row - b * a.heads;
    const uint32_t lane = threadIdx.x & 63u, wave = tq_uniform32(threadIdx.x >> 6), n = lane & 31u, h = lane >> 5;
    const uint32_t length = many_length(a, b);
    float m = MANY_NONE, l = 0.f;
    tq_f16v acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = tq_zero16();
    const uint32_t first = (a.plain[0].n + 31u) / 32u, all = first + (a.plain[1].n + 31u) / 32u;
    for (uint32_t w = wave; w < all; w += PLAIN_WAVES) {
        const uint32_t which = w < first ? 0u : 1u, t0 = 32u * (which ? w - first : w);
        const TqManyPlain &seg = a.plain[which];
        float x[16];
        plain_logits<DT>(a, seg, which, row, b, kv, t0, tile * 32u + n, lane, length, DP / 16u, x);
        const float shrink = softmax_tile(x, m, l);
        if (__any(shrink != 1.f)) {
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) acc[i] *= shrink;
        }
        // Step s of the value product contracts over the tokens that lane half h has weights of: 16 s + 4 h + 0 ... 3 and 16 s + 8 + 4 h + 0 ... 3.
        const uint8_t *v = seg.v + ((long long)b * seg.v_batch + (long long)kv * seg.v_head) * ES;
        bool wild = false;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            tq_u4 p[3];
            const float(&ps)[8] = *reinterpret_cast<const float(*)[8]>(&x[8 * s]);
            bf16_terms(ps, p);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const uint32_t d = 32u * i + n;
                float e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t t = t0 + 16u * s + acc_row(j, h);
                    e[j] = d < a.D && t < seg.n ? plain_element(v + ((long long)t * seg.v_token + d) * ES, DT) : 0.f;
                    if (!(fabsf(e[j]) < __builtin_inff())) { wild = true; e[j] = 0.f; }
                }
                tq_u4 vt[3];
                bf16_terms(e, vt);
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        if (j + k < 3) acc[i] = mfma_bf16(vt[j], p[k], acc[i]);
            }
        }
        if (__any(wild)) {
            // An infinite or NaN value must reach the queries that see its token, be their weight too small for a number or not, and no other: a product would spread it as 0 * inf.
            const uint32_t own = ManyQuery(a, min(tile * 32u + n, a.M - 1u)).t;
#pragma unroll
            for (int r = 0; r < 16; ++r) lds_p[wave][acc_row(r, h)][n] = x[r];
            wave_sync();
#pragma unroll 1
            for (uint32_t t = 0; t < min(32u, seg.n - t0); ++t) {
                const float p = lds_p[wave][t][n];
                const bool sees = plain_seen(a, which, b, own, t0 + t, length);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const uint32_t d = 32u * i + acc_row(r, h);
                        if (d < a.D && sees) {
                            const float e = plain_element(v + ((long long)(t0 + t) * seg.v_token + d) * ES, DT);
                            if (!(fabsf(e) < __builtin_inff())) acc[i][r] = fmaf(p, e, acc[i][r]);
                        }
                    }
            }
            wave_sync();
        }
    }
    put_sums<DP>(a.plain_rec + ((size_t)blockIdx.x * a.plain_records + wave) * record_floats(DP), lane, m, l, acc, 1.f);
}

template <int DT>
__global__ __launch_bounds__(64) void tq_many_plain_weights_kernel(TqManyArgs a, uint32_t steps) {
    plain_weights<DT>(a, blockIdx.x, steps, threadIdx.x);
}

// ---- packed tokens, any head dimension ------------------------------------------------------------------------------------------
// levels of a codebook as two fp16 terms, times 2^LEVEL_SHIFT
__device__ __forceinline__ void stage_levels(uint32_t *lds, const uint8_t *table, uint32_t bits) {
    const float *level = reinterpret_cast<const float *>(table + reinterpret_cast<const TqTableHeader *>(table)->off_centroids);
    for (uint32_t i = threadIdx.x; i < (1u << bits); i += blockDim.x) lds[i] = fp16_terms(level[i] * (float)(1 << LEVEL_SHIFT));
}

// Codes as they lie in bytes, most significant first
struct CodeShape {
    uint32_t bits, lg, mask, bytes;      // 2^lg codes a byte
    __device__ __forceinline__ CodeShape(uint32_t bits_, uint32_t D) : bits(bits_) {
        lg = bits >= 5u ? 0u : bits >= 3u ? 1u : bits == 2u ? 2u : 3u;
        mask = (1u << bits) - 1u;
        bytes = (D + (1u << lg) - 1u) >> lg;
    }
    __device__ __forceinline__ uint32_t code(const uint8_t *vec, uint32_t d) const {     // (d past the end: some code of the vector's last byte)
        const uint32_t at = min(d >> lg, bytes - 1u), k = (1u << lg) - 1u - (d & ((1u << lg) - 1u));
        return ((uint32_t)vec[at] >> (bits * k)) & mask;
    }
};

// a run of tokens' packed bytes into LDS, by one wave
__device__ __forceinline__ void stage_run(uint8_t *lds, const uint8_t *src, uint32_t bytes, uint32_t lane) {
    if (!(((uintptr_t)src | bytes) & 3u)) {
        for (uint32_t i = 4u * lane; i < bytes; i += 256u) *reinterpret_cast<uint32_t *>(lds + i) = tq_gload4(src + i);
    } else {
        for (uint32_t i = lane; i < bytes; i += 64u) lds[i] = *((const TQ_GLOBAL uint8_t *)src + i);
    }
}

constexpr int ANY_WAVES = 4;

// Base-2 logits of 32 staged tokens x 32 queries: levels and queries in two fp16 terms each (22 bits), as float32 arithmetic.
template <int DP>
__device__ __forceinline__ tq_f16v any_products(const uint8_t *keys, const CodeShape &ks, const uint32_t *levels, const uint8_t *q_op, uint32_t lane) {
    const uint32_t n = lane & 31u, h = lane >> 5;
    tq_f16v s = tq_zero16();
#pragma unroll 2
    for (uint32_t step = 0; step < DP / 16u; ++step) {
        uint32_t t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = levels[ks.code(keys + n * ks.bytes, h * (DP / 2u) + 8u * step + i)];
        tq_u4 hi, lo;
        fp16_operands(t, hi, lo);
        const tq_u4 qh = *reinterpret_cast<const tq_u4 *>(q_op + (step * 64u + lane) * 16u), ql = *reinterpret_cast<const tq_u4 *>(q_op + (DP / 16u + step) * 1024u + lane * 16u);
        s = mfma_f16(hi, qh, s);
        s = mfma_f16(hi, ql, s);
        s = mfma_f16(lo, qh, s);
    }
    return s;
}

// The simplest form that is right for every head dimension and code width: a wave stages 32 tokens' bytes in LDS and looks every code up by itself, which is what it takes its time
// for: 128 wide, 16 sequences of 8192 tokens x 64 query vectors a head 785 us (the kernel with tables 76), 1 x 2048 x 32 69 (19).  It is for what that one is not built for:
// 1 bit, head dimensions below 64, 72 ... 96 that are not whole words of packed bytes, above 96 but 128 and 256; fewer than 32 tokens; unaligned bytes.
template <int DP>
__global__ __launch_bounds__(64 * ANY_WAVES) void tq_many_any_kernel(TqManyArgs a) {
    __shared__ uint32_t lds_k[256], lds_v[256];
    __shared__ __attribute__((aligned(16))) uint8_t lds_q[2 * DP / 16 * 1024];
    __shared__ __attribute__((aligned(16))) uint8_t lds_raw[ANY_WAVES][2][32 * DP];
    __shared__ __attribute__((aligned(16))) float lds_norm[ANY_WAVES][2][32];
    const uint32_t split = blockIdx.x % a.splits, at = blockIdx.x / a.splits, row = at / a.tiles, b = row / a.heads;
    const uint32_t lane = threadIdx.x & 63u, wave = tq_uniform32(threadIdx.x >> 6), n = lane & 31u, h = lane >> 5;
    const CodeShape ks(a.bits_k, a.D), vs(a.bits_v, a.D);
    stage_levels(lds_k, a.table_k, a.bits_k);
    stage_levels(lds_v, a.table_v, a.bits_v);
    tq_copy_to_lds(lds_q, a.q_op + (size_t)at * q_operand_bytes(DP), q_operand_bytes(DP), threadIdx.x, blockDim.x);
    const float q_scale = a.q_scale[at * 32u + n];
    __syncthreads();
    const uint32_t seen = min(a.tokens, many_length(a, b));
    const uint32_t end = min(seen, split * a.chunk + a.chunk);
    const size_t slot0 = (size_t)row * a.packed_row_stride;
    const uint8_t *mask = a.mask ? a.mask + (long long)b * a.mask_stride : nullptr;
    float m = MANY_NONE, l = 0.f;
    int v_top = -200;                            // 2^v_top <= largest value norm so far < 2^(v_top + 1)
    tq_f16v acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = tq_zero16();
    for (uint32_t t0 = split * a.chunk + 32u * wave; t0 < end; t0 += 32u * ANY_WAVES) {
        const uint32_t count = min(32u, end - t0);
        uint8_t *keys = lds_raw[wave][0], *values = lds_raw[wave][1];
        float *kn = lds_norm[wave][0], *vn = lds_norm[wave][1];
        stage_run(keys, a.k_idx + (slot0 + t0) * ks.bytes, count * ks.bytes, lane);
        stage_run(values, a.v_idx + (slot0 + t0) * vs.bytes, count * vs.bytes, lane);
        const bool own = n < count && (!mask || mask[t0 + min(n, count - 1u)]);
        const uint16_t *norms = h ? a.v_norms : a.k_norms;
        const float norm = own ? (float)__builtin_bit_cast(_Float16, tq_gload2(norms + slot0 + t0 + n)) : 0.f;
        const uint32_t hidden = ~(uint32_t)__ballot(own);                  // bit t: token t0 + t is not seen
        (h ? vn : kn)[n] = norm;
        // the largest value norm of the run: the sums are kept in units that go with the largest so far
        float top = h ? fabsf(norm) : 0.f;
#pragma unroll
        for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
        const int run_top = max(-100, min(16, (int)(__float_as_uint(top) >> 23) - 127));
        wave_sync();
        const tq_f16v s = any_products<DP>(keys, ks, lds_k, lds_q, lane);
        float x[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = (hidden >> acc_row(r, h)) & 1u ? MANY_NONE : s[r] * (kn[acc_row(r, h)] * q_scale);
        float shrink = softmax_tile(x, m, l);
        if (run_top > v_top) {
            shrink *= __uint_as_float((uint32_t)max(0, 127 + v_top - run_top) << 23);
            v_top = run_top;
        }
        if (__any(shrink != 1.f)) {
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) acc[i] *= shrink;
        }
        const float unit = __uint_as_float((uint32_t)(127 + P_TOP - v_top) << 23);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            uint32_t t[8];
            tq_u4 ph, pl;
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = fp16_terms(x[8 * st + j] * (vn[16u * st + acc_row(j, h)] * unit));
            fp16_operands(t, ph, pl);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = lds_v[vs.code(values + (16u * st + acc_row(j, h)) * vs.bytes, 32u * i + n)];
                tq_u4 hi, lo;
                fp16_operands(t, hi, lo);
                acc[i] = mfma_f16(hi, ph, acc[i]);
                acc[i] = mfma_f16(hi, pl, acc[i]);
                acc[i] = mfma_f16(lo, ph, acc[i]);
            }
        }
        wave_sync();
    }
    const float back = v_top < -100 ? 0.f : __uint_as_float((uint32_t)(127 + v_top - P_TOP - LEVEL_SHIFT) << 23);
    put_sums<DP>(a.rec + ((size_t)at * a.records + split * ANY_WAVES + wave) * record_floats(DP), lane, m, l, acc, back);
}

// What the packed tokens receive: wave = 32 tokens, all query tiles of the row in order.
template <int DP>
__global__ __launch_bounds__(64 * ANY_WAVES) void tq_many_any_weights_kernel(TqManyArgs a, uint32_t blocks) {
    __shared__ uint32_t lds_k[256];
    __shared__ __attribute__((aligned(16))) uint8_t lds_raw[ANY_WAVES][32 * DP];
    __shared__ __attribute__((aligned(16))) float lds_norm[ANY_WAVES][32];
    const uint32_t row = blockIdx.x / blocks, b = row / a.heads;
    const uint32_t lane = threadIdx.x & 63u, wave = tq_uniform32(threadIdx.x >> 6), n = lane & 31u, h = lane >> 5;
    const CodeShape ks(a.bits_k, a.D);
    stage_levels(lds_k, a.table_k, a.bits_k);
    __syncthreads();
    const uint32_t seen = min(a.tokens, many_length(a, b)), t0 = 32u * ((blockIdx.x - row * blocks) * ANY_WAVES + wave);
    if (t0 >= seen) return;
    const size_t slot0 = (size_t)row * a.packed_row_stride;
    const uint32_t count = min(32u, seen - t0);
    stage_run(lds_raw[wave], a.k_idx + (slot0 + t0) * ks.bytes, count * ks.bytes, lane);
    const bool own = n < count && (!a.mask || a.mask[(long long)b * a.mask_stride + t0 + min(n, count - 1u)]);
    if (h == 0u) lds_norm[wave][n] = own ? (float)__builtin_bit_cast(_Float16, tq_gload2(a.k_norms + slot0 + t0 + n)) : 0.f;
    const uint32_t hidden = ~(uint32_t)__ballot(own);
    wave_sync();
    float w[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = 0.f;
    for (uint32_t tile = 0; tile < a.tiles; ++tile) {
        const size_t at = (size_t)row * a.tiles + tile;
        const tq_f16v s = any_products<DP>(lds_raw[wave], ks, lds_k, a.q_op + at * q_operand_bytes(DP), lane);
        const float *stat = a.stat + at * MANY_STATS;
        const float m = stat[n], inv = stat[32u + n], most = stat[64u + n], q_scale = a.q_scale[at * 32u + n];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint32_t t = acc_row(r, h);
            if (!((hidden >> t) & 1u) && inv != 0.f) w[r] = fmaf(__builtin_amdgcn_exp2f(weight_exponent(s[r], lds_norm[wave][t] * q_scale, m, most)), inv, w[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) w[r] += __shfl_xor(w[r], i);
    float mine = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) mine = n == (uint32_t)r ? w[r] : mine;
    const uint32_t t = acc_row((int)(n & 15u), h);
    if (n < 16u && t < count && !((hidden >> t) & 1u)) a.weights[(long long)row * a.w_stride + t0 + t] += mine;
}

// ---- merge ------------------------------------------------------------------------------------------------------------------------
// Block (row, tile, C of its 32 queries), DP / 32 waves: the records' sums with their factors, the packed ones turned back by Pi_v (two fp16 terms each of Pi_v^T,
// from the value codec's table, and of the sums: 22 bits), the uncompressed ones added, everything divided by the sum of weights.
// A query that sees nothing gets zeros.  C = 8 where tiles are fewer than 128: the records are then read by four times as many blocks (8 tiles x 31 records: the call 47 us instead of
// 60; 96 x 3: 52.0 and 53.5; but 256 x 2: 76.4 and, with C = 32, 73.2).  7 us for 8 tiles x 8 records of 128, 10.5 for 8 x 31.
// A launch of few blocks lasts as long as its chain of loads: what does not depend on anything (references, sums, the first records, Pi_v) is asked for at once.
constexpr uint32_t MERGE_RECORDS = 260;
template <int DP, int C>
__global__ __launch_bounds__(2 * DP) void tq_many_merge_kernel(TqManyArgs a) {
    constexpr uint32_t NT = 2 * DP, ROW = DP + 4, PARTS = NT / C, UNITS = C * DP / 4, STEPS = DP / 16, CH = STEPS <= 8 ? STEPS : 8;      // (NT is a multiple of 64)
    constexpr uint32_t UPT = (UNITS + NT - 1) / NT;                         // units of four coordinates a thread
    __shared__ __attribute__((aligned(16))) float lds_o[2][C * ROW];        // packed, plain
    __shared__ float lds_f[MERGE_RECORDS][C], lds_red[2][PARTS][C], lds_inv[C];
    const uint32_t group = blockIdx.x % (32u / C), at = blockIdx.x / (32u / C);
    const uint32_t row = at / a.tiles, tile = at - row * a.tiles, col0 = group * C;
    if (tile * 32u + col0 >= a.M && !a.stat) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tq_uniform32(tid >> 6), n32 = lane & 31u, h = lane >> 5;
    const TQ_GLOBAL float *rec = (const TQ_GLOBAL float *)a.rec + (size_t)at * a.records * record_floats(DP);
    const TQ_GLOBAL float *plain = (const TQ_GLOBAL float *)a.plain_rec + (size_t)at * a.plain_records * record_floats(DP);
    const uint32_t all = a.records + a.plain_records;
    auto record = [&](uint32_t i) { return i < a.records ? rec + (size_t)i * record_floats(DP) : plain + (size_t)(i - a.records) * record_floats(DP); };
    const uint32_t c = tid % C, part = tid / C;
    // ---- references and sums, two records a thread at first
    float ref[2], tot[2];
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
        const uint32_t i = part + k * PARTS;
        const TQ_GLOBAL float *p = record(min(i, all - 1u)) + col0 + c;
        ref[k] = p[0];
        tot[k] = p[32];
    }
    // ---- a unit's first eight packed records and its first plain one
    tq_f4 v[UPT == 1 ? 8 : 1], w[1];
    const uint32_t q0 = tid / (DP / 4u), e0 = (tid - q0 * (DP / 4u)) * 4u;
    if constexpr (UPT == 1) {
        const uint32_t off = 64u + (col0 + q0) * DP + e0;
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(record(min(k, all - 1u)) + off);
        w[0] = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(record(all - 1u) + off);
    }
    // ---- Pi_v (128 wide the table's operands have an order of their own, see tq_table.h)
    const uint8_t *pi = a.table_v + TQ_OFF_AT_F16(a.D) + ((size_t)wave * STEPS * 64u + lane) * 16u;
    tq_u4 ph[CH], pl[CH];
    auto load_pi = [&](uint32_t s0) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t s = 0; s < CH; ++s)
            if (s0 + s < STEPS) { ph[s] = tq_gload16(pi + (size_t)(s0 + s) * 1024u); pl[s] = tq_gload16(pi + TQ_OPERAND_BYTES_FOR(a.D) + (size_t)(s0 + s) * 1024u); }
    };
    load_pi(0);
    __builtin_amdgcn_sched_barrier(0);
    // ---- factors
    float top = MANY_NONE;
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k)
        if (part + k * PARTS < all) top = fmaxf(top, ref[k]);
    for (uint32_t i = part + 2u * PARTS; i < all; i += PARTS) top = fmaxf(top, record(i)[col0 + c]);
    lds_red[0][part][c] = top;
    __syncthreads();
#pragma unroll 8
    for (uint32_t k = 0; k < PARTS; ++k) top = fmaxf(top, lds_red[0][k][c]);
    float sum = 0.f;
    // A record without a largest logit is one of no token, with sums of zero, or one whose logits are all NaN: its sum of weights tells.  Nothing is left out for a factor
    // of zero: what is infinite or NaN in a record goes on into the result, however the tokens are split.
    auto factor = [&](uint32_t i, float r, float t) {
        const float f = r != MANY_NONE ? __builtin_amdgcn_exp2f(r - top) : t == 0.f ? 0.f : __builtin_nanf("");
        lds_f[i][c] = f;
        sum = fmaf(t, f, sum);
    };
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k)
        if (part + k * PARTS < all) factor(part + k * PARTS, ref[k], tot[k]);
    for (uint32_t i = part + 2u * PARTS; i < all; i += PARTS) factor(i, record(i)[col0 + c], record(i)[32u + col0 + c]);
    lds_red[1][part][c] = sum;
    __syncthreads();
    if (tid < (uint32_t)C) {
        float l = 0.f;
#pragma unroll 8
        for (uint32_t k = 0; k < PARTS; ++k) l += lds_red[1][k][tid];
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        lds_inv[tid] = inv;
        if (a.stat) put_stat(a.stat + (size_t)at * MANY_STATS, col0 + tid, tile * 32u + col0 + tid < a.M && inv != 0.f, top, l, inv);
    }
    // ---- sums
    auto add = [&](tq_f4 &o, tq_f4 x, float f) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
    };
#pragma unroll
    for (uint32_t u0 = 0; u0 < UPT; ++u0) {
        const uint32_t u = tid + u0 * NT;
        if (UNITS % NT && u >= UNITS) break;
        const uint32_t q = u / (DP / 4u), d = (u - q * (DP / 4u)) * 4u;
        tq_f4 o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        const uint32_t off = 64u + (col0 + q) * DP + d;
        uint32_t r0 = 0;
        if constexpr (UPT == 1) {
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (k < a.records) add(o[0], v[k], lds_f[k][q]);
            r0 = 8u;
        }
        for (; r0 < a.records; r0 += 8u) {
            tq_f4 x[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) x[k] = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(rec + (size_t)min(r0 + k, a.records - 1u) * record_floats(DP) + off);
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (r0 + k < a.records) add(o[0], x[k], lds_f[r0 + k][q]);
        }
        if (UPT == 1 && a.plain_records == 1u) add(o[1], w[0], lds_f[all - 1u][q]);
        else
            for (uint32_t r = 0; r < a.plain_records; ++r)
                add(o[1], *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(plain + (size_t)r * record_floats(DP) + off), lds_f[a.records + r][q]);
        if (DP != a.D)               // (what lies past the last coordinate may be anything)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) o[0][e] = d + e < a.D ? o[0][e] : 0.f;
        *reinterpret_cast<tq_f4 *>(&lds_o[0][q * ROW + d]) = o[0];
        *reinterpret_cast<tq_f4 *>(&lds_o[1][q * ROW + d]) = o[1];
    }
    __syncthreads();
    // ---- back out of the codec's space; columns past C repeat the others
    const uint32_t q = n32 % C;
    float largest = 0.f;
#pragma unroll 4
    for (uint32_t d = 0; d < DP / 2u; d += 4u) {
        const tq_f4 x = *reinterpret_cast<const tq_f4 *>(&lds_o[0][q * ROW + h * (DP / 2u) + d]);
#pragma unroll
        for (int e = 0; e < 4; ++e) largest = fmaxf(largest, fabsf(x[e]) < __builtin_inff() ? fabsf(x[e]) : 0.f);
    }
    largest = halves_max(largest);
    const int up = largest > 0.f ? max(-100, min(100, Q_TOP - ((int)(__float_as_uint(largest) >> 23) - 127))) : 0;
    const float f = __uint_as_float((uint32_t)(127 + up) << 23);
    const bool tuned = a.D == TQ_HEAD_DIM;
    tq_f16v acc = tq_zero16();
#pragma unroll 1
    for (uint32_t s0 = 0;;) {
#pragma unroll
        for (uint32_t s = 0; s < CH; ++s) {
            if (s0 + s >= STEPS) break;
            const uint32_t j = tuned ? 64u * h + 8u * (s0 + s) : 16u * (s0 + s) + 8u * h;
            tq_u4 oh, ol;
            fp16_split8(*reinterpret_cast<const tq_f4 *>(&lds_o[0][q * ROW + j]), *reinterpret_cast<const tq_f4 *>(&lds_o[0][q * ROW + j + 4u]), f, oh, ol);
            acc = mfma_f16(ph[s], oh, acc);
            acc = mfma_f16(ph[s], ol, acc);
            acc = mfma_f16(pl[s], oh, acc);
        }
        s0 += CH;
        if (s0 >= STEPS) break;
        load_pi(s0);
    }
    const uint32_t m = tile * 32u + col0 + q;
    if (m >= a.M || n32 >= (uint32_t)C) return;
    const float inv = lds_inv[q], back = __uint_as_float((uint32_t)(127 - up) << 23);
    const uint32_t d0 = tuned ? 64u * h + 16u * wave : 32u * wave + 16u * h;
    float o[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) o[r] = inv == 0.f ? 0.f : fmaf(acc[r], back, d0 + r < DP ? lds_o[1][q * ROW + d0 + r] : 0.f) * inv;
    store_result(a, row, m, d0, o);
}

}  // namespace
