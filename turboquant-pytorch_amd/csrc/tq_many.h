// Attention of several query tokens over a packed history and uncompressed tokens (tq_many.hip): what its kernels and the
// sources that instantiate them share.
//
// A row is a (sequence, kv head); its M = group * queries query vectors are worked on in tiles of 32, the columns of a 32 x 32 matrix
// product.  With q' = Pi_k q, logit(t, m) = norm_t * sum_j level[code_tj] q'_mj, so the keys are never turned back: the product runs over
// the levels themselves.  Values the same way: sum_t p_tm norm_t level[code_tj] is turned by Pi_v once per query, at the end.
#pragma once
#include "tq_device.h"

struct TqManyPlain {                 // uncompressed tokens of a row: token t of head h of sequence b at b * batch + h * head + t * token elements
    const uint8_t *k, *v;
    long long k_batch, k_head, k_token, v_batch, v_head, v_token;
    uint32_t n;
};

struct TqManyArgs {
    const uint8_t *q;                // query head j, token i of sequence b at b * q_batch + j * q_head + i * q_token elements
    uint8_t *out;                    // dense [batch, query heads, queries, D]
    long long q_batch, q_head, q_token;
    const uint8_t *k_idx, *v_idx;
    const uint16_t *k_norms, *v_norms;
    const uint8_t *table_k, *table_v;
    TqManyPlain plain[2];            // behind the packed tokens: the window, and the drafted tokens
    const int32_t *lengths;          // keys of sequence b that count (packed, then window), or null: all
    const uint8_t *mask;             // [batch, mask_stride] truth value of every key (packed, then window), or null
    const uint8_t *tree;             // drafted token j is seen by query i if tree[b * tree_batch + i * plain[1].n + j], or null: if j <= i
    long long mask_stride, tree_batch;
    float *weights;                  // [rows, w_stride] what every key (packed, then window) receives is added here; or null
    long long w_stride;
    uint8_t *q_op;                   // rotated queries as operands, see q_operand_bytes
    float *q_scale;                  // [rows, tiles, 32] what a query's products are multiplied with
    float *rec;                      // [rows, tiles, records][32 largest logits, 32 sums, 32 x DP value sums]: packed tokens' (value space of the codec)
    float *plain_rec;                // the same of the uncompressed tokens (plain space)
    float *stat;                     // [rows, tiles][32 largest logits, 32 reciprocal sums, 32 largest exponents], see put_stat (only with weights)
    float scale;
    uint32_t rows, heads, group, queries, M, tiles, tokens, packed_row_stride, D, bits_k, bits_v, dtype;
    uint32_t splits, chunk, records, plain_records;
    uint32_t plain_blocks;           // blocks of a launch, its first ones, that work on the uncompressed tokens
    uint32_t aligned;                // vectors of queries and uncompressed tokens can be read 16 bytes at a time
};

namespace {

typedef float tq_f4 __attribute__((ext_vector_type(4)));

constexpr float MANY_NONE = -3.0e38f;        // largest logit of no token at all
constexpr int LEVEL_SHIFT = 6;               // levels enter the products times 2^6: their second fp16 term stays above the subnormals' grid
constexpr int Q_TOP = 13;                    // the largest coordinate of rotated queries that are scaled together lies in [2^13, 2^14)
constexpr int P_TOP = 14;                    // weight * value norm, at most 2^15
constexpr int PLAIN_WAVES = 4;
constexpr float LOG2E = 1.44269504088896340736f;

// Rotated queries of a tile: per fp16 term (leading, rest) and step s of 16 coordinates 64 lanes x 16 bytes; lane (n = lane % 32, hk = lane / 32) has
// query n, coordinates hk * DP / 2 + 8 s ... + 7 (a lane's share of a packed key is then one run of bytes).
__host__ __device__ constexpr uint32_t q_operand_bytes(uint32_t dp) { return 2u * (dp / 16u) * 1024u; }
__host__ __device__ constexpr uint32_t record_floats(uint32_t dp) { return 64u + 32u * dp; }

// Whether the kept sums' launch works on 16 columns instead of 32: no more query vectors a row, and a window of 16-bit elements (float32's in three terms would spill beside two
// blocks a compute unit)
__host__ __device__ inline bool many_few(const TqManyArgs &a, uint32_t dp) { return a.M <= 16u && a.dtype != TQ_F32 && (dp == 64u || dp == 128u || dp == 256u); }

// What the launches that add up what keys receive know of a query: weight = 2^(logit - largest) / sum.  They have the logit from another order of sums than the attention's launch,
// and of one in the millions the last bit is more than an exponent can be: no weight becomes larger than one (2^0.01 for rounding).  A query that is none, or sees nothing
// (`some` false), gives nothing.
constexpr uint32_t MANY_STATS = 96;
__device__ __forceinline__ void put_stat(float *stat, uint32_t n, bool some, float largest, float sum, float inv) {
    stat[n] = some ? largest : -MANY_NONE;
    stat[32u + n] = some ? inv : 0.f;
    stat[64u + n] = some ? __builtin_amdgcn_logf(sum) + 0.01f : 0.f;
}
// The exponent, from a product and what it is to be multiplied by.  (Where that is NaN the query's sum is, too.)
__device__ __forceinline__ float weight_exponent(float s, float f, float largest, float most) { return fminf(fmaf(s, f, -largest), most); }

// Row of a result register r of a 32 x 32 product in lane half h
__device__ __forceinline__ constexpr uint32_t acc_row(int r, uint32_t h) { return 8u * (uint32_t)(r / 4) + 4u * h + (uint32_t)(r % 4); }

// Order of this wave's LDS accesses among its lanes
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Over the two lanes that share a column
__device__ __forceinline__ float halves_max(float x) {
    const auto two = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(two[0]), __uint_as_float(two[1]));
}
__device__ __forceinline__ float halves_add(float x) {
    const auto two = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(two[0]) + __uint_as_float(two[1]);
}

// By which power of two a query whose largest coordinate is `top` is scaled to have it in [2^Q_TOP, 2^(Q_TOP + 1)).  (2^-114 does that for the largest float.)
__device__ __forceinline__ int query_shift(float top) { return top > 0.f ? max(-114, min(100, Q_TOP - ((int)(__float_as_uint(top) >> 23) - 127))) : 0; }

// float -> two fp16 terms, packed (leading | rest << 16): 22 bits while neither term falls below 2^-14.  Infinities and NaN have no rest.
__device__ __forceinline__ uint32_t fp16_terms(float x) {
    const _Float16 hi = (_Float16)x;
    const float r = x - (float)hi;
    const _Float16 lo = (_Float16)(r == r ? r : 0.f);
    return (uint32_t)__builtin_bit_cast(uint16_t, hi) | ((uint32_t)__builtin_bit_cast(uint16_t, lo) << 16);
}
// Eight floats, times f -> operands of both terms, in half the instructions (an infinity's rest is NaN: where everything turns into NaN anyway)
__device__ __forceinline__ void fp16_split8(tq_f4 x, tq_f4 y, float f, tq_u4 &hi, tq_u4 &lo) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const float a = (d < 2 ? x[2 * d] : y[2 * d - 4]) * f, b = (d < 2 ? x[2 * d + 1] : y[2 * d - 3]) * f;
        const tq_half2 h = {(_Float16)a, (_Float16)b};
        const tq_half2 l = {(_Float16)(a - (float)h[0]), (_Float16)(b - (float)h[1])};
        hi[d] = __builtin_bit_cast(uint32_t, h);
        lo[d] = __builtin_bit_cast(uint32_t, l);
    }
}
// eight of them -> two operands
__device__ __forceinline__ void fp16_operands(const uint32_t (&t)[8], tq_u4 &hi, tq_u4 &lo) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        hi[d] = __builtin_amdgcn_perm(t[2 * d + 1], t[2 * d], 0x05040100u);
        lo[d] = __builtin_amdgcn_perm(t[2 * d + 1], t[2 * d], 0x07060302u);
    }
}

// Eight floats -> three bf16 terms that add up to them (an infinity or NaN has only its first).
__device__ __forceinline__ void bf16_terms(const float (&x)[8], tq_u4 (&t)[3]) {
    uint32_t a[8], b[8], c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a[i] = __float_as_uint(x[i]) & 0xffff0000u;
        float r = x[i] - __uint_as_float(a[i]);
        r = r == r ? r : 0.f;
        b[i] = __float_as_uint(r) & 0xffff0000u;
        c[i] = __float_as_uint(r - __uint_as_float(b[i]));
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        t[0][d] = __builtin_amdgcn_perm(a[2 * d + 1], a[2 * d], 0x07060302u);
        t[1][d] = __builtin_amdgcn_perm(b[2 * d + 1], b[2 * d], 0x07060302u);
        t[2][d] = __builtin_amdgcn_perm(c[2 * d + 1], c[2 * d], 0x07060302u);
    }
}

__device__ __forceinline__ float plain_element(const uint8_t *p, uint32_t dtype) {
    if (dtype == TQ_F32) return *reinterpret_cast<const TQ_GLOBAL float *>((const TQ_GLOBAL uint8_t *)p);
    const uint16_t h = tq_gload2(reinterpret_cast<const uint16_t *>(p));
    return dtype == TQ_F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
}

// Elements [first, first + 8) of a vector as NT bf16 terms that add up to them (bf16: 1, fp16: 2, float32: 3); those from D on are zero.
template <int DT> constexpr int plain_terms() { return DT == TQ_BF16 ? 1 : DT == TQ_F16 ? 2 : 3; }
template <int DT>
__device__ __forceinline__ void load_plain8(const uint8_t *vec, uint32_t first, uint32_t D, bool aligned, tq_u4 (&t)[3]) {
    constexpr uint32_t ES = DT == TQ_F32 ? 4u : 2u;
    const uint8_t *p = vec + first * ES;
    float x[8];
    if (first >= D) {
        t[0] = t[1] = t[2] = tq_u4{0u, 0u, 0u, 0u};
        return;
    }
    if (aligned) {           // (D is a multiple of 8 then)
        const tq_u4 a = tq_gload16(p);
        if constexpr (DT == TQ_BF16) {
            t[0] = a;
            return;
        } else if constexpr (DT == TQ_F16) {
            const tq_half8 h = __builtin_bit_cast(tq_half8, a);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
        } else {
            const tq_u4 b = tq_gload16(p + 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[i] = __uint_as_float(a[i]); x[4 + i] = __uint_as_float(b[i]); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = first + i < D ? plain_element(p + i * ES, DT) : 0.f;
    }
    bf16_terms(x, t);
}

// Position of a row's query vector m: query head and token
struct ManyQuery {
    uint32_t g, t;
    __device__ __forceinline__ ManyQuery(const TqManyArgs &a, uint32_t m) : g(m / a.queries), t(m - g * a.queries) {}
};
__device__ __forceinline__ const uint8_t *many_query(const TqManyArgs &a, uint32_t row, uint32_t m, uint32_t elem_bytes) {
    const uint32_t b = row / a.heads, h = row - b * a.heads;
    const ManyQuery q(a, m);
    return a.q + ((long long)b * a.q_batch + (long long)(h * a.group + q.g) * a.q_head + (long long)q.t * a.q_token) * elem_bytes;
}

// Whether a query with token position `own` sees uncompressed token t (`which`: 0 window, 1 drafts)
__device__ __forceinline__ bool plain_seen(const TqManyArgs &a, uint32_t which, uint32_t b, uint32_t own, uint32_t t, uint32_t length) {
    if (which == 0u) {
        const uint32_t at = a.tokens + t;
        return at < length && (!a.mask || a.mask[(long long)b * a.mask_stride + at]);
    }
    return a.tree ? a.tree[(long long)b * a.tree_batch + (long long)own * a.plain[1].n + t] != 0 : t <= own;
}

// Coordinates d0 ... d0 + 15 of query vector m's result
__device__ __forceinline__ void store_result(const TqManyArgs &a, uint32_t row, uint32_t m, uint32_t d0, const float (&o)[16]) {
    const ManyQuery q(a, m);
    const size_t first = (((size_t)row * a.group + q.g) * a.queries + q.t) * a.D + d0;
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

// Keys of sequence b (packed, then window) that can count
__device__ __forceinline__ uint32_t many_length(const TqManyArgs &a, uint32_t b) {
    const uint32_t all = a.tokens + a.plain[0].n;
    if (!a.lengths) return all;
    const int32_t l = a.lengths[b];
    return l < 0 ? 0u : min((uint32_t)l, all);
}

// Base-2 logits of 32 uncompressed tokens x 32 queries, MANY_NONE where a token is not seen
template <int DT>
__device__ __forceinline__ void plain_logits(const TqManyArgs &a, const TqManyPlain &seg, uint32_t which, uint32_t row, uint32_t b, uint32_t kv, uint32_t t0, uint32_t m,
                                             uint32_t lane, uint32_t length, uint32_t steps, float (&x)[16]) {
    constexpr uint32_t ES = DT == TQ_F32 ? 4u : 2u;
    constexpr int NT = plain_terms<DT>();
    const uint32_t n = lane & 31u, h = lane >> 5;
    const uint8_t *k = seg.k + ((long long)b * seg.k_batch + (long long)kv * seg.k_head + (long long)min(t0 + n, seg.n - 1u) * seg.k_token) * ES;
    const uint8_t *q = many_query(a, row, min(m, a.M - 1u), ES);
    tq_f16v acc = tq_zero16();
    for (uint32_t s = 0; s < steps; ++s) {
        tq_u4 kt[3], qt[3];
        load_plain8<DT>(k, 16u * s + 8u * h, a.D, a.aligned, kt);
        load_plain8<DT>(q, 16u * s + 8u * h, a.D, a.aligned, qt);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                if (i + j < 3) acc = mfma_bf16(kt[i], qt[j], acc);
    }
    const uint32_t i = ManyQuery(a, min(m, a.M - 1u)).t;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const uint32_t t = t0 + acc_row(r, h);
        const bool seen = t < seg.n && plain_seen(a, which, b, i, t, length);
        x[r] = seen ? acc[r] * (a.scale * LOG2E) : MANY_NONE;
    }
}

// What the window's tokens receive is added to a.weights: wave = 32 tokens, all query tiles of the row in order, so that a token's sum is made by one wave in a fixed order.
template <int DT>
__device__ __forceinline__ void plain_weights(const TqManyArgs &a, uint32_t item, uint32_t steps, uint32_t lane) {
    const TqManyPlain &seg = a.plain[0];
    const uint32_t groups = (seg.n + 31u) / 32u;
    const uint32_t row = item / groups, t0 = 32u * (item - row * groups), b = row / a.heads, kv = row - b * a.heads;
    const uint32_t n = lane & 31u, h = lane >> 5, length = many_length(a, b);
    float w[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = 0.f;
    for (uint32_t tile = 0; tile < a.tiles; ++tile) {
        float x[16];
        plain_logits<DT>(a, seg, 0u, row, b, kv, t0, tile * 32u + n, lane, length, steps, x);
        const float *stat = a.stat + ((size_t)row * a.tiles + tile) * MANY_STATS;
        const float m = stat[n], inv = stat[32u + n], most = stat[64u + n];
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (x[r] != MANY_NONE && inv != 0.f) w[r] = fmaf(__builtin_amdgcn_exp2f(weight_exponent(x[r], 1.f, m, most)), inv, w[r]);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) w[r] += __shfl_xor(w[r], i);
    float own = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) own = n == (uint32_t)r ? w[r] : own;
    const uint32_t t = t0 + acc_row((int)(n & 15u), h);
    if (n < 16u && t < seg.n && a.tokens + t < length) a.weights[(long long)row * a.w_stride + a.tokens + t] += own;
}

}  // namespace

// Launches tq_many_fast_kernel for one padded head dimension; ipbk, ipbv = codes per byte (1, 2, 4), qt = tiles of 32 queries a block, kt, vt = fp16 terms on the key and value side
int tq_many_launch_d64(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqManyArgs &a, int qt, int kt, int vt);
int tq_many_launch_d96(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqManyArgs &a, int qt, int kt, int vt);
int tq_many_launch_d128(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqManyArgs &a, int qt, int kt, int vt);
int tq_many_launch_d256(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqManyArgs &a, int qt, int kt, int vt);
// the same for tq_many_weights_kernel, `blocks` a row
int tq_many_weights_launch_d64(int ipbk, dim3 grid, hipStream_t s, const TqManyArgs &a, uint32_t blocks);
int tq_many_weights_launch_d96(int ipbk, dim3 grid, hipStream_t s, const TqManyArgs &a, uint32_t blocks);
int tq_many_weights_launch_d128(int ipbk, dim3 grid, hipStream_t s, const TqManyArgs &a, uint32_t blocks);
int tq_many_weights_launch_d256(int ipbk, dim3 grid, hipStream_t s, const TqManyArgs &a, uint32_t blocks);
