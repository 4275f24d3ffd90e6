// Of every row of a packed store the `keep` tokens with the largest weights, in their order, into another store: tq_evict.
// Two launches: which tokens stay (a block a row), and their bytes; of rows of more than 32768 tokens, five: a block a segment.
#include "tq_device.h"

namespace {

constexpr int SELECT_THREADS = 1024;

struct EvictArgs {
    const float *weights;            // [rows, w_stride]; the first `tokens` of a row are the packed tokens', `rest` more follow
    float *weights_out;              // [rows, w_out_stride]
    long long *kept;                 // [rows, keep] slots that stay, ascending
    const uint8_t *idx[2];
    const uint16_t *norms[2];
    uint8_t *idx_out[2];             // dense [rows, keep]
    uint16_t *norms_out[2];
    long long w_stride, w_out_stride, row_stride, out_stride;
    uint32_t rows, tokens, keep, rest, bytes[2], unit[2];
    uint32_t *scratch;               // of rows of more than 32768 tokens: [rows][3 rounds][segments][2048] counts, [rows][segments] states
    uint32_t segments, segment_tokens;
};

// Weights as whole numbers of the same order: NaN above everything, the two zeros equal.
__device__ __forceinline__ uint32_t order_of(float w) {
    uint32_t u = __float_as_uint(w);
    if (w != w) return 0xffffffffu;
    if (u == 0x80000000u) u = 0u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the threads before this one, and over all
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *lds, uint32_t &total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (uint32_t i = 1; i < 64; i <<= 1) {
        const uint32_t y = __shfl_up(x, i);
        if (lane >= i) x += y;
    }
    if (lane == 63u) lds[wave] = x;
    __syncthreads();
    uint32_t before = 0u;
    total = 0u;
    for (uint32_t w = 0; w < SELECT_THREADS / 64; ++w) {
        if (w < wave) before += lds[w];
        total += lds[w];
    }
    __syncthreads();
    return before + x - v;
}

// Block = row, its weights in registers (E a thread, token e * 1024 + thread), up to 32768 tokens (the call, 8 rows of 32768: 30 us; 128 of 8191: 45 with E = 16, 48 with 32;
// 8 of 1152: 18 with 4, 24 with 32). Bound by its own steps one after the other: 10, 20 and 13 us for 4 KB, 128 KB and 32 KB a row.
// The keep-th largest weight lies in a range of whole numbers, at first all there are.  While more than 256 tokens lie in it, it is cut into 2048 parts, the tokens of each are counted
// in LDS, and the part with the keep-th one is the next range: a floating-point number's bits go with its logarithm, so that sums spread over the parts and few of the
// counts' atomics meet (counting by the leading byte instead took 110 us for 8 x 32768 tokens; those at the lower end, zeros, are counted by ballots).
// What is left is packed, and four threads count those above each (up to 1024 of them bit by bit, with a barrier each, took 13, 27 and 18 us in all).  Tokens above the result stay, and of those equal to it the first ones; places come
// from counts per wave and register, in the tokens' order.
template <int E>
__global__ __launch_bounds__(SELECT_THREADS) void tq_evict_select_kernel(EvictArgs a) {
    constexpr uint32_t WAVES = SELECT_THREADS / 64, PARTS = 2048, FEW = 256;
    __shared__ __attribute__((aligned(16))) uint32_t lds_few[FEW + 4];
    __shared__ uint32_t lds_part[PARTS], lds_count[WAVES], lds_ends[2][WAVES], lds_place[E * WAVES], lds_found[3], lds_n;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tq_uniform32(tid >> 6);
    const TQ_GLOBAL float *w = (const TQ_GLOBAL float *)a.weights + (long long)row * a.w_stride;
    uint32_t key[E], lo = 0xffffffffu, hi = 0u;           // a token that is none: 0, less than any number's
    auto each = [&](auto f) __attribute__((always_inline)) {      // f(key) of all tokens, by all threads together
#pragma unroll
        for (int e = 0; e < E; ++e) f(key[e]);
    };
    {
        constexpr int CH = E < 16 ? E : 16;
#pragma unroll
        for (int e0 = 0; e0 < E; e0 += CH) {
            float v[CH];
#pragma unroll
            for (int e = 0; e < CH; ++e) v[e] = w[min((e0 + e) * SELECT_THREADS + tid, a.tokens - 1u)];
#pragma unroll
            for (int e = 0; e < CH; ++e) key[e0 + e] = (e0 + e) * SELECT_THREADS + tid < a.tokens ? order_of(v[e]) : 0u;
        }
    }
    each([&](uint32_t k) {
        hi = max(hi, k);
        lo = min(lo, k - 1u);                             // (none: as large as can be)
    });
#pragma unroll
    for (int i = 32; i; i >>= 1) { lo = min(lo, (uint32_t)__shfl_xor(lo, i)); hi = max(hi, (uint32_t)__shfl_xor(hi, i)); }
    if (lane == 0u) { lds_ends[0][wave] = lo; lds_ends[1][wave] = hi; }
    if (tid == 0u) lds_n = 0u;
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < WAVES; ++k) { lo = min(lo, lds_ends[0][k]); hi = max(hi, lds_ends[1][k]); }
    lo += 1u;                                             // (a row has a token at least)
    uint32_t left = a.keep, agree = a.tokens;             // agree tokens in [lo, hi], of which the largest `left` stay; all above hi do
    while (agree > FEW && lo < hi && left < agree) {
        const uint32_t width = 32u - (uint32_t)__builtin_clz(hi - lo), shift = width > 11u ? width - 11u : 0u;
#pragma unroll
        for (uint32_t k = 0; k < PARTS / SELECT_THREADS; ++k) lds_part[tid + k * SELECT_THREADS] = 0u;
        __syncthreads();
        uint32_t lowest = 0u;
        each([&](uint32_t k) {
            lowest += (uint32_t)__popcll(__ballot(k == lo));
            if (k > lo && k <= hi) atomicAdd(&lds_part[(k - lo) >> shift], 1u);
        });
        if (lane == 0u && lowest) atomicAdd(&lds_part[0], lowest);
        __syncthreads();
        // from the upper end: two parts a thread
        const uint32_t p1 = PARTS - 1u - 2u * tid, c1 = lds_part[p1], c0 = lds_part[p1 - 1u];
        uint32_t all;
        const uint32_t above = block_scan(c1 + c0, lds_count, all);
        if (above < left && above + c1 + c0 >= left) {
            const bool upper = above + c1 >= left;
            lds_found[0] = upper ? p1 : p1 - 1u;
            lds_found[1] = upper ? above : above + c1;
            lds_found[2] = upper ? c1 : c0;
        }
        __syncthreads();
        const uint32_t part = lds_found[0];
        left -= lds_found[1];
        agree = lds_found[2];
        lo += part << shift;
        hi = lo + min(hi - lo, (1u << shift) - 1u);         // (the last part may reach past the largest number there is)
        __syncthreads();
    }
    uint32_t border = lo;                                  // with left == agree all from lo on stay, with lo == hi the first `left` of them
    if (lo < hi && left < agree) {
        each([&](uint32_t k) {
            if (k >= lo && k <= hi) lds_few[atomicAdd(&lds_n, 1u)] = k;          // (in any order: they are only counted)
        });
        if (tid < 4u) lds_few[agree + tid] = 0u;
        __syncthreads();
        static_assert(4u * FEW == SELECT_THREADS, "four threads a token");
        const uint32_t own = lds_few[min(tid / 4u, agree)];
        uint32_t over = 0u, same = 0u;
#pragma unroll 4
        for (uint32_t i = 4u * (tid & 3u); i < agree; i += 16u) {
            const tq_u4 x = *reinterpret_cast<const tq_u4 *>(lds_few + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) { over += x[k] > own ? 1u : 0u; same += x[k] == own ? 1u : 0u; }
        }
#pragma unroll
        for (int i = 1; i < 4; i <<= 1) { over += (uint32_t)__shfl_xor(over, i); same += (uint32_t)__shfl_xor(same, i); }
        if (tid / 4u < agree && over < left && over + same >= left) { lds_found[0] = own; lds_found[1] = over; lds_found[2] = same; }        // (its equals say the same)
        __syncthreads();
        border = lds_found[0];
        left -= lds_found[1];
        agree = lds_found[2];
    }
    // ---- places
    TQ_GLOBAL long long *kept = (TQ_GLOBAL long long *)a.kept + (long long)row * a.keep;
    auto before_lane = [&](unsigned long long m) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u)); };
    auto scan = [&]() {                                    // lds_place, [register][wave]: counts -> sums of those before
        __syncthreads();
        uint32_t all;
        const uint32_t v = tid < E * WAVES ? lds_place[tid] : 0u, x = block_scan(v, lds_count, all);
        if (tid < E * WAVES) lds_place[tid] = x;
        __syncthreads();
    };
    static_assert(E * WAVES <= SELECT_THREADS, "a count a thread");
    if (left < agree) {                                    // of the tokens equal to the border only the first `left` stay: the others become none
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t c = (uint32_t)__popcll(__ballot(key[e] == border));
            if (lane == 0u) lds_place[e * WAVES + wave] = c;
        }
        scan();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool same = key[e] == border;
            const uint32_t rank = lds_place[e * WAVES + wave] + before_lane(__ballot(same));
            if (same && rank >= left) key[e] = 0u;
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t c = (uint32_t)__popcll(__ballot(key[e] >= border));
        if (lane == 0u) lds_place[e * WAVES + wave] = c;
    }
    scan();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const bool stays = key[e] >= border;
        const uint32_t at = lds_place[e * WAVES + wave] + before_lane(__ballot(stays));
        if (stays) kept[at] = e * SELECT_THREADS + tid;
    }
}

// ---- rows of more than 32768 tokens -----------------------------------------------------------------------------------------
// Block (row, segment of its tokens); three launches that count the 2048 values of the next eleven bits (ten at last) among the segment's tokens that
// agree with the border so far, and one that writes places. Each begins with what the counts before it say: the border's next digit, and how many tokens of the segments before
// its own lie above it (a thread adds two digits over all segments). Counts are whole numbers and every block finds the same border: nothing depends on an order.
// The call: 8 rows of 131072 tokens 63 us (a block a row, its weights read again for every pass: 133), one of 2^20 82 (794), 8 of 40000 42 (61); up to 32768 tokens the kernel above is
// the faster one (8 of 32768 29 us).  Bound by the chain of five launches, and for many rows by the bytes that are moved.
constexpr uint32_t LONG_DIGITS = 2048, LONG_SEGMENTS = 64, LONG_SEGMENT = 16384, LONG_AHEAD = 16;      // LONG_AHEAD: loads of a thread under way

struct LongState { uint32_t prefix, left, agree, before; };        // border's bits so far, tokens that stay of the `agree` that have them, tokens above it in the segments before

__device__ __forceinline__ uint32_t long_digit(uint32_t key, int round) { return round == 0 ? key >> 21 : round == 1 ? (key >> 10) & 2047u : key & 1023u; }

// What round's counts say; equal: of the segments before, tokens that have the border's bits
__device__ __forceinline__ LongState long_settle(const EvictArgs &a, int round, LongState was, uint32_t row, uint32_t segment, uint32_t *lds, uint32_t *lds_found, uint32_t &equal) {
    const uint32_t tid = threadIdx.x, p1 = LONG_DIGITS - 1u - 2u * tid;
    const TQ_GLOBAL uint32_t *counts = (const TQ_GLOBAL uint32_t *)a.scratch + ((size_t)row * 3u + round) * a.segments * LONG_DIGITS + (p1 - 1u);
    uint32_t c0 = 0u, c1 = 0u, b0 = 0u, b1 = 0u;
#pragma unroll 8
    for (uint32_t s = 0; s < a.segments; ++s) {
        const uint32_t x0 = counts[s * LONG_DIGITS], x1 = counts[s * LONG_DIGITS + 1u];
        c0 += x0; c1 += x1;
        b0 += s < segment ? x0 : 0u; b1 += s < segment ? x1 : 0u;
    }
    uint32_t all;
    const uint32_t above = block_scan(c1 + c0, lds, all), before = block_scan(b1 + b0, lds, all);
    if (above < was.left && above + c1 + c0 >= was.left) {
        const bool upper = above + c1 >= was.left;
        lds_found[0] = upper ? p1 : p1 - 1u;
        lds_found[1] = upper ? above : above + c1;
        lds_found[2] = upper ? c1 : c0;
        lds_found[3] = upper ? before : before + b1;
        lds_found[4] = upper ? b1 : b0;
    }
    __syncthreads();
    equal = lds_found[4];
    return LongState{round == 0 ? lds_found[0] : (was.prefix << (round == 1 ? 11 : 10)) | lds_found[0], was.left - lds_found[1], lds_found[2], was.before + lds_found[3]};
}

__device__ __forceinline__ TQ_GLOBAL uint32_t *long_state(const EvictArgs &a, uint32_t row, uint32_t segment) {
    return (TQ_GLOBAL uint32_t *)a.scratch + (size_t)a.rows * 3u * a.segments * LONG_DIGITS + ((size_t)row * a.segments + segment) * 4u;
}

template <int ROUND>
__device__ __forceinline__ LongState long_now(const EvictArgs &a, uint32_t row, uint32_t segment, uint32_t *lds, uint32_t *lds_found, uint32_t &equal) {
    LongState was = {0u, a.keep, a.tokens, 0u};
    equal = 0u;
    if constexpr (ROUND > 0) {
        const TQ_GLOBAL uint32_t *state = long_state(a, row, segment);
        if constexpr (ROUND > 1) was = LongState{state[0], state[1], state[2], state[3]};
        was = long_settle(a, ROUND - 1, was, row, segment, lds, lds_found, equal);
    }
    return was;
}

template <int ROUND>
__global__ __launch_bounds__(SELECT_THREADS) void tq_evict_count_kernel(EvictArgs a) {
    __shared__ uint32_t lds_part[LONG_DIGITS], lds_scan[SELECT_THREADS / 64], lds_found[5];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, row = blockIdx.x / a.segments, segment = blockIdx.x - row * a.segments;
    const uint32_t begin = segment * a.segment_tokens, end = min(a.tokens, begin + a.segment_tokens);
    lds_part[tid] = lds_part[tid + SELECT_THREADS] = 0u;
    uint32_t equal;
    const LongState now = long_now<ROUND>(a, row, segment, lds_scan, lds_found, equal);
    if (ROUND > 0 && tid == 0u) {
        TQ_GLOBAL uint32_t *state = long_state(a, row, segment);
        state[0] = now.prefix; state[1] = now.left; state[2] = now.agree; state[3] = now.before;
    }
    __syncthreads();
    const TQ_GLOBAL float *w = (const TQ_GLOBAL float *)a.weights + (long long)row * a.w_stride;
    for (uint32_t i0 = begin; i0 < end; i0 += LONG_AHEAD * SELECT_THREADS) {
        float v[LONG_AHEAD];
#pragma unroll
        for (uint32_t k = 0; k < LONG_AHEAD; ++k) v[k] = w[min(i0 + k * SELECT_THREADS + tid, a.tokens - 1u)];
#pragma unroll
        for (uint32_t k = 0; k < LONG_AHEAD; ++k) {
            const uint32_t key = order_of(v[k]), digit = long_digit(key, ROUND);
            const bool counts = i0 + k * SELECT_THREADS + tid < end && (ROUND == 0 || key >> (ROUND == 1 ? 21 : 10) == now.prefix);
            const unsigned long long who = __ballot(counts);
            if (!who) continue;
            const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)digit, (int)__builtin_ctzll(who));
            if (__ballot(counts && digit == first) == who) {                       // (one value for all, as of tokens that have received nothing: no 64 additions to one place)
                if (lane == 0u) atomicAdd(&lds_part[first], (uint32_t)__popcll(who));
            } else if (counts) atomicAdd(&lds_part[digit], 1u);
        }
    }
    __syncthreads();
    TQ_GLOBAL uint32_t *out = (TQ_GLOBAL uint32_t *)a.scratch + (((size_t)row * 3u + ROUND) * a.segments + segment) * LONG_DIGITS;
    out[tid] = lds_part[tid];
    out[tid + SELECT_THREADS] = lds_part[tid + SELECT_THREADS];
}

// A sixteenth of the segment a wave: counted, then written
__global__ __launch_bounds__(SELECT_THREADS) void tq_evict_place_kernel(EvictArgs a) {
    constexpr uint32_t WAVES = SELECT_THREADS / 64;
    __shared__ uint32_t lds_scan[WAVES], lds_found[5], lds_more[2][WAVES];
    const uint32_t lane = threadIdx.x & 63u, wave = tq_uniform32(threadIdx.x >> 6), row = blockIdx.x / a.segments, segment = blockIdx.x - row * a.segments;
    uint32_t equal;
    const LongState now = long_now<3>(a, row, segment, lds_scan, lds_found, equal);
    const uint32_t border = now.prefix;
    const uint32_t first = segment * a.segment_tokens, last = min(a.tokens, first + a.segment_tokens), part = a.segment_tokens / WAVES;
    const uint32_t begin = min(last, first + wave * part), end = min(last, begin + part);
    const TQ_GLOBAL float *w = (const TQ_GLOBAL float *)a.weights + (long long)row * a.w_stride;
    TQ_GLOBAL long long *kept = (TQ_GLOBAL long long *)a.kept + (long long)row * a.keep;
    auto before_lane = [&](unsigned long long m) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u)); };
    auto tokens = [&](auto f) __attribute__((always_inline)) {               // f(token of this lane, key) of 64 at a time, in order
        for (uint32_t i0 = begin; i0 < end; i0 += LONG_AHEAD * 64u) {
            float v[LONG_AHEAD];
#pragma unroll
            for (uint32_t k = 0; k < LONG_AHEAD; ++k) v[k] = w[min(i0 + k * 64u + lane, a.tokens - 1u)];
#pragma unroll
            for (uint32_t k = 0; k < LONG_AHEAD; ++k) f(i0 + k * 64u + lane, i0 + k * 64u + lane < end ? order_of(v[k]) : 0u);
        }
    };
    uint32_t more = 0u, same = 0u;
    tokens([&](uint32_t, uint32_t k) {
        more += (uint32_t)__popcll(__ballot(k > border));
        same += (uint32_t)__popcll(__ballot(k == border));
    });
    if (lane == 0u) { lds_more[0][wave] = more; lds_more[1][wave] = same; }
    __syncthreads();
    uint32_t out = now.before;
#pragma unroll
    for (uint32_t k = 0; k < WAVES; ++k)
        if (k < wave) { out += lds_more[0][k]; equal += lds_more[1][k]; }
    out += min(equal, now.left);                            // (of those equal to the border the first `left` stay)
    tokens([&](uint32_t i, uint32_t k) {
        const unsigned long long equals = __ballot(k == border);
        const bool stays = k > border || (k == border && equal + before_lane(equals) < now.left);
        const unsigned long long staying = __ballot(stays);
        if (stays) kept[out + before_lane(staying)] = i;
        equal += (uint32_t)__popcll(equals);
        out += (uint32_t)__popcll(staying);
    });
}

long long long_segments(long long tokens) {
    const long long n = (tokens + LONG_SEGMENT - 1) / LONG_SEGMENT;
    return n < (long long)LONG_SEGMENTS ? n : (long long)LONG_SEGMENTS;
}

template <typename T>
__device__ __forceinline__ void move_codes(const uint8_t *src, uint8_t *dst, uint32_t bytes, uint32_t first, uint32_t step) {
    for (uint32_t i = first * sizeof(T); i < bytes; i += step * sizeof(T)) *reinterpret_cast<T *>(dst + i) = *reinterpret_cast<const T *>(src + i);
}

// Eight lanes a token: 8 rows of 16384 kept 9 us, 128 of 4097 (64 and 32 bytes of codes) 31 us, 118 MB read and written at 3.8 TB/s.
__global__ __launch_bounds__(256) void tq_evict_move_kernel(EvictArgs a, uint32_t blocks) {
    const uint32_t row = blockIdx.x / blocks, j = (blockIdx.x - row * blocks) * 32u + threadIdx.x / 8u, part = threadIdx.x & 7u;
    if (j >= a.keep + a.rest) return;
    const float *w = a.weights + (long long)row * a.w_stride;
    float *w_out = a.weights_out + (long long)row * a.w_out_stride;
    if (j >= a.keep) {
        if (part == 0u) w_out[j] = w[a.tokens + (j - a.keep)];
        return;
    }
    const uint32_t from = (uint32_t)a.kept[(long long)row * a.keep + j];
    const size_t src = (size_t)row * a.row_stride + from, dst = (size_t)row * a.out_stride + j;
    if (part == 0u) w_out[j] = w[from];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (part == (uint32_t)s) a.norms_out[s][dst] = a.norms[s][src];
        const uint8_t *p = a.idx[s] + src * a.bytes[s];
        uint8_t *q = a.idx_out[s] + dst * a.bytes[s];
        if (a.unit[s] == 16u) move_codes<tq_u4>(p, q, a.bytes[s], part, 8u);
        else if (a.unit[s] == 4u) move_codes<uint32_t>(p, q, a.bytes[s], part, 8u);
        else move_codes<uint8_t>(p, q, a.bytes[s], part, 8u);
    }
}

}  // namespace

extern "C" long long tq_evict_scratch(long long rows, long long tokens) {
    if (rows < 0 || rows > 0x7fffffff || tokens < 0 || tokens > 0x7fffffff - 65536) return TQ_ERR_SIZE;
    return tokens <= 32 * SELECT_THREADS ? 0 : rows * long_segments(tokens) * (3 * (long long)LONG_DIGITS + 4);
}

extern "C" int tq_evict(const tq_packed_store *from, const tq_packed_store *to, const float *weights, long long weights_stride, float *weights_out,
                        long long weights_out_stride, long long rest, long long rows, long long tokens, long long keep, int head_dim, int bits_k, int bits_v, long long *kept, uint32_t *scratch,
                        long long scratch_words, void *stream) {
    if (!from || !to) return TQ_ERR_NULL;
    if (bits_k < 1 || bits_k > 8 || bits_v < 1 || bits_v > 8) return TQ_ERR_BITS;
    if (head_dim < TQ_ANYDIM_MIN || head_dim > TQ_ANYDIM_MAX) return TQ_ERR_HEAD_DIM;
    const long long most = 0x7fffffff;
    if (rows < 0 || rows > most || tokens < 0 || tokens > most - 65536 || keep < 0 || keep > tokens || rest < 0 || rest > 65536) return TQ_ERR_SIZE;
    if (from->packed_row_stride < 0 || to->packed_row_stride < 0 || from->packed_row_stride > most || to->packed_row_stride > most) return TQ_ERR_SIZE;
    const long long src = from->packed_row_stride ? from->packed_row_stride : tokens, dst = to->packed_row_stride ? to->packed_row_stride : keep;
    if (rows > 1 && (src < tokens || dst < keep || weights_stride < tokens + rest || weights_out_stride < keep + rest)) return TQ_ERR_SIZE;
    const long long blocks = (keep + rest + 31) / 32;
    if (rows == 0 || blocks == 0) return TQ_OK;
    if (blocks > most / rows) return TQ_ERR_SIZE;
    if (!weights || !weights_out) return TQ_ERR_NULL;
    if (keep && (!kept || !from->k_idx || !from->k_norms || !from->v_idx || !from->v_norms || !to->k_idx || !to->k_norms || !to->v_idx || !to->v_norms)) return TQ_ERR_NULL;
    if (((uintptr_t)weights & 3u) || ((uintptr_t)weights_out & 3u) || ((uintptr_t)kept & 7u) ||
        (((uintptr_t)from->k_norms | (uintptr_t)from->v_norms | (uintptr_t)to->k_norms | (uintptr_t)to->v_norms) & 1u))
        return TQ_ERR_ALIGN;
    const long long words = keep ? tq_evict_scratch(rows, tokens) : 0;
    if (words && !scratch) return TQ_ERR_NULL;
    if ((uintptr_t)scratch & 3u) return TQ_ERR_ALIGN;
    if (scratch_words < words) return TQ_ERR_CAPACITY;
    EvictArgs a{};
    a.weights = weights; a.weights_out = weights_out; a.kept = kept;
    a.idx[0] = from->k_idx; a.idx[1] = from->v_idx; a.norms[0] = from->k_norms; a.norms[1] = from->v_norms;
    a.idx_out[0] = to->k_idx; a.idx_out[1] = to->v_idx; a.norms_out[0] = to->k_norms; a.norms_out[1] = to->v_norms;
    a.w_stride = weights_stride; a.w_out_stride = weights_out_stride; a.row_stride = src; a.out_stride = dst;
    a.rows = (uint32_t)rows; a.tokens = (uint32_t)tokens; a.keep = (uint32_t)keep; a.rest = (uint32_t)rest;
    for (int s = 0; s < 2; ++s) {
        a.bytes[s] = (uint32_t)tq_bytes_per_vector(head_dim, s ? bits_v : bits_k);
        const uintptr_t low = (uintptr_t)a.idx[s] | (uintptr_t)a.idx_out[s] | a.bytes[s];
        a.unit[s] = !(low & 15u) ? 16u : !(low & 3u) ? 4u : 1u;
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (keep) {
        const dim3 g((unsigned)rows), t(SELECT_THREADS);
        if (tokens <= SELECT_THREADS) hipLaunchKernelGGL((tq_evict_select_kernel<1>), g, t, 0, st, a);
        else if (tokens <= 4 * SELECT_THREADS) hipLaunchKernelGGL((tq_evict_select_kernel<4>), g, t, 0, st, a);
        else if (tokens <= 16 * SELECT_THREADS) hipLaunchKernelGGL((tq_evict_select_kernel<16>), g, t, 0, st, a);
        else if (tokens <= 32 * SELECT_THREADS) hipLaunchKernelGGL((tq_evict_select_kernel<32>), g, t, 0, st, a);
        else {
            a.scratch = scratch;
            a.segment_tokens = (uint32_t)(((tokens + long_segments(tokens) - 1) / long_segments(tokens) + SELECT_THREADS - 1) / SELECT_THREADS * SELECT_THREADS);
            a.segments = (uint32_t)long_segments(tokens);
            const dim3 blocks_of_segments((unsigned)(rows * a.segments));
            hipLaunchKernelGGL((tq_evict_count_kernel<0>), blocks_of_segments, t, 0, st, a);
            hipLaunchKernelGGL((tq_evict_count_kernel<1>), blocks_of_segments, t, 0, st, a);
            hipLaunchKernelGGL((tq_evict_count_kernel<2>), blocks_of_segments, t, 0, st, a);
            hipLaunchKernelGGL(tq_evict_place_kernel, blocks_of_segments, t, 0, st, a);
        }
    }
    hipLaunchKernelGGL(tq_evict_move_kernel, dim3((unsigned)(rows * blocks)), dim3(256), 0, st, a, (uint32_t)blocks);
    return (int)hipGetLastError();
}
