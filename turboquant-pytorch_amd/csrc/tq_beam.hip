// Beam search's choice: of beams x vocabulary the continuations with the largest summed log probability, tq_beam_select.
//
// sum(k, v) = score_k + logit_kv - log sum_v exp(logit_kv).  Within a beam sums have the order of the logits, so that a part of a row can name its `best` largest logits
// before the row's sum of exponentials is known.  Two launches: parts of rows (their largest logits, and largest and sum of exponentials), each logit read once and held in
// registers; then a block a sequence joins the sums in 64 bits and chooses.
#include "tq_device.h"

namespace {

constexpr int PART_THREADS = 512, JOIN_THREADS = 1024;
constexpr int BEST_MAX = 64;
constexpr uint32_t PART_HELD = 512, JOIN_HELD = 1024;        // candidates that pass the threshold and are ranked by comparing all

struct BeamArgs {
    const uint8_t *logits;
    const float *scores;             // [batch, beams]
    long long batch_stride, beam_stride, score_stride;       // elements
    float *stat;                     // [rows][parts][2]: largest logit, sum of exponentials against it
    float *cand;                     // [rows][parts][best] logits
    uint32_t *cand_token;            // the same: their tokens, NO_TOKEN where a part has fewer
    float *values;                   // [batch, best]
    long long *tokens, *parents;
    uint32_t beams, vocab, best, parts;
};
constexpr uint32_t NO_TOKEN = 0xffffffffu;

// Floats as whole numbers of the same order, above zero, which stands for none; the two zeros are equal.
__device__ __forceinline__ uint32_t beam_order(float x) {
    uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The n-th largest of a wave's values (0 where fewer lanes have one): bits from the top, until exactly n are left.
__device__ __forceinline__ uint32_t nth_of_wave(uint32_t key, uint32_t n) {
    uint32_t t = 0u;
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t with = t | (1u << bit);
        const uint32_t count = (uint32_t)__popcll(__ballot(key >= with));
        if (count >= n) t = with;
        if (count == n) break;
    }
    return t;
}

template <typename T>
__device__ __forceinline__ T wave_max(T x) {
#pragma unroll
    for (int i = 32; i; i >>= 1) { const T y = __shfl_xor(x, i); x = y > x ? y : x; }
    return x;
}

// Part of a row: E logits a thread, sixteen bytes at a time.  Thresholds first: a wave's n-th largest of its lanes' largest has n values at or above it, so what lies
// below the largest of the waves' thresholds is out; of random logits one to three times `best` are left, which are ranked by comparing all.  Where ties leave more
// than fit (equal logits), the block takes the largest `best` times over.
template <int DT, int E>
__global__ __launch_bounds__(PART_THREADS) void tq_beam_part_kernel(BeamArgs a) {
    constexpr int ES = DT == TQ_F32 ? 4 : 2, V = 16 / ES, LOADS = E / V, WAVES = PART_THREADS / 64;
    __shared__ float lds_x[PART_HELD];
    __shared__ uint32_t lds_i[PART_HELD];
    __shared__ float lds_m[WAVES], lds_s[WAVES];
    __shared__ uint32_t lds_t[WAVES], lds_n;
    __shared__ unsigned long long lds_best[WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts, b = row / a.beams, k = row - b * a.beams;
    const uint8_t *src = a.logits + ((long long)b * a.batch_stride + (long long)k * a.beam_stride) * ES;
    const uint32_t first = part * (PART_THREADS * E);
    const bool aligned = !((uintptr_t)src & 15u);
    float x[E];
    const float none = -__builtin_inff();
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
        const uint32_t at = first + (l * PART_THREADS + tid) * V;
        if (aligned && at + V <= a.vocab) {
            const tq_u4 v = tq_gload16(src + (size_t)at * ES);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (DT == TQ_F32) x[l * V + e] = __uint_as_float(v[e]);
                else {
                    const uint32_t h = e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xffffu;
                    x[l * V + e] = DT == TQ_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __uint_as_float(h << 16);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float y = none;
                if (at + e < a.vocab) {
                    const uint8_t *p = src + (size_t)(at + e) * ES;
                    if constexpr (DT == TQ_F32) y = *reinterpret_cast<const TQ_GLOBAL float *>((const TQ_GLOBAL uint8_t *)p);
                    else {
                        const uint16_t h = *reinterpret_cast<const TQ_GLOBAL uint16_t *>((const TQ_GLOBAL uint8_t *)p);
                        y = DT == TQ_F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
                    }
                }
                x[l * V + e] = y;
            }
        }
    }
    auto token_of = [&](int i) { return first + ((i / V) * PART_THREADS + tid) * V + i % V; };
    if (tid == 0u) lds_n = 0u;
    float top = x[0];
#pragma unroll
    for (int i = 1; i < E; ++i) top = fmaxf(top, x[i]);
    const uint32_t t = nth_of_wave(token_of(0) < a.vocab ? beam_order(top) : 0u, a.best);
    const float m = wave_max(top);
    float sum = 0.f;
    const float ref = m == none ? 0.f : m;
#pragma unroll
    for (int i = 0; i < E; ++i) sum += __builtin_amdgcn_exp2f((x[i] - ref) * 1.44269504088896340736f);
#pragma unroll
    for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
    if (lane == 0u) {
        lds_t[wave] = t;
        lds_m[wave] = m;
        lds_s[wave] = sum;
    }
    __syncthreads();
    uint32_t least = 0u;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) least = max(least, lds_t[w]);
    if (tid == 0u) {
        float largest = lds_m[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) largest = fmaxf(largest, lds_m[w]);
        float all = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) all += lds_s[w] * (lds_m[w] == none ? (lds_s[w] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f((lds_m[w] - largest) * 1.44269504088896340736f));
        float *stat = a.stat + 2u * (size_t)blockIdx.x;
        stat[0] = largest;
        stat[1] = all;
    }
    // ---- what passes
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint32_t token = token_of(i);
        const bool in = token < a.vocab && beam_order(x[i]) >= least;
        if (__any(in)) {
            if (in) {
                const uint32_t at = atomicAdd(&lds_n, 1u);
                if (at < PART_HELD) { lds_x[at] = x[i]; lds_i[at] = token; }
            }
        }
    }
    __syncthreads();
    const uint32_t n = lds_n;
    float *cand = a.cand + (size_t)blockIdx.x * a.best;
    uint32_t *cand_token = a.cand_token + (size_t)blockIdx.x * a.best;
    if (n <= PART_HELD) {
        for (uint32_t i = tid; i < n; i += PART_THREADS) {
            const uint32_t key = beam_order(lds_x[i]), token = lds_i[i];
            uint32_t rank = 0u;
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t other = beam_order(lds_x[j]);
                rank += (other > key || (other == key && lds_i[j] < token)) ? 1u : 0u;
            }
            if (rank < a.best) { cand[rank] = lds_x[i]; cand_token[rank] = token; }
        }
        if (tid >= n && tid < a.best) cand_token[tid] = NO_TOKEN;
        return;
    }
    unsigned long long last = ~0ull;         // order and token of the one taken last, as one number that falls
#pragma unroll 1
    for (uint32_t r = 0; r < a.best; ++r) {
        unsigned long long mine = 0ull;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const uint32_t token = token_of(i);
            const unsigned long long u = token < a.vocab ? ((unsigned long long)beam_order(x[i]) << 32) | (uint32_t)~token : 0ull;
            if (u < last && u > mine) mine = u;
        }
        mine = wave_max(mine);
        if (lane == 0u) lds_best[wave] = mine;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mine = lds_best[w] > mine ? lds_best[w] : mine;
        __syncthreads();
        last = mine;
        if (tid == 0u) {
            const uint32_t key = (uint32_t)(mine >> 32);
            cand[r] = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
            cand_token[r] = mine ? ~(uint32_t)mine : NO_TOKEN;
        }
    }
}

struct Choice {
    double sum;
    uint32_t at;             // beam * vocab + token
};
__device__ __forceinline__ bool before(const Choice &x, const Choice &y) { return x.sum > y.sum || (x.sum == y.sum && x.at < y.at); }

// Block = sequence.  Sums in 64 bits: log probabilities of different beams meet here, and 32 would make ties of what is none.  A beam whose log probabilities are no numbers (a NaN or
// an infinity among logits or scores) counts with sums of -infinity.  Thresholds as above, on sums rounded to 32 bits (which keeps their order), twice: of all candidates, and of
// those that passed; what is left is ranked by comparing all in 64 bits.
__global__ __launch_bounds__(JOIN_THREADS) void tq_beam_join_kernel(BeamArgs a) {
    constexpr int WAVES = JOIN_THREADS / 64;
    extern __shared__ double lds_base[];                     // [beams] score - log of the sum of exponentials
    __shared__ Choice lds_c[JOIN_HELD];
    __shared__ uint32_t lds_t[WAVES], lds_n[2];
    __shared__ Choice lds_best[WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, b = blockIdx.x, slots = a.parts * a.best, all = a.beams * slots;
    const size_t row0 = (size_t)b * a.beams;
    if (tid < 2u) lds_n[tid] = 0u;
    for (uint32_t k = wave; k < a.beams; k += WAVES) {
        const float *stat = a.stat + 2u * (row0 + k) * a.parts;
        float m = -__builtin_inff();
        for (uint32_t p = lane; p < a.parts; p += 64u) m = fmaxf(m, stat[2u * p]);
        m = wave_max(m);
        double s = 0.0;
        for (uint32_t p = lane; p < a.parts; p += 64u)
            if (stat[2u * p + 1u] != 0.f) s += (double)stat[2u * p + 1u] * exp((double)stat[2u * p] - (double)m);
#pragma unroll
        for (int i = 32; i; i >>= 1) s += __shfl_xor(s, i);
        if (lane == 0u) lds_base[k] = (double)a.scores[(long long)b * a.score_stride + k] - ((double)m + log(s));
    }
    __syncthreads();
    // Candidate i: none (false), or its sum
    auto candidate = [&](uint32_t i, Choice &c) {
        const uint32_t k = i / slots, slot = i - k * slots;
        const double base = lds_base[k];
        if (!(fabs(base) < __builtin_inf())) {               // (its first tokens, as among equals)
            c.sum = -__builtin_inf();
            c.at = k * a.vocab + slot;
            return slot < a.best && slot < a.vocab;
        }
        const uint32_t token = a.cand_token[row0 * slots + i];
        c.sum = base + (double)a.cand[row0 * slots + i];
        c.at = k * a.vocab + token;
        return token != NO_TOKEN;
    };
    uint32_t most = 0u;
    for (uint32_t i = tid; i < all; i += JOIN_THREADS) {
        Choice c;
        if (candidate(i, c)) most = max(most, beam_order((float)c.sum));
    }
    uint32_t t = nth_of_wave(most, a.best);
    if (lane == 0u) lds_t[wave] = t;
    __syncthreads();
    uint32_t least = 1u;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) least = max(least, lds_t[w]);
    for (uint32_t i = tid; i < all; i += JOIN_THREADS) {
        Choice c;
        if (candidate(i, c) && beam_order((float)c.sum) >= least) {
            const uint32_t at = atomicAdd(&lds_n[0], 1u);
            if (at < JOIN_HELD) lds_c[at] = c;
        }
    }
    __syncthreads();
    uint32_t n = lds_n[0];
    auto put = [&](uint32_t r, const Choice &c) {
        const size_t at = (size_t)b * a.best + r;
        a.values[at] = (float)c.sum;
        a.tokens[at] = c.at % a.vocab;
        a.parents[at] = c.at / a.vocab;
    };
    if (n <= JOIN_HELD) {
        Choice c = {0.0, 0u};
        if (tid < n) c = lds_c[tid];
        t = nth_of_wave(tid < n ? beam_order((float)c.sum) : 0u, a.best);
        if (lane == 0u) lds_t[wave] = t;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) least = max(least, lds_t[w]);
        const bool in = tid < n && beam_order((float)c.sum) >= least;
        if (in) lds_c[atomicAdd(&lds_n[1], 1u)] = c;
        __syncthreads();
        n = lds_n[1];
        if (tid < n) {
            c = lds_c[tid];
            uint32_t rank = 0u;
            for (uint32_t j = 0; j < n; ++j) rank += before(lds_c[j], c) ? 1u : 0u;
            if (rank < a.best) put(rank, c);
        }
        return;
    }
    // (ties without end: the largest, `best` times over)
    Choice last = {__builtin_inf(), 0u};
    bool any = false;
#pragma unroll 1
    for (uint32_t r = 0; r < a.best; ++r) {
        Choice mine = {-__builtin_inf(), NO_TOKEN};
        for (uint32_t i = tid; i < all; i += JOIN_THREADS) {
            Choice c;
            if (candidate(i, c) && (!any || before(last, c)) && before(c, mine)) mine = c;
        }
#pragma unroll
        for (int i = 32; i; i >>= 1) {
            const Choice other = {__shfl_xor(mine.sum, i), (uint32_t)__shfl_xor((int)mine.at, i)};
            if (before(other, mine)) mine = other;
        }
        if (lane == 0u) lds_best[wave] = mine;
        __syncthreads();
        for (int w = 0; w < WAVES; ++w)
            if (before(lds_best[w], mine)) mine = lds_best[w];
        __syncthreads();
        last = mine;
        any = true;
        if (tid == 0u) put(r, mine);
    }
}

// Logits a thread of the first launch holds: 32, or 8 where that would give fewer blocks than the card has compute units.
int held(long long rows, long long vocab, int cus) { return rows * ((vocab + 32 * PART_THREADS - 1) / (32 * PART_THREADS)) >= cus ? 32 : 8; }

struct BeamPlan {
    int per_thread;
    long long rows, parts, bytes;
};
int beam_plan(long long batch, long long beams, long long vocab, long long best, BeamPlan &p) {
    const long long most = 0x7fffffff;
    if (batch < 0 || beams < 0 || vocab < 0 || best < 0 || batch > most || beams > 1024 || vocab > most || best > BEST_MAX) return TQ_ERR_SIZE;
    if (beams && vocab > most / beams) return TQ_ERR_SIZE;
    if (batch && best > beams * vocab) return TQ_ERR_SIZE;
    int cus = 0;
    if (tq_device_cus(cus)) cus = 256;
    p.rows = batch * beams;
    p.per_thread = held(p.rows, vocab, cus);
    p.parts = (vocab + p.per_thread * PART_THREADS - 1) / (p.per_thread * PART_THREADS);
    if (p.parts && p.rows > most / p.parts) return TQ_ERR_SIZE;
    if (beams && p.parts * beams > most / (best ? best : 1)) return TQ_ERR_SIZE;
    p.bytes = p.rows * p.parts * (8 + 8 * best);
    return TQ_OK;
}

template <int DT>
void launch_parts(const BeamArgs &a, const BeamPlan &p, hipStream_t s) {
    const dim3 g((unsigned)(p.rows * p.parts)), t(PART_THREADS);
    if (p.per_thread == 32) hipLaunchKernelGGL((tq_beam_part_kernel<DT, 32>), g, t, 0, s, a);
    else hipLaunchKernelGGL((tq_beam_part_kernel<DT, 8>), g, t, 0, s, a);
}

}  // namespace

extern "C" long long tq_beam_scratch(long long batch, long long beams, long long vocab, long long best) {
    BeamPlan p;
    const int rc = beam_plan(batch, beams, vocab, best, p);
    return rc ? rc : p.bytes;
}

extern "C" int tq_beam_select(const void *logits, int dtype, long long batch, long long beams, long long vocab, long long batch_stride, long long beam_stride,
                              const float *scores, long long score_stride, long long best, float *values, long long *tokens, long long *parents, void *scratch,
                              long long scratch_bytes, void *stream) {
    if (dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16) return TQ_ERR_DTYPE;
    BeamPlan p;
    const int rc = beam_plan(batch, beams, vocab, best, p);
    if (rc) return rc;
    if (batch == 0 || best == 0) return TQ_OK;
    if (!logits || !scores || !values || !tokens || !parents || !scratch) return TQ_ERR_NULL;
    if (((uintptr_t)logits & (dtype == TQ_F32 ? 3u : 1u)) || ((uintptr_t)scores & 3u) || ((uintptr_t)values & 3u) || (((uintptr_t)tokens | (uintptr_t)parents) & 7u) ||
        ((uintptr_t)scratch & 7u))
        return TQ_ERR_ALIGN;
    if (scratch_bytes < p.bytes) return TQ_ERR_CAPACITY;
    BeamArgs a{};
    a.logits = static_cast<const uint8_t *>(logits);
    a.scores = scores;
    a.batch_stride = batch_stride; a.beam_stride = beam_stride; a.score_stride = score_stride;
    const long long parts = p.rows * p.parts;
    a.stat = static_cast<float *>(scratch);
    a.cand = a.stat + 2 * parts;
    a.cand_token = reinterpret_cast<uint32_t *>(a.cand + parts * best);
    a.values = values; a.tokens = tokens; a.parents = parents;
    a.beams = (uint32_t)beams; a.vocab = (uint32_t)vocab; a.best = (uint32_t)best; a.parts = (uint32_t)p.parts;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == TQ_F32) launch_parts<TQ_F32>(a, p, s);
    else if (dtype == TQ_F16) launch_parts<TQ_F16>(a, p, s);
    else launch_parts<TQ_BF16>(a, p, s);
    hipLaunchKernelGGL(tq_beam_join_kernel, dim3((unsigned)batch), dim3(JOIN_THREADS), (size_t)beams * sizeof(double), s, a);
    return (int)hipGetLastError();
}
