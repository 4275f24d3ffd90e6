// Beam search's choice: of beams x vocabulary the continuations with the largest summed log probability, tq_beam_select.
//
// sum(k, v) = score_k + logit_kv - log sum_v exp(logit_kv).  Within a beam sums have the order of the logits, so that a part of a row can name its `best` largest logits
// before the row's sum of exponentials is known.  Two launches: parts of rows (their largest logits, and largest and sum of exponentials), each logit read once and held in
// registers; then a block a sequence joins the sums in 64 bits and chooses.  (The sums of exponentials are of 32 bits, from lane to row: terms of one sign, so that some 2^-22 of a logarithm is lost.)
#include <type_traits>

#include "tq_lut.h"

namespace {

constexpr int PART_WAVES = 4, JOIN_THREADS = 512;
constexpr int BEST_MAX = 64;
constexpr uint32_t JOIN_HELD = 1024;         // candidates that pass the threshold and are ranked by comparing all

struct BeamArgs {
    const uint8_t *logits;
    const float *scores;             // [batch, beams]
    long long batch_stride, beam_stride, score_stride;       // elements
    float *stat;                     // [rows][parts][2]: largest logit, sum of exponentials against it
    float *cand;                     // [rows][parts][best] logits
    uint32_t *cand_token;            // the same: their tokens, NO_TOKEN where a part has fewer
    float *values;                   // [batch, best]
    long long *tokens, *parents;
    uint32_t rows, beams, vocab, best, parts, chunks;
};
constexpr uint32_t NO_TOKEN = 0xffffffffu;
constexpr float LOG2E_F = 1.44269504088896340736f;

// Sixteen bytes at the address of any element
typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t Halves __attribute__((ext_vector_type(4), aligned(2)));
template <int ES>
__device__ __forceinline__ tq_u4 load_piece(const uint8_t *p) {
    if constexpr (ES == 4) return *reinterpret_cast<const TQ_GLOBAL Words *>((const TQ_GLOBAL uint8_t *)p);
    else return *reinterpret_cast<const TQ_GLOBAL Halves *>((const TQ_GLOBAL uint8_t *)p);
}

// Order of this wave's LDS accesses among its lanes
__device__ __forceinline__ void wave_sync_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

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
__device__ __forceinline__ uint32_t lanes_before(unsigned long long mask) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u)); }

// A wave's candidates in LDS: up to BEST_MAX that were best so far, and up to 64 new ones.
struct BeamList {
    float x[BEST_MAX + 64];
    uint32_t token[BEST_MAX + 64];
};

// The `best` of a list to its front, as they lie (in order they would fill every `best`'th place of the join's first groups alone: 32 of 16 beams x 262144 took 267 us instead of 56); answers
// with the order of the last one.  Of few, each in turn out of its lane's registers against all others (24 cycles a candidate); of more, the n-th largest bit by bit, as above (60 cycles a bit; LOW: bits that the
// logits' type leaves alike), and of those that equal it the ones of the lowest tokens, one by one: 16 x 8 x 128256 float32 logits 32.5 us by the first way alone, 28 with both; 4 x 32000 by the second alone 13.5 for 11.5.
template <int LOW>
__device__ __forceinline__ uint32_t keep_best(BeamList &list, uint32_t &count, uint32_t best, uint32_t lane) {
    wave_sync_lds();
    const uint32_t all = count;
    const float x0 = list.x[lane], x1 = list.x[64u + lane];
    const uint32_t t0 = list.token[lane], t1 = list.token[64u + lane];
    const uint32_t k0 = lane < all ? beam_order(x0) : 0u, k1 = 64u + lane < all ? beam_order(x1) : 0u;
    wave_sync_lds();
    count = min(all, best);
    if (all <= best) return 0u;
    bool in0, in1;
    uint32_t last;
    if (all <= 48u) {
        uint32_t r0 = 0u;
#pragma unroll 4
        for (uint32_t j = 0; j < all; ++j) {
            const uint32_t key = (uint32_t)__builtin_amdgcn_readlane((int)k0, (int)j), token = (uint32_t)__builtin_amdgcn_readlane((int)t0, (int)j);
            r0 += key > k0 || (key == k0 && token < t0) ? 1u : 0u;
        }
        in0 = lane < all && r0 < best;
        in1 = false;
        last = (uint32_t)__builtin_amdgcn_readlane((int)k0, __builtin_ctzll(__ballot(in0 && r0 + 1u == best)));
    } else {
        uint32_t left = all;             // at or above `last`
        last = 0u;
#pragma unroll 1
        for (int bit = 31; bit >= LOW && left != best; --bit) {
            const uint32_t with = last | (1u << bit), n = (uint32_t)__popcll(__ballot(k0 >= with)) + (uint32_t)__popcll(__ballot(k1 >= with));
            if (n >= best) { last = with; left = n; }
        }
        in0 = k0 >= last;
        in1 = k1 >= last;
        if (left != best) {              // equal ones: those of them that come last are out
            const uint32_t top = (LOW ? (1u << LOW) - 1u : 0u) | last;
#pragma unroll 1
            for (; left > best; --left) {
                const uint32_t most = wave_max(max(in0 && k0 <= top ? t0 : 0u, in1 && k1 <= top ? t1 : 0u));
                if (in0 && k0 <= top && t0 == most) in0 = false;
                else if (in1 && k1 <= top && t1 == most) in1 = false;
            }
        }
    }
    const unsigned long long m0 = __ballot(in0), m1 = __ballot(in1);
    const uint32_t to0 = lanes_before(m0), to1 = (uint32_t)__popcll(m0) + lanes_before(m1);
    if (in0) { list.x[to0] = x0; list.token[to0] = t0; }
    if (in1) { list.x[to1] = x1; list.token[to1] = t1; }
    wave_sync_lds();
    return last;
}

// Wave = part of a row, in chunks of 64 E logits that lie in registers, sixteen bytes a load, the next chunk's on their way meanwhile.  The n-th largest of the lanes' largest has n
// values at or above it, so what lies below it (and, later on, not above the n-th largest so far) is out; what is left is ranked by comparing all, each in turn out of its lane's registers.
// Where ties leave more than fit (equal logits), the best of a chunk are taken one by one.
template <int DT, int E>
__global__ __launch_bounds__(64 * PART_WAVES) void tq_beam_part_kernel(BeamArgs a) {
    constexpr int ES = DT == TQ_F32 ? 4 : 2, V = 16 / ES, LOADS = E / V, LOW = DT == TQ_F32 ? 0 : DT == TQ_F16 ? 13 : 16;
    constexpr uint32_t CHUNK = 64u * E;
    __shared__ BeamList lists[PART_WAVES];
    const uint32_t lane = threadIdx.x & 63u, wave = tq_uniform32(threadIdx.x >> 6), at = blockIdx.x * PART_WAVES + wave;
    if (at >= a.rows * a.parts) return;
    const uint32_t row = at / a.parts, part = at - row * a.parts, b = row / a.beams, k = row - b * a.beams;
    const uint8_t *src = a.logits + ((long long)b * a.batch_stride + (long long)k * a.beam_stride) * ES;
    // Every chunk but the row's last one is whole pieces of 16 bytes, wherever in memory the row begins: which lane adds an exponential depends on its token alone, so that equal logits have
    // equal sums, bit for bit.  The last chunk goes element by element, neighbours in neighbouring lanes.
    const uint32_t stop = a.vocab, begin = part * (a.chunks * CHUNK), end = min(stop, begin + a.chunks * CHUNK);
    BeamList &list = lists[wave];
    const float none = -__builtin_inff();
    tq_u4 raw[LOADS];
    auto is_whole = [&](uint32_t first) { return first + CHUNK <= stop; };
    auto load = [&](uint32_t first) __attribute__((always_inline)) {
        if (is_whole(first)) {
#pragma unroll
            for (int l = 0; l < LOADS; ++l) raw[l] = load_piece<ES>(src + (size_t)(first + (l * 64u + lane) * V) * ES);
            return;
        }
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                if constexpr (DT == TQ_F32) {
                    const uint32_t p = first + (4 * l + d) * 64u + lane;
                    raw[l][d] = p < stop ? tq_gload4(src + (size_t)p * 4u) : 0xff800000u;
                } else {
                    const uint32_t none16 = DT == TQ_F16 ? 0xfc00u : 0xff80u, p = first + (8 * l + 2 * d) * 64u + lane, q = p + 64u;
                    const uint16_t *h = reinterpret_cast<const uint16_t *>(src);
                    raw[l][d] = (p < stop ? (uint32_t)tq_gload2(h + p) : none16) | ((q < stop ? (uint32_t)tq_gload2(h + q) : none16) << 16);
                }
            }
        }
    };
    if (begin < end) load(begin);
    uint32_t count = 0u, bound = 0u;         // candidates held; at least `best` of this part so far are of this order or above (0: not known)
    float m = none, sum = 0.f;               // this lane's sum of exponentials against the wave's largest
#pragma unroll 1
    for (uint32_t first = begin; first < end; first += CHUNK) {
        float x[E];
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (DT == TQ_F32) x[l * V + e] = __uint_as_float(raw[l][e]);
                else {
                    const uint32_t h = e & 1 ? raw[l][e / 2] >> 16 : raw[l][e / 2] & 0xffffu;
                    x[l * V + e] = DT == TQ_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __uint_as_float(h << 16);
                }
            }
        if (first + CHUNK < end) load(first + CHUNK);
        const bool whole = is_whole(first);
        auto place_of = [&](int i) { return first + (whole ? ((i / V) * 64u + lane) * V + i % V : 64u * i + lane); };
        auto is_token = [&](int i) { return whole || place_of(i) < stop; };
        float top = x[0];
#pragma unroll
        for (int i = 1; i < E; ++i) top = fmaxf(top, x[i]);
        const float largest = fmaxf(m, reduce_wave(top, OpMax()));
        const float ref = largest == none ? 0.f : largest;
        sum *= __builtin_amdgcn_exp2f((m - ref) * LOG2E_F);
        m = largest;
#pragma unroll
        for (int i = 0; i < E; ++i) sum += __builtin_amdgcn_exp2f((x[i] - ref) * LOG2E_F);
        // ---- what passes: above the bound so far (an equal one of later tokens comes after those it is made of); at first, or where that lets too many by, what is at or above the
        // chunk's threshold
        uint32_t fresh = 0u, need = max(bound ? bound + 1u : 0u, 0x007fffffu);             // (-infinity)
        float need_x;
        auto collect = [&](auto careful) __attribute__((always_inline)) {
            fresh = 0u;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const bool in = x[i] >= need_x && (!decltype(careful)::value || is_token(i));
                const unsigned long long mask = __ballot(in);
                if (mask == 0ull) continue;
                const uint32_t to = fresh + lanes_before(mask);
                if (in && to < 64u) {
                    list.x[count + to] = x[i];
                    list.token[count + to] = place_of(i);
                }
                fresh += (uint32_t)__popcll(mask);
            }
        };
#pragma unroll 1
        for (bool known = bound != 0u;; known = false) {
            if (!known) {
                const uint32_t t = nth_of_wave(first + lane < stop ? beam_order(top) : 0u, a.best);
                need = max(need, t);
                if (t > bound) bound = t;
            }
            need_x = __uint_as_float(need & 0x80000000u ? need & 0x7fffffffu : ~need);        // (compared as floats: NaN never passes)
            fresh = 0u;
            if (!__any(top >= need_x)) break;
            // (what a chunk that is not whole has no logit for is -infinity)
            if (need == 0x007fffffu) collect(std::true_type{});
            else collect(std::false_type{});
            if (!known || fresh <= 64u) break;
        }
        if (fresh > 64u) {
            unsigned long long last = ~0ull;         // order and token of the one taken last, as one number that falls
            fresh = 0u;
#pragma unroll 1
            for (uint32_t r = 0; r < a.best; ++r) {
                unsigned long long mine = 0ull;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const unsigned long long u = is_token(i) && x[i] >= need_x ? ((unsigned long long)beam_order(x[i]) << 32) | (uint32_t)~place_of(i) : 0ull;
                    if (u < last && u > mine) mine = u;
                }
                last = wave_max(mine);
                if (!last) break;
                const uint32_t key = (uint32_t)(last >> 32);
                if (lane == 0u) {
                    list.x[count + r] = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
                    list.token[count + r] = ~(uint32_t)last;
                }
                ++fresh;
            }
        }
        count += fresh;
        if (count > 64u) bound = max(bound, keep_best<LOW>(list, count, a.best, lane));
    }
    if (count > a.best) keep_best<LOW>(list, count, a.best, lane);
    wave_sync_lds();
    sum = reduce_wave(sum, OpAdd());
    if (lane == 0u) {
        a.stat[2u * (size_t)at] = m;
        a.stat[2u * (size_t)at + 1u] = sum;
    }
    if (lane < a.best) {
        a.cand[(size_t)at * a.best + lane] = lane < count ? list.x[lane] : 0.f;
        a.cand_token[(size_t)at * a.best + lane] = lane < count ? list.token[lane] : NO_TOKEN;
    }
}

struct Choice {
    double sum;
    uint32_t at;             // beam * vocab + token
};
__device__ __forceinline__ bool before(const Choice &x, const Choice &y) { return x.sum > y.sum || (x.sum == y.sum && x.at < y.at); }

// Block = sequence.  Sums in 64 bits: log probabilities of different beams meet here, and 32 would make ties of what is none.  A beam whose log probabilities are no numbers (a NaN or
// an infinity among logits or scores) counts with sums of -infinity.  The threshold as above, on sums rounded to 32 bits (which keeps their order): of 64 groups of threads the n-th
// largest of their largest.  Some twenty of `best` = 16 pass, which one wave ranks, each in turn out of its lane's registers.  Candidates are loaded before their beams' sums are known.
__global__ __launch_bounds__(JOIN_THREADS) void tq_beam_join_kernel(BeamArgs a) {
    constexpr int WAVES = JOIN_THREADS / 64, HELD = 4;
    extern __shared__ double lds_base[];                     // [beams] score - log of the sum of exponentials
    __shared__ Choice lds_c[JOIN_HELD];
    __shared__ uint32_t lds_t[JOIN_THREADS], lds_n;
    __shared__ Choice lds_best[WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, b = blockIdx.x, slots = a.parts * a.best, all = a.beams * slots;
    const size_t row0 = (size_t)b * a.beams;
    const TQ_GLOBAL float *cand = (const TQ_GLOBAL float *)a.cand + row0 * slots;
    const TQ_GLOBAL uint32_t *cand_token = (const TQ_GLOBAL uint32_t *)a.cand_token + row0 * slots;
    float hx[HELD];
    uint32_t ht[HELD];
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const uint32_t i = min(tid + (uint32_t)j * JOIN_THREADS, all - 1u);
        hx[j] = cand[i];
        ht[j] = cand_token[i];
    }
    if (tid == 0u) lds_n = 0u;
    for (uint32_t k = wave; k < a.beams; k += WAVES) {
        const TQ_GLOBAL float *stat = (const TQ_GLOBAL float *)a.stat + 2u * (row0 + k) * a.parts;
        const float score = a.scores[(long long)b * a.score_stride + k];
        float m = -__builtin_inff();
        for (uint32_t p = lane; p < a.parts; p += 64u) m = fmaxf(m, stat[2u * p]);
        m = reduce_wave(m, OpMax());
        float s = 0.f;
        for (uint32_t p = lane; p < a.parts; p += 64u) {
            const float own = stat[2u * p + 1u];
            if (own != 0.f) s = fmaf(own, __builtin_amdgcn_exp2f((stat[2u * p] - m) * LOG2E_F), s);
        }
        s = reduce_wave(s, OpAdd());
        if (lane == 0u) lds_base[k] = (double)score - ((double)m + log((double)s));
    }
    __syncthreads();
    // Candidate i, of a logit and its token: none (false), or its sum
    auto score_of = [&](uint32_t i, float x, uint32_t token, Choice &c) {
        const uint32_t k = i / slots, slot = i - k * slots;
        const double base = lds_base[k];
        if (!(fabs(base) < __builtin_inf())) {               // (its first tokens, as among equals)
            c.sum = -__builtin_inf();
            c.at = k * a.vocab + slot;
            return slot < a.best && slot < a.vocab;
        }
        c.sum = base + (double)x;
        c.at = k * a.vocab + token;
        return token != NO_TOKEN;
    };
    auto each = [&](auto use) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const uint32_t i = tid + (uint32_t)j * JOIN_THREADS;
            Choice c;
            if (i < all && score_of(i, hx[j], ht[j], c)) use(c);
        }
        for (uint32_t i = tid + HELD * JOIN_THREADS; i < all; i += JOIN_THREADS) {
            Choice c;
            if (score_of(i, cand[i], cand_token[i], c)) use(c);
        }
    };
    uint32_t most = 0u;
    each([&](const Choice &c) { most = max(most, beam_order((float)c.sum)); });
    lds_t[tid] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) most = max(w ? most : 0u, lds_t[WAVES * lane + w]);
    const uint32_t least = max(nth_of_wave(most, a.best), 1u);
    each([&](const Choice &c) {
        if (beam_order((float)c.sum) < least) return;
        const uint32_t at = atomicAdd(&lds_n, 1u);
        if (at < JOIN_HELD) lds_c[at] = c;
    });
    __syncthreads();
    const uint32_t n = lds_n;
    auto put = [&](uint32_t r, const Choice &c) {
        const size_t at = (size_t)b * a.best + r;
        a.values[at] = (float)c.sum;
        a.tokens[at] = c.at % a.vocab;
        a.parents[at] = c.at / a.vocab;
    };
    if (n <= 64u) {
        if (wave) return;
        const Choice c = lane < n ? lds_c[lane] : Choice{-__builtin_inf(), NO_TOKEN};
        const unsigned long long bits = __builtin_bit_cast(unsigned long long, c.sum);
        uint32_t rank = 0u;
#pragma unroll 4
        for (uint32_t j = 0; j < n; ++j) {
            const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), (int)j), lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, (int)j);
            const Choice other = {__builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo), (uint32_t)__builtin_amdgcn_readlane((int)c.at, (int)j)};
            rank += before(other, c) ? 1u : 0u;
        }
        if (lane < n && rank < a.best) put(rank, c);
        return;
    }
    if (n <= JOIN_HELD) {
        for (uint32_t i = tid; i < n; i += JOIN_THREADS) {
            const Choice c = lds_c[i];
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
        each([&](const Choice &c) {
            if ((!any || before(last, c)) && before(c, mine)) mine = c;
        });
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

struct BeamPlan {
    int per_lane, chunks;            // logits a lane holds at a time, and how often
    long long rows, parts, bytes;
};
// Chunks of 2048 logits a wave, up to four, where that leaves two waves a SIMD; of 512 where there are not as many of the larger ones.
int beam_plan(long long batch, long long beams, long long vocab, long long best, BeamPlan &p) {
    const long long most = 0x7fffffff;
    if (batch < 0 || beams < 0 || vocab < 0 || best < 0 || batch > most || beams > 1024 || vocab > most || best > BEST_MAX) return TQ_ERR_SIZE;
    if (beams && vocab > most / beams) return TQ_ERR_SIZE;
    if (batch && best > beams * vocab) return TQ_ERR_SIZE;
    int cus = 0;
    if (tq_device_cus(cus)) cus = 256;
    p.rows = batch * beams;
    const long long waves = 8LL * cus;
    p.per_lane = p.rows * ((vocab + 2047) / 2048) >= waves ? 32 : 8;
    const long long chunk = 64LL * p.per_lane, all = (vocab + chunk - 1) / chunk;
    p.chunks = 1;
    while (p.chunks < 4 && p.rows * ((all + 2 * p.chunks - 1) / (2 * p.chunks)) >= waves) p.chunks *= 2;
    // (a row's sums are joined by one block: no more than 64 parts, unless chunks get many)
    while ((all + p.chunks - 1) / p.chunks > 64 && p.chunks < 64) p.chunks *= 2;
    p.parts = (all + p.chunks - 1) / p.chunks;
    if (p.parts && p.rows > most / p.parts) return TQ_ERR_SIZE;
    if (beams && p.parts * beams > most / (best ? best : 1)) return TQ_ERR_SIZE;
    p.bytes = p.rows * p.parts * (8 + 8 * best);
    return TQ_OK;
}

template <int DT>
void launch_parts(const BeamArgs &a, const BeamPlan &p, hipStream_t s) {
    const dim3 g((unsigned)((p.rows * p.parts + PART_WAVES - 1) / PART_WAVES)), t(64 * PART_WAVES);
    if (p.per_lane == 32) hipLaunchKernelGGL((tq_beam_part_kernel<DT, 32>), g, t, 0, s, a);
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
    a.rows = (uint32_t)p.rows; a.chunks = (uint32_t)p.chunks; a.beams = (uint32_t)beams; a.vocab = (uint32_t)vocab; a.best = (uint32_t)best; a.parts = (uint32_t)p.parts;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == TQ_F32) launch_parts<TQ_F32>(a, p, s);
    else if (dtype == TQ_F16) launch_parts<TQ_F16>(a, p, s);
    else launch_parts<TQ_BF16>(a, p, s);
    hipLaunchKernelGGL(tq_beam_join_kernel, dim3((unsigned)batch), dim3(JOIN_THREADS), (size_t)beams * sizeof(double), s, a);
    return (int)hipGetLastError();
}
