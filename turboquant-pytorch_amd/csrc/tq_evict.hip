// Of every row of a packed store the `keep` tokens with the largest weights, in their order, into another store: tq_evict.
// Two launches: which tokens stay (a block a row), and their bytes.
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

// Block = row.  The keep-th largest weight is found eight bits at a time from counts of the tokens that agree with it so far; the tokens above it
// stay, and of those equal to it the first ones.
__global__ __launch_bounds__(SELECT_THREADS) void tq_evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t lds_count[256], lds_scan[SELECT_THREADS / 64], lds_found[2];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float *w = a.weights + (long long)row * a.w_stride;
    uint32_t prefix = 0u, left = a.keep;          // left: how many of those that agree with the prefix stay
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256u) lds_count[tid] = 0u;
        __syncthreads();
        for (uint32_t i = tid; i < a.tokens; i += SELECT_THREADS) {
            const uint32_t u = order_of(w[i]);
            if (shift == 24 || (u ^ prefix) >> (shift + 8) == 0u) atomicAdd(&lds_count[(u >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0u) {
            uint32_t above = 0u, digit = 255u;
            while (digit > 0u && above + lds_count[digit] < left) above += lds_count[digit--];
            lds_found[0] = digit;
            lds_found[1] = above;
        }
        __syncthreads();
        prefix |= lds_found[0] << shift;
        left -= lds_found[1];
        __syncthreads();
    }
    long long *kept = a.kept + (long long)row * a.keep;
    uint32_t out = 0u, equal = 0u;                // over the tokens before this round
    for (uint32_t i0 = 0; i0 < a.tokens; i0 += SELECT_THREADS) {
        const uint32_t i = i0 + tid;
        const uint32_t u = i < a.tokens ? order_of(w[i]) : 0u;
        const bool above = i < a.tokens && u > prefix, same = i < a.tokens && u == prefix;
        uint32_t all;
        const uint32_t rank = equal + block_scan(same ? 1u : 0u, lds_scan, all);
        equal += all;
        const bool stays = above || (same && rank < left);
        const uint32_t at = out + block_scan(stays ? 1u : 0u, lds_scan, all);
        out += all;
        if (stays) kept[at] = i;
    }
}

template <typename T>
__device__ __forceinline__ void move_codes(const uint8_t *src, uint8_t *dst, uint32_t bytes, uint32_t first, uint32_t step) {
    for (uint32_t i = first * sizeof(T); i < bytes; i += step * sizeof(T)) *reinterpret_cast<T *>(dst + i) = *reinterpret_cast<const T *>(src + i);
}

// Eight lanes a token
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

extern "C" int tq_evict(const tq_packed_store *from, const tq_packed_store *to, const float *weights, long long weights_stride, float *weights_out,
                        long long weights_out_stride, long long rest, long long rows, long long tokens, long long keep, int head_dim, int bits_k, int bits_v, long long *kept, void *stream) {
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
    if (keep) hipLaunchKernelGGL(tq_evict_select_kernel, dim3((unsigned)rows), dim3(SELECT_THREADS), 0, st, a);
    hipLaunchKernelGGL(tq_evict_move_kernel, dim3((unsigned)(rows * blocks)), dim3(256), 0, st, a, (uint32_t)blocks);
    return (int)hipGetLastError();
}
