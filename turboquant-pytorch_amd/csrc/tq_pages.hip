// Stores of tokens moved about as they are: rows of a cache that follow the beams chosen (tq_reorder), pages copied between and within pools (tq_copy_pages), and
// new tokens put into the pages that are not packed yet (tq_put_tokens).  All of it is bound by memory.
#include "tq_device.h"

namespace {

constexpr int MOVE_THREADS = 256;

template <typename T>
__device__ __forceinline__ T get(const uint8_t *p) { return *reinterpret_cast<const TQ_GLOBAL T *>((const TQ_GLOBAL uint8_t *)p); }
template <typename T>
__device__ __forceinline__ void put(uint8_t *p, T v) { *reinterpret_cast<TQ_GLOBAL T *>((TQ_GLOBAL uint8_t *)p) = v; }

// ---- rows that follow others, in place -----------------------------------------------------------------------------------------
struct Segment {                     // [batch][heads][bytes]
    uint8_t *base;
    long long batch_stride, head_stride;
    uint32_t pieces;                 // a head's bytes in pieces of the launch's unit
    uint32_t first_block;            // of the launch
};
constexpr int SEGMENTS = 64;
struct ReorderArgs {
    const long long *parents;        // [batch]
    uint32_t batch, heads, count;
    Segment segment[SEGMENTS];
};

// Block = `COLUMNS` pieces of a segment, of all sequences: rows that change are read, all of them, before one is written, so that nothing is kept aside in memory and rows that stay
// where they are cost nothing.  A thread has every (threads / COLUMNS)-th sequence, K of them at most.  Parents outside the batch leave the row as it is.
template <typename T, int THREADS, int COLUMNS, int K>
__global__ __launch_bounds__(THREADS) void tq_reorder_kernel(ReorderArgs a) {
    constexpr uint32_t STEP = THREADS / COLUMNS;
    uint32_t lo = 0u, hi = a.count;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (a.segment[mid].first_block <= blockIdx.x) lo = mid;
        else hi = mid;
    }
    const Segment &s = a.segment[lo];
    const unsigned long long at = (unsigned long long)(blockIdx.x - s.first_block) * COLUMNS + threadIdx.x % COLUMNS;
    const bool some = at < (unsigned long long)s.pieces * a.heads;
    const uint32_t head = some ? (uint32_t)(at / s.pieces) : 0u, piece = some ? (uint32_t)(at - (unsigned long long)head * s.pieces) : 0u;
    uint8_t *p = s.base + (long long)head * s.head_stride + (long long)piece * (long long)sizeof(T);
    const uint32_t first = COLUMNS == 64 ? tq_uniform32(threadIdx.x / COLUMNS) : threadIdx.x / COLUMNS;       // (a wave's: parents and addresses on the scalar unit)
    T v[K];
    uint32_t moved = 0u;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t b = first + (uint32_t)k * STEP;
        if (!some || b >= a.batch) continue;
        const long long from = a.parents[b];
        if (from == (long long)b || from < 0 || from >= (long long)a.batch) continue;
        v[k] = get<T>(p + from * s.batch_stride);
        moved |= 1u << k;
    }
    __builtin_amdgcn_s_waitcnt(0);           // what this wave has asked for is there before another one of the block writes
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k)
        if ((moved >> k) & 1u) put<T>(p + (long long)(first + (uint32_t)k * STEP) * s.batch_stride, v[k]);
}

template <typename T>
void launch_reorder(const ReorderArgs &a, uint32_t columns, uint32_t blocks, hipStream_t s) {
    if (columns == 64u) {
        if (a.batch <= 8u) hipLaunchKernelGGL((tq_reorder_kernel<T, MOVE_THREADS, 64, 2>), dim3(blocks), dim3(MOVE_THREADS), 0, s, a);
        else hipLaunchKernelGGL((tq_reorder_kernel<T, MOVE_THREADS, 64, 16>), dim3(blocks), dim3(MOVE_THREADS), 0, s, a);
    } else hipLaunchKernelGGL((tq_reorder_kernel<T, 1024, 16, 16>), dim3(blocks), dim3(1024), 0, s, a);
}

// ---- pages ---------------------------------------------------------------------------------------------------------------------
constexpr int PAIRS = 256;
struct CopyArgs {
    const uint8_t *from;
    uint8_t *to;
    long long from_stride, to_stride;        // bytes between pages
    uint32_t rows, row_bytes;                // a page is `rows` runs, row_bytes apart
    int32_t src[PAIRS], dst[PAIRS];
    uint32_t used[PAIRS];                    // bytes of every run that are copied
};

// Block = a share of one page.  Eight pieces a thread are under way at once; what is copied is not read again soon, so neither side asks the caches to keep it.
__global__ __launch_bounds__(MOVE_THREADS) void tq_copy_pages_kernel(CopyArgs a, uint32_t blocks) {
    constexpr int K = 8;
    const uint32_t pair = blockIdx.x / blocks, part = blockIdx.x - pair * blocks, pieces = a.used[pair] / 16u;
    const uint8_t *src = a.from + (long long)a.src[pair] * a.from_stride;
    uint8_t *dst = a.to + (long long)a.dst[pair] * a.to_stride;
    const unsigned long long all = (unsigned long long)pieces * a.rows;
    for (unsigned long long i0 = (unsigned long long)part * (K * MOVE_THREADS); i0 < all; i0 += (unsigned long long)blocks * (K * MOVE_THREADS)) {
        tq_u4 v[K];
        unsigned long long off[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const unsigned long long i = i0 + (uint32_t)k * MOVE_THREADS + threadIdx.x;
            const unsigned long long row = a.rows == 1u ? 0ull : (unsigned long long)((uint32_t)i / pieces);      // (a page is less than 2^32 pieces)
            off[k] = row * a.row_bytes + (i - row * pieces) * 16u;
            if (i < all) v[k] = tq_gload16_stream(src + off[k]);
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (i0 + (uint32_t)k * MOVE_THREADS + threadIdx.x < all) tq_gstore16_stream(dst + off[k], v[k]);
    }
}

// ---- new tokens ----------------------------------------------------------------------------------------------------------------
struct PutArgs {
    const uint8_t *src[2];                   // keys, values: token i, head h at i * token_stride + h * head_stride bytes
    long long token_stride[2], head_stride[2];
    uint8_t *pool;                           // page p, keys or values s, head h, place t at p * page_stride + s * side_stride + (h * page_tokens + t) * vector
    const int32_t *slots;                    // [tokens] page * page_tokens + place, or -1: the token is passed over
    long long page_stride, side_stride;
    uint32_t tokens, heads, vector, page_tokens, shift;
};
template <typename T>
__global__ __launch_bounds__(MOVE_THREADS) void tq_put_tokens_kernel(PutArgs a) {
    const uint32_t pieces = a.vector / sizeof(T);
    const unsigned long long each = (unsigned long long)pieces * a.heads, all = 2u * each * a.tokens;
    for (unsigned long long i = (unsigned long long)blockIdx.x * MOVE_THREADS + threadIdx.x; i < all; i += (unsigned long long)gridDim.x * MOVE_THREADS) {
        const uint32_t piece = (uint32_t)(i % pieces);
        const unsigned long long vec = i / pieces;
        const uint32_t h = (uint32_t)(vec % a.heads);
        const unsigned long long two = vec / a.heads;
        const uint32_t s = two >= a.tokens ? 1u : 0u, token = (uint32_t)(two - (s ? a.tokens : 0u));
        const uint32_t slot = (uint32_t)a.slots[token], page = slot >> a.shift, place = slot & (a.page_tokens - 1u);
        if (slot == 0xffffffffu) continue;       // (-1: of a step that is over)
        const T v = get<T>((s ? a.src[1] : a.src[0]) + (long long)token * (s ? a.token_stride[1] : a.token_stride[0]) +
                           (long long)h * (s ? a.head_stride[1] : a.head_stride[0]) + (size_t)piece * sizeof(T));
        put<T>(a.pool + (long long)page * a.page_stride + (long long)s * a.side_stride + ((long long)h * a.page_tokens + place) * (long long)a.vector + (size_t)piece * sizeof(T), v);
    }
}

}  // namespace

extern "C" int tq_reorder(const tq_move_segment *segments, int n_segments, long long batch, long long heads, const long long *parents, void *stream) {
    const long long most = 0x7fffffff;
    if (n_segments < 0 || batch < 0 || heads < 0 || heads > most) return TQ_ERR_SIZE;
    if (batch > 1024) return TQ_ERR_CAPACITY;
    if (n_segments == 0 || batch == 0 || heads == 0) return TQ_OK;
    if (!segments || !parents) return TQ_ERR_NULL;
    if ((uintptr_t)parents & 7u) return TQ_ERR_ALIGN;
    // every check comes before the first launch
    const uint32_t columns = batch <= 64 ? 64u : 16u;
    auto unit_of = [](const tq_move_segment &g) -> uint32_t {
        const unsigned long long low = (unsigned long long)(uintptr_t)g.base | (unsigned long long)g.batch_stride | (unsigned long long)g.head_stride | (unsigned long long)g.bytes;
        return !(low & 15u) ? 16u : !(low & 3u) ? 4u : !(low & 1u) ? 2u : 1u;
    };
    for (int i = 0; i < n_segments; ++i) {
        const tq_move_segment &g = segments[i];
        if (g.bytes < 0 || (g.bytes && !g.base)) return g.bytes < 0 ? TQ_ERR_SIZE : TQ_ERR_NULL;
        if ((heads > 1 && g.head_stride < g.bytes) || g.batch_stride < 0 || g.head_stride < 0) return TQ_ERR_SIZE;
        if (g.bytes > most || (batch > 1 && g.batch_stride < (heads - 1) * g.head_stride + g.bytes)) return TQ_ERR_SIZE;
        if (g.bytes / unit_of(g) > most / heads) return TQ_ERR_SIZE;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t units[4] = {16u, 4u, 2u, 1u};
    for (uint32_t unit : units) {
        ReorderArgs a{};
        a.parents = parents;
        a.batch = (uint32_t)batch; a.heads = (uint32_t)heads;
        uint32_t blocks = 0u;
        auto launch = [&]() {
            if (!a.count) return;
            if (unit == 16u) launch_reorder<tq_u4>(a, columns, blocks, s);
            else if (unit == 4u) launch_reorder<uint32_t>(a, columns, blocks, s);
            else if (unit == 2u) launch_reorder<uint16_t>(a, columns, blocks, s);
            else launch_reorder<uint8_t>(a, columns, blocks, s);
            a.count = 0u;
            blocks = 0u;
        };
        for (int i = 0; i < n_segments; ++i) {
            const tq_move_segment &g = segments[i];
            if (!g.bytes || unit_of(g) != unit) continue;
            const uint32_t pieces = (uint32_t)(g.bytes / unit);
            const unsigned long long need = ((unsigned long long)pieces * a.heads + columns - 1u) / columns;
            if (a.count == SEGMENTS || blocks + need > 0x7fffffffull) launch();
            a.segment[a.count++] = Segment{static_cast<uint8_t *>(g.base), g.batch_stride, g.head_stride, pieces, blocks};
            blocks += (uint32_t)need;
        }
        launch();
    }
    return (int)hipGetLastError();
}

extern "C" int tq_copy_pages(const void *from, long long from_stride, void *to, long long to_stride, long long rows, long long row_bytes, const tq_page_pair *pairs, long long n_pairs,
                             void *stream) {
    const long long most = 0x7fffffff;
    if (n_pairs < 0 || rows < 0 || rows > most || row_bytes < 0 || row_bytes > most || from_stride < 0 || to_stride < 0) return TQ_ERR_SIZE;
    if (n_pairs == 0 || rows == 0 || row_bytes == 0) return TQ_OK;
    if (!from || !to || !pairs) return TQ_ERR_NULL;
    if ((((uintptr_t)from | (uintptr_t)to) & 15u) || ((from_stride | to_stride | row_bytes) & 15)) return TQ_ERR_ALIGN;
    long long largest = 0;
    for (long long i = 0; i < n_pairs; ++i) {
        if (pairs[i].from < 0 || pairs[i].to < 0 || pairs[i].bytes < 0 || pairs[i].bytes > row_bytes) return TQ_ERR_SIZE;
        if (pairs[i].bytes & 15) return TQ_ERR_ALIGN;
        if (pairs[i].bytes > largest) largest = pairs[i].bytes;
    }
    if (row_bytes / 16 > 0xffffffffLL / rows) return TQ_ERR_SIZE;
    if (rows > 1 && (from_stride < rows * row_bytes || to_stride < rows * row_bytes)) return TQ_ERR_SIZE;
    int cus = 0;
    if (tq_device_cus(cus)) cus = 256;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    for (long long i0 = 0; i0 < n_pairs; i0 += PAIRS) {
        const long long n = n_pairs - i0 < PAIRS ? n_pairs - i0 : PAIRS;
        CopyArgs a{};
        a.from = static_cast<const uint8_t *>(from); a.to = static_cast<uint8_t *>(to);
        a.from_stride = from_stride; a.to_stride = to_stride;
        a.rows = (uint32_t)rows; a.row_bytes = (uint32_t)row_bytes;
        for (long long i = 0; i < n; ++i) {
            a.src[i] = pairs[i0 + i].from;
            a.dst[i] = pairs[i0 + i].to;
            a.used[i] = (uint32_t)pairs[i0 + i].bytes;
        }
        // a block has 32 KiB under way; no more blocks a page than that, and sixteen a compute unit in all
        long long blocks = (largest * rows + 128 * MOVE_THREADS - 1) / (128 * MOVE_THREADS), share = (16LL * cus + n - 1) / n;
        if (blocks > share) blocks = share;
        if (blocks < 1) blocks = 1;
        hipLaunchKernelGGL(tq_copy_pages_kernel, dim3((unsigned)(n * blocks)), dim3(MOVE_THREADS), 0, s, a, (uint32_t)blocks);
    }
    return (int)hipGetLastError();
}

extern "C" int tq_put_tokens(const void *keys, const void *values, long long k_token_stride, long long k_head_stride, long long v_token_stride, long long v_head_stride,
                             void *pool, long long page_stride, long long side_stride, const int32_t *slots, long long tokens, long long heads, long long vector_bytes,
                             int page_tokens, void *stream) {
    const long long most = 0x7fffffff;
    if (tokens < 0 || heads < 0 || vector_bytes < 0 || tokens > most || heads > most || vector_bytes > 65536 || page_stride < 0 || side_stride < 0) return TQ_ERR_SIZE;
    if (page_tokens < 1 || (page_tokens & (page_tokens - 1))) return TQ_ERR_SIZE;
    if (tokens == 0 || heads == 0 || vector_bytes == 0) return TQ_OK;
    if (!keys || !values || !pool || !slots) return TQ_ERR_NULL;
    if ((uintptr_t)slots & 3u) return TQ_ERR_ALIGN;
    PutArgs a{};
    a.src[0] = static_cast<const uint8_t *>(keys); a.src[1] = static_cast<const uint8_t *>(values);
    a.token_stride[0] = k_token_stride; a.token_stride[1] = v_token_stride;
    a.head_stride[0] = k_head_stride; a.head_stride[1] = v_head_stride;
    a.pool = static_cast<uint8_t *>(pool); a.slots = slots;
    a.page_stride = page_stride; a.side_stride = side_stride;
    a.tokens = (uint32_t)tokens; a.heads = (uint32_t)heads; a.vector = (uint32_t)vector_bytes;
    a.page_tokens = (uint32_t)page_tokens; a.shift = (uint32_t)__builtin_ctz((unsigned)page_tokens);
    const unsigned long long low = (uintptr_t)keys | (uintptr_t)values | (uintptr_t)pool | (unsigned long long)(k_token_stride | k_head_stride | v_token_stride | v_head_stride) |
                                   (unsigned long long)(page_stride | side_stride | vector_bytes);
    if (low & 1u) return TQ_ERR_ALIGN;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const long long unit = !(low & 15u) ? 16 : !(low & 3u) ? 4 : 2;
    long long blocks = (2 * tokens * heads * (vector_bytes / unit) + MOVE_THREADS - 1) / MOVE_THREADS;
    if (blocks > 65536) blocks = 65536;
    const dim3 g((unsigned)blocks), t(MOVE_THREADS);
    if (unit == 16) hipLaunchKernelGGL((tq_put_tokens_kernel<tq_u4>), g, t, 0, s, a);
    else if (unit == 4) hipLaunchKernelGGL((tq_put_tokens_kernel<uint32_t>), g, t, 0, s, a);
    else hipLaunchKernelGGL((tq_put_tokens_kernel<uint16_t>), g, t, 0, s, a);
    return (int)hipGetLastError();
}
