// softmax(scale q K^T) V of any number of query tokens per sequence over a packed history, the window behind it and tokens that are in no
// cache (drafts), with lengths and masks: tq_attend_many.  Launches, where a kernel with tables is built (fast): packed and uncompressed tokens, a block a split of a row's
// packed ones (tq_many_fast.h); merge, unless every row is in one split; and where the caller keeps count, what every key has received.  Otherwise one more
// each for the queries into the codec's space and for the uncompressed tokens (tq_many_kernel.h).
#include "tq_many_kernel.h"

namespace {

constexpr int MAX_SPLITS = 64;

int padded(int D) { return TQ_PADDED_DIM(D); }

long long plain_tiles(const tq_attend_request *r) { return (r->window.tokens + 31) / 32 + (r->drafts.tokens + 31) / 32; }

struct Plan {
    long long rows, tiles, groups, splits, records, plain_records;
    long long operands, stats, scales, floats;          // float32 values of scratch: rotated queries, statistics, scales, and all with the records
    int qt, kt, vt;                  // tiles a block and fp16 terms of the kernels for one padded head dimension; qt = 0: the one for all
};

// Whether a head dimension and its code widths have a kernel of their own.
bool fast(const tq_attend_request *r) {
    const int ik = 8 / r->bits_k, iv = 8 / r->bits_v, D = r->head_dim;
    if (ik > 4 || iv > 4 || r->tokens < 32) return false;
    if (D == 64 || D == 128 || D == 256)
        return !((uintptr_t)r->k_idx & (tq_packed_alignment(D, r->bits_k) - 1u)) && !((uintptr_t)r->v_idx & (tq_packed_alignment(D, r->bits_v) - 1u));
    // 65 to 96: whole groups of eight elements, and words of packed bytes
    return D > 64 && D <= 96 && !(D & 7) && !(D / ik & 3) && !(D % ik) && !(D / iv & 3) && !(D % iv) && !(((uintptr_t)r->k_idx | (uintptr_t)r->v_idx) & 3u);
}

// Splits of the tokens among blocks of which one is resident per compute unit: rounds of blocks, each as long as a block's tokens and, in tokens, what its start and its
// end cost (1500) and its uncompressed tokens (1000; `others`: blocks of those in the same launch), and for the merge 1000 and 30 a split.  A token with two terms of
// everything (float32) counts three times.  Measured (us) against other numbers of splits, 8 key/value heads of 128: 2048 tokens x 32 query vectors 19.1 with 8 (1: 32.5,
// 4: 20.2), 8192 x 32 21.5 with 16 (8: 24.0, 32: 31.1), 131072 x 32 47.4 with 31 (24: 50.9, 16: 61.7, 64: 66.2), 16 sequences of 8192 x 64 as below, 32 of 8192 x 4 with kept
// sums 123 with 1 (2: 140); float32 rows of 1003 tokens, 80 wide, 22.0 with 4 (1: 25.1).
long long fast_splits(int cus, long long blocks, long long others, long long tokens, int vt) {
    const long long weight = vt == 2 ? 3 : 1;
    long long most = (tokens + 255) / 256, best = 1, best_cost = 0;
    if (most > MAX_SPLITS) most = MAX_SPLITS;
    for (long long s = 1; s <= most; ++s) {
        const long long rounds = (blocks * s + cus - 1) / cus, extra = s == 1 ? rounds * (others ? 1000 : 0) : blocks * s + others > rounds * cus ? (others + cus - 1) / cus * 1000 : 0;
        const long long cost = rounds * ((tokens + s - 1) / s * weight + 1500) + extra + (s > 1 ? 1000 : 0) + 30 * s;
        if (s == 1 || cost < best_cost) { best = s; best_cost = cost; }
        if (rounds > 16 && s > 1) break;
    }
    return best;
}

int plan(const tq_attend_request *r, Plan &p) {
    p.rows = r->batch * r->heads;
    p.tiles = (r->group * r->n_queries + 31) / 32;
    const long long at = p.rows * p.tiles;
    p.splits = 1;
    p.qt = p.kt = p.vt = 0;
    p.groups = p.tiles;
    if (at && r->tokens && fast(r)) {
        p.kt = r->dtype == TQ_BF16 && !r->weights ? 1 : 2;
        p.vt = r->dtype == TQ_F32 ? 2 : 1;
        // Two tiles of queries a block share what is read and decoded.  One, where that fills no more than a round of blocks without splitting a row: 16 sequences
        // of 8192 tokens, 64 query vectors a head, 76 us against 91, 2 of 1024 x 512 29 against 40; but 8 of 4096 x 2048 541 against 419, 1 of 32768 x 256 78 against 68.
        int cus = 0;
        if (tq_device_cus(cus)) cus = 256;
        const long long others = plain_tiles(r) ? at : 0;
        p.qt = 1;
        p.splits = fast_splits(cus, at, others, r->tokens, p.vt);
        if (p.kt == 1 && r->head_dim != 256 && p.tiles > 1 && (p.splits > 1 || at > cus)) {
            p.qt = 2;
            p.groups = (p.tiles + 1) / 2;
            p.splits = fast_splits(cus, p.rows * p.groups, others ? p.rows * p.groups : 0, r->tokens, p.vt);
        }
    } else if (at && r->tokens) {
        int cus = 0;
        if (tq_device_cus(cus)) cus = 256;
        p.splits = (2 * cus + at - 1) / at;
        const long long most = (r->tokens + 127) / 128;
        if (p.splits > most) p.splits = most;
        if (p.splits > MAX_SPLITS) p.splits = MAX_SPLITS;
        if (p.splits < 1) p.splits = 1;
    }
    const bool whole = p.qt && p.splits == 1;          // a block has all of its queries' tokens: no records, no merge
    p.records = whole || !r->tokens ? 0 : p.splits * (p.qt ? 1 : ANY_WAVES);
    p.plain_records = whole || !plain_tiles(r) ? 0 : (p.qt ? 1 : PLAIN_WAVES);
    const long long dp = padded(r->head_dim);
    // Only what is written: kernels with tables rotate their queries themselves and write the operands out for the launch that adds up what keys receive, the only one that
    // reads statistics.  (Four at least: a caller always has something to hand over.)
    p.operands = p.qt && !r->weights ? 0 : at * ((long long)q_operand_bytes((uint32_t)dp) / 4);
    p.stats = r->weights ? at * MANY_STATS : 0;
    p.scales = p.qt && !r->weights ? 0 : at * 32;
    p.floats = p.operands + at * (p.records + p.plain_records) * record_floats((uint32_t)dp) + p.stats + p.scales;
    if (p.floats < 4) p.floats = 4;
    return at * (p.splits + 1) * 4 > 0x7fffffffLL ? TQ_ERR_SIZE : TQ_OK;
}

int check(const tq_attend_request *r) {
    if (!r) return TQ_ERR_NULL;
    if (r->dtype != TQ_F32 && r->dtype != TQ_F16 && r->dtype != TQ_BF16) return TQ_ERR_DTYPE;
    if (r->bits_k < 1 || r->bits_k > 8 || r->bits_v < 1 || r->bits_v > 8) return TQ_ERR_BITS;
    if (r->head_dim < TQ_ANYDIM_MIN || r->head_dim > TQ_ANYDIM_MAX) return TQ_ERR_HEAD_DIM;
    const long long most = 0x7fffffff;
    if (r->batch < 0 || r->heads < 0 || r->group < 0 || r->n_queries < 0 || r->tokens < 0 || r->window.tokens < 0 || r->drafts.tokens < 0) return TQ_ERR_SIZE;
    if (r->batch > most || r->heads > most || r->group > most || r->n_queries > most || r->tokens > most - 65536 || r->window.tokens > 65536 || r->drafts.tokens > 65536)
        return TQ_ERR_SIZE;
    if (r->batch * r->heads > most || r->heads * r->group > most || r->group * r->n_queries > most / 2) return TQ_ERR_SIZE;
    const long long rows = r->batch * r->heads, tiles = (r->group * r->n_queries + 31) / 32;
    if (rows && tiles > most / rows) return TQ_ERR_SIZE;
    if (r->packed_row_stride < 0 || r->packed_row_stride > most || (r->packed_row_stride && r->packed_row_stride < r->tokens)) return TQ_ERR_SIZE;
    return TQ_OK;
}

bool aligned16(const tq_plain_tokens &t, long long es) {
    return !(((uintptr_t)t.k | (uintptr_t)t.v) & 15u) && !((t.k_batch * es) & 15) && !((t.k_head * es) & 15) && !((t.k_token * es) & 15) && !((t.v_batch * es) & 15) &&
           !((t.v_head * es) & 15) && !((t.v_token * es) & 15);
}

TqManyPlain plain_of(const tq_plain_tokens &t) {
    return TqManyPlain{static_cast<const uint8_t *>(t.k), static_cast<const uint8_t *>(t.v), t.k_batch, t.k_head, t.k_token, t.v_batch, t.v_head, t.v_token, (uint32_t)t.tokens};
}

// Results where there is no token at all.  (Elements are two or four bytes.)
__global__ __launch_bounds__(256) void tq_many_zero_kernel(uint16_t *out, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256u + threadIdx.x; i < n; i += (size_t)gridDim.x * 256u) ((TQ_GLOBAL uint16_t *)out)[i] = 0u;
}

template <int DP>
void launch_dim(const TqManyArgs &a, const Plan &plan, hipStream_t s) {
    const uint32_t at = a.rows * a.tiles;
    if (plan.qt) {
        const dim3 g((unsigned)(plan.rows * plan.groups * plan.splits + a.plain_blocks));
        const int ik = 8 / (int)a.bits_k, iv = 8 / (int)a.bits_v;
        if constexpr (DP == 64) tq_many_launch_d64(ik, iv, g, s, a, plan.qt, plan.kt, plan.vt);
        if constexpr (DP == 96) tq_many_launch_d96(ik, iv, g, s, a, plan.qt, plan.kt, plan.vt);
        if constexpr (DP == 128) tq_many_launch_d128(ik, iv, g, s, a, plan.qt, plan.kt, plan.vt);
        if constexpr (DP == 256) tq_many_launch_d256(ik, iv, g, s, a, plan.qt, plan.kt, plan.vt);
    } else if (a.records) hipLaunchKernelGGL((tq_many_any_kernel<DP>), dim3(at * a.splits), dim3(64 * ANY_WAVES), 0, s, a);
    if (a.plain_records && !plan.qt) {
        const dim3 g(at), t(64 * PLAIN_WAVES);
        if (a.dtype == TQ_F32) hipLaunchKernelGGL((tq_many_plain_kernel<DP, TQ_F32>), g, t, 0, s, a);
        else if (a.dtype == TQ_F16) hipLaunchKernelGGL((tq_many_plain_kernel<DP, TQ_F16>), g, t, 0, s, a);
        else hipLaunchKernelGGL((tq_many_plain_kernel<DP, TQ_BF16>), g, t, 0, s, a);
    }
    if (a.records || a.plain_records) {
        if (at < 128u) hipLaunchKernelGGL((tq_many_merge_kernel<DP, 8>), dim3(at * 4u), dim3(2 * DP), 0, s, a);
        else hipLaunchKernelGGL((tq_many_merge_kernel<DP, 32>), dim3(at), dim3(2 * DP), 0, s, a);
    }
    if (!a.weights) return;
    if (a.tokens && plan.qt) {
        int cus = 0;
        if (tq_device_cus(cus)) cus = 256;
        // one block is resident per compute unit, or two where it has no more than 16 query vectors; the window's come first
        const uint32_t most = (a.tokens + 255u) / 256u, window = (a.rows * ((a.plain[0].n + 31u) / 32u) + 7u) / 8u;
        const uint32_t places = (uint32_t)cus * (many_few(a, DP) && DP != 256 ? 2u : 1u);
        // (their places are kept where that takes an eighth of the others' at most: 8 rows of 32768 tokens, 9.7 us with 63 blocks a row and 10.1 with 64; 256 of 8192, 45.5 with 1, 40.9 with 2)
        const uint32_t every = max(places / a.rows, 1u), fewer = places > window ? (places - window) / a.rows : 0u;
        uint32_t blocks = 8u * fewer >= 7u * every ? fewer : every;
        if (blocks > most) blocks = most;
        const dim3 g(a.rows * blocks + window);
        const int ik = 8 / (int)a.bits_k;
        if constexpr (DP == 64) tq_many_weights_launch_d64(ik, g, s, a, blocks);
        if constexpr (DP == 96) tq_many_weights_launch_d96(ik, g, s, a, blocks);
        if constexpr (DP == 128) tq_many_weights_launch_d128(ik, g, s, a, blocks);
        if constexpr (DP == 256) tq_many_weights_launch_d256(ik, g, s, a, blocks);
        return;
    }
    if (a.tokens) {
        const uint32_t blocks = (a.tokens + 32u * ANY_WAVES - 1u) / (32u * ANY_WAVES);
        hipLaunchKernelGGL((tq_many_any_weights_kernel<DP>), dim3(a.rows * blocks), dim3(64 * ANY_WAVES), 0, s, a, blocks);
    }
    if (a.plain[0].n) {
        const dim3 g(a.rows * ((a.plain[0].n + 31u) / 32u));
        if (a.dtype == TQ_F32) hipLaunchKernelGGL((tq_many_plain_weights_kernel<TQ_F32>), g, dim3(64), 0, s, a, DP / 16u);
        else if (a.dtype == TQ_F16) hipLaunchKernelGGL((tq_many_plain_weights_kernel<TQ_F16>), g, dim3(64), 0, s, a, DP / 16u);
        else hipLaunchKernelGGL((tq_many_plain_weights_kernel<TQ_BF16>), g, dim3(64), 0, s, a, DP / 16u);
    }
}

}  // namespace

extern "C" long long tq_attend_many_scratch(const tq_attend_request *request) {
    const int rc = check(request);
    if (rc) return rc;
    Plan p;
    const int bad = plan(request, p);
    return bad ? bad : p.floats;
}

extern "C" int tq_attend_many(const tq_attend_request *request, float *scratch, long long scratch_floats, void *stream) {
    int rc = check(request);
    if (rc) return rc;
    const tq_attend_request &r = *request;
    Plan p;
    rc = plan(request, p);
    if (rc) return rc;
    if (p.rows * p.tiles == 0) return TQ_OK;
    if (!r.queries || !r.out || !r.table_k || !r.table_v || !scratch) return TQ_ERR_NULL;
    if (r.tokens && (!r.k_idx || !r.k_norms || !r.v_idx || !r.v_norms)) return TQ_ERR_NULL;
    if ((r.window.tokens && (!r.window.k || !r.window.v)) || (r.drafts.tokens && (!r.drafts.k || !r.drafts.v))) return TQ_ERR_NULL;
    const long long total = r.tokens + r.window.tokens;
    if (r.mask && r.batch > 1 && r.mask_stride < total) return TQ_ERR_SIZE;
    if (r.weights && p.rows > 1 && r.weights_stride < total) return TQ_ERR_SIZE;
    if (!r.tree && r.drafts.tokens && r.drafts.tokens != r.n_queries) return TQ_ERR_SIZE;
    const long long es = r.dtype == TQ_F32 ? 4 : 2;
    if (((uintptr_t)r.table_k & 15u) || ((uintptr_t)r.table_v & 15u) || ((uintptr_t)scratch & 15u) || ((uintptr_t)r.k_norms & 1u) || ((uintptr_t)r.v_norms & 1u) ||
        ((uintptr_t)r.lengths & 3u) || ((uintptr_t)r.weights & 3u) || ((uintptr_t)r.queries & (es - 1)) || ((uintptr_t)r.out & (es - 1)))
        return TQ_ERR_ALIGN;
    if (scratch_floats < p.floats) return TQ_ERR_CAPACITY;
    const uint32_t dp = (uint32_t)padded(r.head_dim);
    const long long at = p.rows * p.tiles;
    TqManyArgs a{};
    a.q = static_cast<const uint8_t *>(r.queries);
    a.out = static_cast<uint8_t *>(r.out);
    a.q_batch = r.q_batch; a.q_head = r.q_head; a.q_token = r.q_token;
    a.k_idx = r.k_idx; a.v_idx = r.v_idx; a.k_norms = r.k_norms; a.v_norms = r.v_norms;
    a.table_k = static_cast<const uint8_t *>(r.table_k); a.table_v = static_cast<const uint8_t *>(r.table_v);
    a.plain[0] = plain_of(r.window); a.plain[1] = plain_of(r.drafts);
    a.lengths = r.lengths; a.mask = r.mask; a.tree = r.tree;
    a.mask_stride = r.mask_stride; a.tree_batch = r.tree_batch;
    a.weights = r.weights; a.w_stride = r.weights_stride;
    // scratch: operands, records, uncompressed tokens' records, statistics, scales
    float *f = scratch;
    a.q_op = reinterpret_cast<uint8_t *>(f); f += p.operands;
    a.rec = f; f += at * p.records * record_floats(dp);
    a.plain_rec = f; f += at * p.plain_records * record_floats(dp);
    if (r.weights) a.stat = f;
    f += p.stats;
    a.q_scale = f;
    a.scale = r.scale;
    a.rows = (uint32_t)p.rows; a.heads = (uint32_t)r.heads; a.group = (uint32_t)r.group; a.queries = (uint32_t)r.n_queries;
    a.M = (uint32_t)(r.group * r.n_queries); a.tiles = (uint32_t)p.tiles; a.tokens = (uint32_t)r.tokens;
    a.packed_row_stride = (uint32_t)(r.packed_row_stride ? r.packed_row_stride : r.tokens);
    a.D = (uint32_t)r.head_dim; a.bits_k = (uint32_t)r.bits_k; a.bits_v = (uint32_t)r.bits_v; a.dtype = (uint32_t)r.dtype;
    a.splits = (uint32_t)p.splits; a.records = (uint32_t)p.records; a.plain_records = (uint32_t)p.plain_records;
    a.chunk = (uint32_t)(((r.tokens + p.splits - 1) / p.splits + 31) / 32 * 32);
    a.aligned = !(r.head_dim & 7) && !((uintptr_t)r.queries & 15u) && !((r.q_batch * es) & 15) && !((r.q_head * es) & 15) && !((r.q_token * es) & 15) &&
                (!r.window.tokens || aligned16(r.window, es)) && (!r.drafts.tokens || aligned16(r.drafts, es));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (!r.tokens && !plain_tiles(request)) {          // (no kernel below has anything to do; sums of no key stay as they are)
        const size_t n = (size_t)(p.rows * r.group * r.n_queries) * (size_t)r.head_dim * (size_t)(es / 2), blocks = (n + 255) / 256;
        hipLaunchKernelGGL(tq_many_zero_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, static_cast<uint16_t *>(r.out), n);
        return (int)hipGetLastError();
    }
    a.plain_blocks = p.qt && p.plain_records ? (uint32_t)(p.rows * p.groups) : 0u;
    if (!p.qt) {
        const dim3 g((unsigned)(p.rows * ((p.tiles + 1) / 2))), t((p.tiles > 1 ? 4 : 2) * dp);
        if (r.dtype == TQ_F32) hipLaunchKernelGGL((tq_many_prepare_kernel<TQ_F32>), g, t, 0, s, a, dp / 32u);
        else if (r.dtype == TQ_F16) hipLaunchKernelGGL((tq_many_prepare_kernel<TQ_F16>), g, t, 0, s, a, dp / 32u);
        else hipLaunchKernelGGL((tq_many_prepare_kernel<TQ_BF16>), g, t, 0, s, a, dp / 32u);
    }
    switch (dp) {
        case 32: launch_dim<32>(a, p, s); break;
        case 64: launch_dim<64>(a, p, s); break;
        case 96: launch_dim<96>(a, p, s); break;
        case 128: launch_dim<128>(a, p, s); break;
        case 160: launch_dim<160>(a, p, s); break;
        case 192: launch_dim<192>(a, p, s); break;
        case 224: launch_dim<224>(a, p, s); break;
        default: launch_dim<256>(a, p, s); break;
    }
    return (int)hipGetLastError();
}
