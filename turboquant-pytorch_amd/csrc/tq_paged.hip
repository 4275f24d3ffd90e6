// softmax(scale q K^T) V of sequences' new tokens over packed and plain pages, scores capped, biased by distance or within a window: tq_paged_attend, and the plan that its
// blocks work by, tq_paged_plan (on the host, where the lengths are known; one plan serves all layers of a step).  Two launches: a block an item of the plan (tq_paged_kernel.h), and
// where a tile's tokens are in several items, a merge.
#include <algorithm>
#include <vector>

#include "tq_paged.h"

namespace {

constexpr int MAX_PIECES = 64;
constexpr int MERGE_THREADS = 256;

// Block = (merge, tile of the pair, share of a tile's results): results are the records' sums, each times 2^(its reference - the largest), over their sums of weights.
template <int DP>
__global__ __launch_bounds__(MERGE_THREADS) void tq_paged_merge_kernel(TqPagedArgs a, uint32_t shares) {
    __shared__ float lds_m[MAX_PIECES * 32], lds_l[MAX_PIECES * 32];
    const uint32_t share = blockIdx.x % shares, at = blockIdx.x / shares, i = at % a.qt, merge = at / a.qt;
    const int32_t *mg = a.merges + (size_t)merge * PAGED_MERGE;
    if (mg[0] < 0) return;                   // (a plan that is over)
    const int32_t *sq = a.seqs + (size_t)mg[0] * PAGED_SEQ;
    const uint32_t tile = (uint32_t)mg[1] + i, kv = (uint32_t)mg[2], records = (uint32_t)mg[4], M = (uint32_t)sq[1] * a.group, tid = threadIdx.x;
    if (tile * 32u >= M) return;
    const size_t step = (size_t)mg[5] * a.qt * paged_record(a.cols, DP);
    const TQ_GLOBAL float *rec = (const TQ_GLOBAL float *)a.rec + ((size_t)mg[3] * a.qt + i) * paged_record(a.cols, DP);
    for (uint32_t j = tid; j < records * a.cols; j += MERGE_THREADS) {
        const uint32_t r = j / a.cols, c = j - r * a.cols;
        lds_m[j] = rec[r * step + c];
        lds_l[j] = rec[r * step + a.cols + c];
    }
    const uint32_t unit = share * MERGE_THREADS + tid, c = unit / (DP / 4u), d = (unit - c * (DP / 4u)) * 4u;
    const uint32_t m = tile * 32u + c;
    const bool some = c < a.cols && m < M && d < a.D;
    __syncthreads();
    if (!some) return;
    float top = MANY_NONE;
    for (uint32_t r = 0; r < records; ++r) top = fmaxf(top, lds_m[r * a.cols + c]);
    float sum = 0.f;
    tq_f4 o = {0.f, 0.f, 0.f, 0.f};
    const TQ_GLOBAL float *p = rec + 2u * a.cols + c * DP + d;
    for (uint32_t r0 = 0; r0 < records; r0 += 8u) {
        tq_f4 x[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) x[k] = *reinterpret_cast<const TQ_GLOBAL tq_f4 *>(p + min(r0 + k, records - 1u) * step);
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            if (r0 + k >= records) continue;
            const float own = lds_m[(r0 + k) * a.cols + c], l = lds_l[(r0 + k) * a.cols + c];
            const float f = own != MANY_NONE ? __builtin_amdgcn_exp2f(own - top) : l == 0.f ? 0.f : __builtin_nanf("");
            sum = fmaf(l, f, sum);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(x[k][e], f, o[e]);
        }
    }
    const float inv = 1.0f / sum;            // (a query sees its own token: a sum of zero is that of logits which are all -infinity, and 0 / 0 the result)
    const uint32_t token = m / a.group;
    const size_t first = ((size_t)((uint32_t)sq[0] + token) * (a.heads * a.group) + kv * a.group + (m - token * a.group)) * a.D + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    if (a.dtype == TQ_F32) {
        TQ_GLOBAL float *out = reinterpret_cast<TQ_GLOBAL float *>((TQ_GLOBAL uint8_t *)a.out) + first;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = o[e];
    } else {
        TQ_GLOBAL uint16_t *out = reinterpret_cast<TQ_GLOBAL uint16_t *>((TQ_GLOBAL uint8_t *)a.out) + first;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = a.dtype == TQ_F16 ? __builtin_bit_cast(uint16_t, (_Float16)o[e]) : __builtin_bit_cast(uint16_t, (__bf16)o[e]);
    }
}

bool supported(int D, int dtype, int bits_k, int bits_v) {
    if (dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16) return false;
    if (bits_k < 2 || bits_k > 8 || bits_v < 2 || bits_v > 8) return false;
    if (D == 64 || D == 128 || D == 256) return true;
    const int ik = 8 / bits_k, iv = 8 / bits_v;       // 65 to 96: whole groups of eight elements, and words of packed bytes
    return D > 64 && D <= 96 && !(D & 7) && !(D % ik) && !(D % iv) && !(D / ik & 3) && !(D / iv & 3);
}

// Times in quarters of a token of the kernel for one tile of 32 query vectors (14 cycles): what a block's packed tokens, its uncompressed ones and its start and end take.  (Clocked 128 wide: two tiles
// 22 cycles a packed token, 45 an uncompressed one, 50 thousand for start, joins and end.)
struct Costs {
    long long token, plain, block;
};
Costs costs(int qt, int dtype) {
    if (dtype == TQ_F32) return {12, 24, 10000};
    if (qt == 2) return {6, 14, 14000};
    return {4, 10, 10000};
}

struct Reach {                       // what a group of tiles sees of its sequence, in runs
    long long packed_from, packed_to, plain_from, plain_to;
    long long runs(const Costs &c) const { return (packed_to - packed_from + 31) / 32 * 32 * c.token + (plain_to - plain_from + 31) / 32 * 32 * c.plain; }
};
Reach reach(const int32_t *s, long long group, long long window, long long tile0, long long tiles, long long run) {
    const long long fresh = s[1], total = s[2], packed = s[3], first_pos = total - fresh + tile0 * 32 / group;
    long long last = ((tile0 + tiles) * 32 - 1) / group;
    if (last > fresh - 1) last = fresh - 1;
    const long long end = total - fresh + last + 1, lo = window && first_pos >= window ? first_pos - window + 1 : 0;
    Reach r;
    r.packed_from = lo / run * run;
    r.packed_to = packed;
    if (lo >= packed) r.packed_from = r.packed_to = 0;
    r.plain_from = lo > packed ? (lo - packed) / 32 * 32 : 0;
    r.plain_to = end - packed;
    return r;
}

struct Group {
    int32_t seq, tile0;
    Reach reach;
    long long cost;
};
struct Item {
    int32_t v[PAGED_ITEM];
    long long cost;
};
struct Shares {                      // how the blocks of a launch share its groups
    std::vector<Group> groups;
    long long piece = 0, time = -1;
    int qt = 1;
};

// Pieces of the longest group from one to MAX_PIECES: the number with the shortest time by the costs above.  As many rounds of blocks as the card takes, each as long as a block
// is on average, and no less than the longest block.
void share(Shares &best, std::vector<Group> &groups, int qt, int dtype, int heads, int cus) {
    const Costs c = costs(qt, dtype);
    long long longest = 0;
    for (Group &g : groups) {
        g.cost = g.reach.runs(c);
        if (g.cost > longest) longest = g.cost;
    }
    bool better = false;
    for (long long k = 1; k <= MAX_PIECES; ++k) {
        const long long piece = (longest + k - 1) / k;
        if (piece < 128 * c.token && k > 1) break;
        long long blocks = 0, all = 0, pieces = 1;
        for (const Group &g : groups) {
            const long long own = g.cost ? (g.cost + piece - 1) / piece : 1;
            blocks += own;
            all += g.cost + own * c.block;
            if (own > pieces) pieces = own;
        }
        blocks *= heads;
        all *= heads;
        const long long rounds = (blocks + cus - 1) / cus;
        long long time = rounds * (all / blocks);
        if (time < piece + c.block) time = piece + c.block;
        if (pieces > 1) time += 4000 + 120 * pieces;
        if (best.time < 0 || time < best.time) { best.time = time; best.piece = piece; best.qt = qt; better = true; }
        if (rounds > 16 && k > 1) break;
    }
    if (better) best.groups.swap(groups);
}

struct Plan {
    std::vector<Item> items;
    std::vector<int32_t> blocks, merges;
    long long records = 0, columns = 1;
    // pieces items[first] ... of one row, `step` from a record to the next
    void join(size_t first, int32_t seq, int32_t tile0, int32_t head, long long vectors, long long step) {
        const long long own = (long long)(items.size() - first);
        merges.insert(merges.end(), {seq, tile0, head, (int32_t)records, (int32_t)own, (int32_t)step, 0, 0});
        columns = std::max(columns, std::min(32LL, vectors));
    }
};

// Sequences with few query vectors: the rows (sequence, kv head) of a launch laid end to end and cut into as many equal shares as there are blocks, one a compute unit; a row that is cut is
// merged.  Or, where that takes less time, whole rows dealt out, the longest first to the block that has least.  Times in packed tokens of a block (4.6 ns: 64 x 16384 x 8 heads of 128 186 us, 64 x 8192
// 110): an uncompressed one three, an item's start and end 2000 (33 sequences of 500 to 16384 tokens 66 us; with 1100, 77), a merge 1200 and 25 a piece.  One sequence of 32768: 25 us in 256 shares, 151 uncut.
constexpr long long FEW_PLAIN = 3, FEW_ITEM = 2000, FEW_MERGE = 1200, FEW_PIECE = 25, FEW_LEAST = 512;
void plan_few(Plan &p, std::vector<Group> &groups, int heads, int cus, const int32_t *sequences, int group) {
    long long all = 0, longest = 0;
    for (Group &g : groups) {
        g.cost = g.reach.packed_to - g.reach.packed_from + FEW_PLAIN * ((g.reach.plain_to - g.reach.plain_from + 31) / 32 * 32);
        all += g.cost * heads;
        longest = std::max(longest, g.cost);
    }
    const long long rows = (long long)groups.size() * heads;
    // whole rows
    std::vector<std::pair<long long, std::vector<std::pair<int32_t, int32_t>>>> dealt((size_t)std::min<long long>(rows, cus));
    {
        std::vector<size_t> order(groups.size());
        for (size_t i = 0; i < order.size(); ++i) order[i] = i;
        std::stable_sort(order.begin(), order.end(), [&](size_t x, size_t y) { return groups[x].cost > groups[y].cost; });
        std::vector<std::pair<long long, size_t>> heap;          // (least first)
        for (size_t i = 0; i < dealt.size(); ++i) heap.emplace_back(0, i);
        const auto more = [](const std::pair<long long, size_t> &x, const std::pair<long long, size_t> &y) { return x > y; };
        for (size_t i : order)
            for (int h = 0; h < heads; ++h) {
                std::pop_heap(heap.begin(), heap.end(), more);
                heap.back().first += groups[i].cost + FEW_ITEM;
                dealt[heap.back().second].second.emplace_back((int32_t)i, h);
                dealt[heap.back().second].first = heap.back().first;
                std::push_heap(heap.begin(), heap.end(), more);
            }
    }
    long long best = 0, blocks = 0, room = 0;
    for (const auto &d : dealt) best = std::max(best, d.first);
    for (long long nb = cus; nb >= 1; nb /= 2) {
        long long share = (all + FEW_ITEM * (rows + nb) + nb - 1) / nb;
        share = std::max(share, std::max(longest / (MAX_PIECES - 4) + FEW_ITEM, FEW_LEAST + FEW_ITEM));
        const long long time = share + FEW_MERGE + FEW_PIECE * (longest / (share - FEW_ITEM) + 1);
        if (time < best) { best = time; blocks = nb; room = share; }
    }
    if (!blocks) {
        for (const auto &d : dealt) {
            p.blocks.push_back((int32_t)p.items.size());
            for (const auto &[i, h] : d.second) {
                const Group &g = groups[(size_t)i];
                p.items.push_back(Item{{g.seq, 0, (int32_t)g.reach.packed_from, (int32_t)g.reach.packed_to, (int32_t)g.reach.plain_from, (int32_t)g.reach.plain_to, -1, h}, 0});
            }
        }
        p.blocks.push_back((int32_t)p.items.size());
        return;
    }
    long long left = room;
    p.blocks.push_back((int32_t)p.items.size());
    for (const Group &g : groups)
        for (int h = 0; h < heads; ++h) {
            const Reach &r = g.reach;
            const size_t first = p.items.size();
            long long t = r.packed_from, u = r.plain_from, cost = g.cost;
            do {
                long long can = left - FEW_ITEM;
                if (can < FEW_LEAST && can < cost) {             // (the next block)
                    p.blocks.push_back((int32_t)p.items.size());
                    left = room;
                    can = left - FEW_ITEM;
                }
                if (cost <= can + FEW_LEAST / 2) can = cost;
                Item it{{g.seq, 0, (int32_t)t, 0, (int32_t)u, 0, -1, h}, 0};
                while (t < r.packed_to && it.cost < can) { t += 64; it.cost += 64; }
                if (t > r.packed_to) { it.cost -= t - r.packed_to; t = r.packed_to; }
                while (t >= r.packed_to && u < r.plain_to && it.cost < can) { u += 32; it.cost += 32 * FEW_PLAIN; }
                if (u > r.plain_to) u = r.plain_to;
                it.v[3] = (int32_t)t;
                it.v[5] = (int32_t)u;
                cost -= it.cost;
                left -= it.cost + FEW_ITEM;
                p.items.push_back(it);
            } while (t < r.packed_to || u < r.plain_to);
            if (p.items.size() - first > 1) {
                p.join(first, g.seq, 0, h, (long long)sequences[(size_t)g.seq * PAGED_SEQ + 1] * group, 1);
                for (size_t i = first; i < p.items.size(); ++i) p.items[i].v[6] = (int32_t)p.records++;
            }
        }
    p.blocks.push_back((int32_t)p.items.size());
}

// The others: a block an item and kv head.
void plan_many(Plan &p, const Shares &best, int heads, int dtype, const int32_t *sequences, int group) {
    const Costs c = costs(best.qt, dtype);
    const size_t begin = p.items.size();
    for (const Group &g : best.groups) {
        const Reach &r = g.reach;
        const long long k = g.cost ? (g.cost + best.piece - 1) / best.piece : 1, each = (g.cost + k - 1) / k;
        const size_t first = p.items.size();
        long long t = r.packed_from, u = r.plain_from;
        do {
            Item it{{g.seq, g.tile0, (int32_t)t, 0, (int32_t)u, 0, -1, -1}, 0};
            while (t < r.packed_to && it.cost < each) { t += 32; it.cost += 32 * c.token; }
            if (t > r.packed_to) t = r.packed_to;
            while (t >= r.packed_to && u < r.plain_to && it.cost < each) { u += 32; it.cost += 32 * c.plain; }
            if (u > r.plain_to) u = r.plain_to;
            it.v[3] = (int32_t)t;
            it.v[5] = (int32_t)u;
            p.items.push_back(it);
        } while (t < r.packed_to || u < r.plain_to);
        if (p.items.size() - first > 1) {
            const long long vectors = (long long)sequences[(size_t)g.seq * PAGED_SEQ + 1] * group - 32LL * g.tile0;
            for (int h = 0; h < heads; ++h) {
                p.join(first, g.seq, g.tile0, h, vectors, heads);
                p.merges[p.merges.size() - PAGED_MERGE + 3] += h;
            }
            for (size_t i = first; i < p.items.size(); ++i, p.records += heads) p.items[i].v[6] = (int32_t)p.records;
        }
    }
    // the longest first: what is short fills the gaps at the end
    std::stable_sort(p.items.begin() + (long)begin, p.items.end(), [](const Item &x, const Item &y) { return x.cost > y.cost; });
}

}  // namespace

extern "C" int tq_paged_supported(int head_dim, int dtype, int bits_k, int bits_v) { return supported(head_dim, dtype, bits_k, bits_v) ? 1 : 0; }

extern "C" int tq_paged_plan(const int32_t *sequences, long long n, int heads, int group, int window, int head_dim, int dtype, int page_tokens, int32_t *items, long long max_items,
                             int32_t *merges, long long max_merges, tq_paged_counts *counts) {
    if (!counts || (n > 0 && !sequences)) return TQ_ERR_NULL;
    if (n < 0 || heads < 1 || group < 1 || window < 0 || max_items < 0 || max_merges < 0) return TQ_ERR_SIZE;
    // Few query vectors a kv head: one token of up to 16 query heads, or some of fewer (16-bit elements; runs of 64 tokens, so pages of no less).
    const bool has_few = dtype != TQ_F32 && page_tokens >= 64 && (head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256);
    long long tiles = 0, most = 0, vectors = 0;
    for (long long b = 0; b < n; ++b) {
        const int32_t *s = sequences + b * PAGED_SEQ;
        if (s[0] < 0 || s[1] < 0 || s[2] < s[1] || s[3] < 0 || s[3] > s[2] - s[1] || s[4] < 0 || s[5] < 0) return TQ_ERR_SIZE;
        if ((long long)s[1] * group > 0x7fffffff - 64) return TQ_ERR_SIZE;
        const long long m = (long long)s[1] * group, t = (m + 31) / 32;
        tiles += t;
        if (has_few && m <= 16) vectors = std::max(vectors, m);
        else most = std::max(most, t);
    }
    *counts = tq_paged_counts{};
    counts->tiles = 1;
    if (!tiles) return TQ_OK;
    int cus = 0;
    if (tq_device_cus(cus)) cus = 256;
    try {
        Plan p;
        for (int few = 1; few >= 0; --few) {
            Shares best;
            // (two tiles a block share what is read and decoded; 96 wide they would spill)
            const bool two = !few && dtype != TQ_F32 && (head_dim == 64 || head_dim == 128) && most > 1;
            for (int qt = 1; qt <= (two ? 2 : 1); ++qt) {
                std::vector<Group> groups;
                for (long long b = 0; b < n; ++b) {
                    const int32_t *s = sequences + b * PAGED_SEQ;
                    const long long m = (long long)s[1] * group, t = (m + 31) / 32;
                    if ((has_few && m <= 16) != (few == 1)) continue;
                    for (long long t0 = 0; t0 < t; t0 += qt) groups.push_back(Group{(int32_t)b, (int32_t)t0, reach(s, group, window, t0, qt, few ? 64 : 32), 0});
                }
                if (groups.empty()) continue;
                if (few) plan_few(p, groups, heads, cus, sequences, group);
                else share(best, groups, qt, dtype, heads, cus);
            }
            if (few) counts->few = (long long)p.items.size();
            else if (!best.groups.empty()) {
                plan_many(p, best, heads, dtype, sequences, group);
                counts->tiles = best.qt;
            }
        }
        counts->items = (long long)p.items.size();
        counts->blocks = p.blocks.empty() ? 0 : (long long)p.blocks.size() - 1;
        counts->merges = (long long)p.merges.size() / PAGED_MERGE;
        counts->records = p.records;
        counts->columns = (int)p.columns;
        counts->vectors = (int)vectors;
        if (counts->items > 0x7fffffff / heads || p.records > 0x7fffffff || counts->merges > 0x7fffffff / 64) return TQ_ERR_SIZE;
        if (counts->items * PAGED_ITEM + (long long)p.blocks.size() > max_items * PAGED_ITEM || counts->merges > max_merges) return TQ_ERR_CAPACITY;
        if (!items || (counts->merges && !merges)) return TQ_ERR_NULL;
        for (size_t i = 0; i < p.items.size(); ++i) std::copy(p.items[i].v, p.items[i].v + PAGED_ITEM, items + i * PAGED_ITEM);
        std::copy(p.blocks.begin(), p.blocks.end(), items + p.items.size() * PAGED_ITEM);
        std::copy(p.merges.begin(), p.merges.end(), merges);
    } catch (...) {
        return TQ_ERR_CAPACITY;              // (no memory)
    }
    return TQ_OK;
}

extern "C" long long tq_paged_scratch(const tq_paged_counts *counts, int heads, int head_dim) {
    if (!counts) return TQ_ERR_NULL;
    if (head_dim < TQ_ANYDIM_MIN || head_dim > TQ_ANYDIM_MAX) return TQ_ERR_HEAD_DIM;
    if (heads < 1 || counts->records < 0 || counts->tiles < 1 || counts->tiles > 2 || counts->columns < 0 || counts->columns > 32) return TQ_ERR_SIZE;
    return counts->records * counts->tiles * (long long)paged_record((uint32_t)counts->columns, (uint32_t)TQ_PADDED_DIM(head_dim));
}

extern "C" int tq_paged_attend(const tq_paged_request *request, float *scratch, long long scratch_floats, void *stream) {
    if (!request) return TQ_ERR_NULL;
    const tq_paged_request &r = *request;
    const tq_paged_counts &n = r.counts;
    if (r.dtype != TQ_F32 && r.dtype != TQ_F16 && r.dtype != TQ_BF16) return TQ_ERR_DTYPE;
    if (r.bits_k < 1 || r.bits_k > 8 || r.bits_v < 1 || r.bits_v > 8) return TQ_ERR_BITS;
    if (!supported(r.head_dim, r.dtype, r.bits_k, r.bits_v)) return TQ_ERR_HEAD_DIM;
    if (r.heads < 1 || r.group < 1 || r.sliding_window < 0 || r.heads * (long long)r.group > 0x7fffffff) return TQ_ERR_SIZE;
    if (r.page_tokens < 32 || (r.page_tokens & (r.page_tokens - 1)) || r.page_tokens > 65536) return TQ_ERR_SIZE;
    if (r.page_tokens > 0x7fffffff / r.heads / (r.head_dim * 4)) return TQ_ERR_SIZE;
    if (!(r.softcap == 0.f || (r.softcap >= 0x1p-100f && r.softcap <= (r.dtype == TQ_F32 ? 0x1p100f : 1024.f))) || n.items < 0 || n.merges < 0 || n.records < 0) return TQ_ERR_SIZE;
    if (n.items == 0) return TQ_OK;
    if (n.few < 0 || n.few > n.items || n.blocks < 0 || n.blocks > 0x7fffffff || (n.few && (n.blocks < 1 || n.vectors < 1 || n.vectors > 16 || r.dtype == TQ_F32 || r.page_tokens < 64 || (r.head_dim & 31)))) return TQ_ERR_SIZE;
    if (n.items > 0x7fffffff / r.heads || n.tiles < 1 || n.tiles > 2 || n.columns < 1 || n.columns > 32) return TQ_ERR_SIZE;
    if (n.tiles == 2 && (r.dtype == TQ_F32 || (r.head_dim != 64 && r.head_dim != 128))) return TQ_ERR_SIZE;
    if (!r.queries || !r.out || !r.packed_pool || !r.plain_pool || !r.table_k || !r.table_v || !r.sequences || !r.tables || !r.items || (n.merges && (!r.merges || !scratch))) return TQ_ERR_NULL;
    const long long es = r.dtype == TQ_F32 ? 4 : 2;
    // vectors of a page as the kernels read them: runs of 32 tokens 16 bytes at a time (packed bytes of uneven dimensions: words)
    if ((((uintptr_t)r.packed_pool | (uintptr_t)r.plain_pool | (uintptr_t)r.table_k | (uintptr_t)r.table_v) & 15u) ||
        ((r.packed_page_stride | r.plain_page_stride | r.k_norms | r.v_idx | r.v_norms | r.plain_values) & 15) || ((uintptr_t)scratch & 15u) || ((uintptr_t)r.queries & (es - 1)) ||
        ((uintptr_t)r.out & (es - 1)) || (((uintptr_t)r.sequences | (uintptr_t)r.tables | (uintptr_t)r.items | (uintptr_t)r.merges | (uintptr_t)r.slopes) & 3u))
        return TQ_ERR_ALIGN;
    if (scratch_floats < tq_paged_scratch(&n, r.heads, r.head_dim)) return TQ_ERR_CAPACITY;
    TqPagedArgs a{};
    a.q = static_cast<const uint8_t *>(r.queries); a.out = static_cast<uint8_t *>(r.out);
    a.q_token = r.q_token; a.q_head = r.q_head;
    a.pool = static_cast<const uint8_t *>(r.packed_pool); a.plain = static_cast<const uint8_t *>(r.plain_pool);
    a.page_stride = r.packed_page_stride; a.plain_stride = r.plain_page_stride;
    a.k_norms = r.k_norms; a.v_idx = r.v_idx; a.v_norms = r.v_norms; a.plain_v = r.plain_values;
    a.table_k = static_cast<const uint8_t *>(r.table_k); a.table_v = static_cast<const uint8_t *>(r.table_v);
    a.seqs = r.sequences; a.tables = r.tables; a.items = r.items; a.merges = r.merges; a.slopes = r.slopes;
    a.rec = scratch;
    a.scale = r.scale; a.cap = r.softcap;
    a.heads = (uint32_t)r.heads; a.group = (uint32_t)r.group; a.D = (uint32_t)r.head_dim; a.dtype = (uint32_t)r.dtype;
    a.bits_k = (uint32_t)r.bits_k; a.bits_v = (uint32_t)r.bits_v;
    a.shift = (uint32_t)__builtin_ctz((unsigned)r.page_tokens);
    a.cols = (uint32_t)n.columns; a.window = (uint32_t)r.sliding_window;
    a.aligned = !((uintptr_t)r.queries & 15u) && !((r.q_token * es) & 15) && !((r.q_head * es) & 15);
    const int kt = r.dtype == TQ_BF16 ? 1 : 2, vt = r.dtype == TQ_F32 ? 2 : 1, dp = TQ_PADDED_DIM(r.head_dim), ik = 8 / r.bits_k, iv = 8 / r.bits_v;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    a.qt = (uint32_t)n.tiles;
    // the plan's first items are those with few query vectors
    const long long few = n.few;
    a.blocks = r.items + n.items * PAGED_ITEM;
    if (few && !a.aligned) return TQ_ERR_ALIGN;
    if (few) {
        const dim3 g((unsigned)n.blocks);
        if (dp == 64) tq_paged_few_launch_d64(ik, iv, g, s, a, (uint32_t)n.vectors);
        else if (dp == 96) tq_paged_few_launch_d96(ik, iv, g, s, a, (uint32_t)n.vectors);
        else if (dp == 128) tq_paged_few_launch_d128(ik, iv, g, s, a, (uint32_t)n.vectors);
        else tq_paged_few_launch_d256(ik, iv, g, s, a, (uint32_t)n.vectors);
    }
    if (n.items > few) {
        const dim3 g((unsigned)((n.items - few) * r.heads));
        TqPagedArgs rest = a;
        rest.items += few * PAGED_ITEM;
        if (dp == 64) tq_paged_launch_d64(ik, iv, g, s, rest, n.tiles, kt, vt);
        else if (dp == 96) tq_paged_launch_d96(ik, iv, g, s, rest, n.tiles, kt, vt);
        else if (dp == 128) tq_paged_launch_d128(ik, iv, g, s, rest, n.tiles, kt, vt);
        else tq_paged_launch_d256(ik, iv, g, s, rest, n.tiles, kt, vt);
    }
    if (n.merges) {
        const uint32_t qt = (uint32_t)n.tiles, shares = ((uint32_t)n.columns * (dp / 4u) + MERGE_THREADS - 1u) / MERGE_THREADS;
        const dim3 gm((unsigned)(n.merges * qt * shares)), t(MERGE_THREADS);
        if (dp == 64) hipLaunchKernelGGL((tq_paged_merge_kernel<64>), gm, t, 0, s, a, shares);
        else if (dp == 96) hipLaunchKernelGGL((tq_paged_merge_kernel<96>), gm, t, 0, s, a, shares);
        else if (dp == 128) hipLaunchKernelGGL((tq_paged_merge_kernel<128>), gm, t, 0, s, a, shares);
        else hipLaunchKernelGGL((tq_paged_merge_kernel<256>), gm, t, 0, s, a, shares);
    }
    return (int)hipGetLastError();
}
