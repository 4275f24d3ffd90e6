// Attention of sequences' new tokens over their pages (tq_paged.hip): what its kernels and the sources that instantiate them share.
//
// A sequence has `total` tokens, the last `fresh` of which are the step's and have queries; its first `packed` tokens lie in packed pages, the others uncompressed in plain
// ones.  Of the query heads that share a kv head, query vector m = token * group + head: the 32 columns of a tile are few tokens, so that what they see begins and ends close together.
#pragma once
#include "tq_many.h"

// Six numbers a sequence, eight apart: first row of its queries, its new tokens, all its tokens, packed ones, and where in the tables its packed and its plain pages begin
constexpr int PAGED_SEQ = 8, PAGED_ITEM = 8, PAGED_MERGE = 8;

struct TqPagedArgs {
    const uint8_t *q;                // new token i, query head j at i * q_token + j * q_head elements
    uint8_t *out;                    // dense [new tokens, query heads, D]
    long long q_token, q_head;
    const uint8_t *pool, *plain;     // this layer's part of page 0
    long long page_stride, plain_stride;             // bytes
    long long k_norms, v_idx, v_norms, plain_v;      // bytes from the layer's key codes (plain: keys)
    const uint8_t *table_k, *table_v;
    const int32_t *seqs, *tables;
    const int32_t *items;            // {sequence (-1, here as in the merges: nothing is done; blocks from -1 to -1 have no items), first tile, packed tokens from, to, plain ones from, to (multiples of 32, or the end), record or -1: all its tokens are here, kv head or -1: one block
                                     // each, whose record is the item's and so many on}
    const int32_t *blocks;           // items of sequences with few query vectors: block i has items [blocks[i], blocks[i + 1])
    const int32_t *merges;           // {sequence, first tile, kv head, first record, records, from one of them to the next, two unused}
    const float *slopes;             // [query heads], or null
    float *rec;                      // [records][qt][cols largest logits, cols sums, cols x DP value sums]
    float scale, cap;                // cap: 0 for none
    uint32_t heads, group, D, dtype, bits_k, bits_v, shift, cols, qt, window, aligned;      // qt: tiles of a record; window: 0 for none
};

namespace {

__host__ __device__ constexpr uint32_t paged_record(uint32_t cols, uint32_t dp) { return cols * (dp + 2u); }

}  // namespace

// Launches tq_paged_kernel for one padded head dimension; ipbk, ipbv = codes per byte (1, 2, 4), qt = tiles of 32 queries a block, kt, vt = fp16 terms on the key and value side
int tq_paged_launch_d64(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, int qt, int kt, int vt);
int tq_paged_launch_d96(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, int qt, int kt, int vt);
int tq_paged_launch_d128(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, int qt, int kt, int vt);
int tq_paged_launch_d256(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, int qt, int kt, int vt);
// Launches tq_paged_few_kernel for one head dimension; vectors: the most query vectors of a kv head of a sequence, at most 16
int tq_paged_few_launch_d64(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, uint32_t vectors);
int tq_paged_few_launch_d96(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, uint32_t vectors);
int tq_paged_few_launch_d128(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, uint32_t vectors);
int tq_paged_few_launch_d256(int ipbk, int ipbv, dim3 grid, hipStream_t s, const TqPagedArgs &a, uint32_t vectors);
