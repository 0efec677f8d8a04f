// hq_paged.h - what the paged cache's append and attention share (gfx950): the
// batch of new tokens, a row's sequence and position, a position's page, and
// the host's checks.
//
// Row t of a batch belongs to the sequence b with starts[b] <= t <
// starts[b+1]; its position is lengths[b] - n_b + (t - starts[b]).
#pragma once

#include "hq_device.h"
#include "hq_internal.h"

namespace hq {

// Positions a table's row may hold: the last chunk's end still fits an int.
constexpr int64_t kMaxPositions = 0x7fffff00;
// Blocks of 256 threads a launch can have.
constexpr int64_t kMaxBlocks = 0xffffff;

struct PagedBatch {
    const uint16_t* keys;        // [pages, kv_heads, page_size, D]
    const uint16_t* values;
    const int32_t* table;        // [sequences, max_pages]
    const int32_t* lengths;
    const int32_t* starts;       // nullable: row b is sequence b's only one
    int32_t* status;             // nullable (attention)
    int pages, page_size, shift; // shift: log2(page_size)
    int sequences, max_pages, tokens;
    int heads, kv_heads, groups;
};

// How many of the rising values at[1 .. n] are at most t: i (wave-uniform;
// every lane calls it; at[0] must exist), and at[i] and (for i < n) at[i + 1].
// Each round of loads leaves a 64th of them.  Of values that do not rise: some
// i from 0 to n.
__device__ __forceinline__ int wave_count_upto(const int32_t* at, int n, int t, int* here, int* next)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int end = n;
    int low = 0;
    while (n > kWave - 2) {
        const int stride = (n - 1) / kWave + 1;
        const int i = (lane + 1) * stride;
        const int past = __popcll(__ballot(i <= n && at[i <= n ? low + i : low] <= t));
        low += past * stride;
        n = min(stride - 1, n - past * stride);
    }
    const int v = at[min(low + lane, end)];
    const int past = __popcll(__ballot(lane >= 1 && lane <= n && v <= t));
    *here = __builtin_amdgcn_readlane(v, past);
    *next = __builtin_amdgcn_readlane(v, past + 1);
    return low + past;
}

// The sequence of a batch row (wave-uniform; every lane calls it), or -1; its first row and its rows.
__device__ __forceinline__ int paged_sequence(const PagedBatch& p, int t, int* first, int* count)
{
    if (!p.starts) {
        *first = t;
        *count = 1;
        return t < p.sequences ? t : -1;
    }
    int a, z;
    const int b = wave_count_upto(p.starts, p.sequences, t, &a, &z);
    *first = a;
    *count = z - a;
    return b >= p.sequences || a < 0 || a > t || z <= t || z > p.tokens ? -1 : b;
}

// The position of sequence b's i-th new row of `count`; negative: before the sequence.
__device__ __forceinline__ int paged_position(const PagedBatch& p, int b, int count, int i)
{
    const int64_t pos = int64_t(p.lengths[b]) - count + i;
    return int(max(pos, int64_t(-1)));
}

// The page of position j of sequence b, or -1.
__device__ __forceinline__ int paged_page(const PagedBatch& p, int b, int j)
{
    const int e = j >> p.shift;
    if (j < 0 || e >= p.max_pages) return -1;
    const int page = p.table[size_t(b) * p.max_pages + e];
    return page < p.pages ? page : -1;
}

// The arguments that append and attention share, checked on the host.
inline int paged_check(const hq_pages* c, const void* rows, const int32_t* starts, int tokens, int heads, const void* out,
                       PagedBatch* b)
{
    if (!c || !rows || !out || !c->keys || !c->values || !c->table || !c->lengths) return HQ_ERR_ARG;
    if (c->pages < 1 || c->kv_heads < 1 || c->sequences < 1 || c->max_pages < 1 || tokens < 0) return HQ_ERR_ARG;
    // (a grid's sizes: append has a block a token, and eight heads a block in y)
    if (tokens > kMaxBlocks || c->sequences > kMaxBlocks || c->kv_heads > 32768) return HQ_ERR_ARG;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return HQ_ERR_ARG;
    if (int64_t(c->max_pages) * c->page_size > kMaxPositions || int64_t(c->sequences) * c->max_pages > 0x7fffffff)
        return HQ_ERR_ARG;
    if (heads < 1 || heads % c->kv_heads || heads / c->kv_heads > 8) return HQ_ERR_ARG;
    if (c->head_dim != 16 && c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return HQ_ERR_ARG;
    if (!starts && tokens != c->sequences) return HQ_ERR_ARG;
    for (const void* q : {rows, out, static_cast<const void*>(c->keys), static_cast<const void*>(c->values)})
        if (reinterpret_cast<uintptr_t>(q) & 15u) return HQ_ERR_ALIGN;
    *b = PagedBatch{c->keys, c->values, c->table, c->lengths, starts, c->status, c->pages, c->page_size,
                    __builtin_ctz(unsigned(c->page_size)), c->sequences, c->max_pages, tokens, heads, c->kv_heads,
                    heads / c->kv_heads};
    return HQ_OK;
}

}  // namespace hq
