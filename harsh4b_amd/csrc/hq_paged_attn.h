// hq_paged_attn.h - the kernels of grouped-query attention of a batch's new
// tokens over the paged K/V cache on gfx950: hq_paged_attention, and with TREE
// hq_paged_attention_tree, whose new tokens are the nodes of drafted trees.
// No reference counterpart: the reference attends one contiguous cache per
// session, token by token (cpu_lightspark.py:389-422).
//
// For a query at position p and the positions j it sees:
//   s_j = q.k_j / sqrt(D),  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
// in one pass over the keys with the running maximum m and sum l.
//
// Precision: K and V are fp16, queries and outputs fp32, so the products run
// on the fp16 matrix cores with the fp32 side in two parts.  A query row is
// scaled by a power of two (its largest value into [2^9, 2^10)) and split
// q = hi + lo, both fp16: 22 bits, and what small values lose is below 2^-34
// of the row's largest.  The weights, scaled to up to 2^14, go as hi + lo
// likewise.  K and V enter exactly; scores, m, l and outputs are fp32.  A
// product costs two matrix instructions this way, against a rate of a
// sixteenth for the fp32 ones.
//
// Tiles: the rows of a tile are (token, head of the group) pairs of one
// sequence and kv head, so a K/V row is read once for all G heads.  Scores
// are computed transposed, S^T = K Q^T: a lane then holds scores of one row
// only, m and l are per lane, and the scores' registers are already the
// operand of O^T = V^T P^T (the order of the keys inside a product is free as
// long as V follows it).
//   small  up to 16 rows (single tokens): 16x16x32 products, each of a block's
//          4 waves on its own 32 keys, K and V straight to registers, the
//          waves' parts joined in LDS.  Bound by HBM: 32 chats of 2048 to
//          4096 positions (419 MB) in 82 us, 5.1 TB/s.
//   large  128 rows, 32 a wave: 32x32x16 products over chunks of 64 keys that
//          the block copies straight to LDS (V is transposed by the reads),
//          two buffers.  Bound by the matrix cores: 2048 tokens at 16384 (515
//          GFLOP, twice that in products of parts) in 867 us, 1.19 PFLOP/s,
//          the matrix cores busy for 72 % of the cycles at a clock of 1.6 GHz
//          that the power allows.
//
// Work: a tile's chunks are cut into pieces of about T = all work / kTarget
// chunks (per sequence: the same number of pieces for all its tiles), each a
// block; a tile of one piece writes its outputs, the others leave partial
// results (m, l, O) that a second launch joins.  Starts and lengths live on
// the device: every wave works the plan out from them, for many sequences a
// launch of its own.
//
// What matrix products cannot mask: 0 x NaN.  Values past a sequence's end are
// zeroed on the way in; where a row's result is not finite for another reason
// (an infinity or NaN in K or V, seen by it or by another row of the tile),
// the row is computed again by paged_row, in fp32 from the visible positions
// alone.
//
// Trees: a sequence's nodes stand in its last slots in their order, each after
// those above it, so a node sees no slot past its own: pieces and spans of
// chunks are those of as many tokens in a row, and only the chunks that reach
// past the tree's base (or lie at a window's edge) have masks: 32 keys' as one
// word, the slots before the base by their range, the nodes by the row's
// ancestor bits (tree_mask).  Trees of up to 32 rows (8 nodes of 4 heads) have
// a third kind of tile:
//   pair   two sets of 16 rows in each wave on the same keys, like small tiles
//          otherwise, with the query's parts split once for the block and its
//          remainders read from LDS (in registers 20 spill).  Bound by HBM: 32
//          chats of 2048 to 4096 positions and trees of up to 8 nodes (425 MB)
//          in 91 us, 4.7 TB/s.
// More rows go to large tiles, though of 33 to 64 half the waves only copy: 32
// chats of 16 nodes 100 us; the same rows as two waves a set, each with half of
// a chunk's keys, 131 (half the time for the copies of the next chunk), as two
// blocks of pairs that share an L2 113, as two sets of waves of one block 118
// (3 us of arithmetic a step of 32 keys).  A prompt's length of tree (2 x 64
// nodes at 40960, 140 GFLOP with the two parts) takes 133 us, 1.05 PFLOP/s.
#pragma once

#include <algorithm>

#include "hq_device.h"
#include "hq_internal.h"
#include "hq_paged.h"

namespace hq {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kChunkKeys = 64;
constexpr int kSmallRows = 16;
constexpr int kTileRows = 128;
// Rows of a tile that streams K and V to registers: 16, of trees up to 32.
template <bool TREE>
constexpr int kStreamRows = TREE ? 2 * kSmallRows : kSmallRows;
constexpr int kStreamNodes = 64;       // of a tree whose tiles do (its ancestors are held in registers)
// Pieces aimed at: one for each place on the chip (two blocks a CU), all
// started at once.  With twice as many, 16 windows of 1024 take 28 us (23), 3
// chats of 40960 92 (86), a question of 501 tokens after 7000 142 (129).
constexpr int kTarget = 512;
constexpr int kSmallMin = 2;           // fewest chunks of a small piece: a step of 32 keys a wave
constexpr int kLargeMin = 4;           // of a large one (100 tokens after 1024: 22.7 us, 23.6 with 2, 22.6 with 3)
// A chunk of a large tile counts as two of a small one: a step of 24 chats and
// a prompt's 250 tokens takes 75 us so, 82 with 1, 79 with 3 (over data that
// the last-level cache does not hold; where it does 67, 75, 72).  Of trees it
// counts as one: a batch of them waits for memory with either tile (32 chats of
// 16 nodes 102 us, 113 with 2 for large tiles; of 32 nodes 122, 125).
constexpr int kLargeCost = 2;
// Where there is a tile for every CU, large ones of so few chunks stay whole:
// a second block on the CU gains less than the join of the parts costs (4 x
// 256 tokens at 512: 34 us, 43 in two pieces each; at 1024 51, 59; 1000 tokens
// at 1000 48, 50).  At 32 chunks it goes both ways: 4 x 256 at 2048 83 whole,
// 87 cut; 1000 at 2000 80, 75.
constexpr int kLargeWhole = 16;
constexpr int kJoinThreads = 256;
constexpr int kJoinBlocks = 4096;
// Tables of up to 8 chunks (512 positions): no tile is cut, and there is no
// join to launch.  One chat of 256: 7.9 us (11.4 with both), of 480 10.5
// (11.7), of 736 12.8 (11.6), and the caller's time for a second launch, 3; 64
// chats of 480 25.9 (29.6).
constexpr int kWholeChunks = 8;
// From here on a launch of one block works the plan out for all sequences, and
// a piece looks itself up (1024 chats of 300: 278 us, 376 with a plan in every
// wave; 256: 82 and 83; 128: 42 and 38).
constexpr int kPlanSequences = 256;
constexpr int kPlanThreads = 1024;

struct PagedAttnParams {
    PagedBatch b;
    const float* query;          // [tokens, heads, D]
    float* out;
    int window, sinks;           // window 0: none
    int tile_tokens;             // tokens of a large tile
    int by_group;                // 65536 / groups + 1, for row_token
    // (TREE) sequences of few chunks have tiles of 16 rows, where each such tile of the batch has a CU: K and V are
    // read once a tile, but from a cache, and a step's arithmetic is half (one chat of 300 and 8 nodes 11.2 us, 15.2
    // in a pair)
    bool narrow;
    bool whole;                  // no tile is cut (short tables): no join
    bool planned;                // the plan is in plan_first, plan_item, plan_count
    int part_rows;               // rows of partial results there is room for
    int32_t* cut;                // [1] whether any tile is cut (0 too where starts fall)
    int32_t* plan_count;         // [1] sequences with rows
    int32_t* plan_first;         // [count + 1] the first piece of each, and how many there are
    int4* plan_item;             // [count] sequence, pieces a tile, first partial row
    int2* desc;                  // [tokens, kv_heads] 2 * pieces + small, first partial row
    float* part_o;               // [part_rows, D]
    float2* part_ml;             // [part_rows] m (of the scores times log2 e), l
    TreeBatch tree;              // (TREE)
};

// The token of a tile's row: r / groups (exact: r < 128, groups <= 8).
__device__ __forceinline__ int row_token(const PagedAttnParams& p, int r) { return (r * p.by_group) >> 16; }

// a / b for 0 <= a < 2^24 and 0 < b < 2^24 (exact: the quotient by the
// reciprocal is off by one at most; a third of a division's instructions, and
// the plan makes five one after another).
__device__ __forceinline__ int quotient(int a, int b)
{
    const int q = int(float(a) * __builtin_amdgcn_rcpf(float(b)));
    const int rest = a - q * b;
    return q + (rest >= b ? 1 : 0) - (rest < 0 ? 1 : 0);
}

// Whether the query at position `pos` sees position j (pages aside).
__device__ __forceinline__ bool paged_visible(int pos, int j, int window, int sinks)
{
    return j <= pos && (window == 0 || j > pos - window || j < sinks);
}

// Keys below the k-th of a mask's 32.
__device__ __forceinline__ uint32_t below(int k) { return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1u; }

// Which of the slots j0 .. j0 + 31 a tree's node sees (pages aside): a node of
// depth `depth` in slot `slot`, of a sequence whose tree's first node is batch
// row `first`, in slot `base`.  nodes: the node's ancestor bits from the node
// in slot max(j0, base) on.
__device__ __forceinline__ uint32_t tree_mask(const PagedAttnParams& p, int depth, int first, int base, int slot, int j0,
                                              uint32_t nodes)
{
    const int pos = base + depth, to_base = base - j0, to_slot = slot + 1 - j0;
    uint32_t before = below(to_base);
    if (p.window > 0) before &= ~below(max(0, pos - p.window + 1) - j0) | below(p.sinks - j0);
    nodes = to_base >= 32 ? 0u : nodes << max(to_base, 0);
    // (a path longer than the window: by the nodes' positions)
    if (p.window > 0 && depth >= p.window)
        for (uint32_t left = nodes & below(to_slot); left; left &= left - 1) {
            const int i = __builtin_ctz(left);
            const int above = p.tree.depths[first + i - to_base];
            if (depth - above >= p.window && base + above >= p.sinks) nodes &= ~(1u << i);
        }
    return depth < 0 ? 0u : (before | nodes) & below(to_slot);
}

// A node's ancestor bits from node `from` on.
__device__ __forceinline__ uint32_t tree_bits(const PagedAttnParams& p, int row, int from)
{
    const uint32_t* bits = p.tree.ancestors + size_t(row) * kTreeWords;
    const int word = min(from >> 5, kTreeWords);
    const uint32_t low = bits[min(word, kTreeWords - 1)], high = bits[min(word + 1, kTreeWords - 1)];
    return uint32_t((uint64_t(word + 1 < kTreeWords ? high : 0u) << 32 | (word < kTreeWords ? low : 0u)) >> (from & 31));
}

constexpr float kLog2e = 0x1.715476p+0f;
constexpr float kWeightScale = 16384.0f;           // 2^14
// Large tiles keep an old maximum until a score passes it by 2^8: their
// weights are 2^6 e^(s-m), up to 2^14.
constexpr float kLargeShift = 6.0f, kLargeScale = 64.0f, kLargeSlack = 8.0f;

// ------------------------------------------------------------- one row, fp32
// One query row over positions [lo, hi) of sequence b, kv head h, in one wave:
// a lane scores one position of 64 at a time and holds D/64 of the output's
// values.  `seen`: whether anything was visible.
// `visible_at(j)`: whether the row sees position j.
template <int D, class F>
__device__ void paged_row(const PagedAttnParams& p, const float* q, int b, int h, int lo, int hi, F&& visible_at,
                          float& m, float& l, float (&o)[2], bool& seen)
{
    const int lane = threadIdx.x & (kWave - 1);
    const float scale = 1.0f / __builtin_sqrtf(float(D));
    const size_t head = size_t(p.b.page_size) * D;
    for (int base = lo; base < hi; base += kWave) {
        const int j = base + lane;
        const int page = j < hi ? paged_page(p.b, b, j) : -1;
        const bool visible = page >= 0 && visible_at(j);
        if (!__any(visible)) continue;
        seen = true;
        const size_t row = (size_t(max(page, 0)) * p.b.kv_heads + h) * head + size_t(j & (p.b.page_size - 1)) * D;
        float s = -__builtin_inff();
        if (visible) {
            const uint4* k = reinterpret_cast<const uint4*>(p.b.keys + row);
            float acc = 0.0f;
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
                const uint4 v = k[c];
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc = __builtin_fmaf(q[8 * c + 2 * i], f16_to_f32(uint16_t(w[i])), acc);
                    acc = __builtin_fmaf(q[8 * c + 2 * i + 1], f16_to_f32(uint16_t(w[i] >> 16)), acc);
                }
            }
            s = acc * scale;
        }
        const float top = fmaxf(m, wave_max64_all(s));
        const float alpha = m == top ? 1.0f : expf(m - top);
        const float e = !visible || (top == -__builtin_inff() && s == top) ? 0.0f : expf(s - top);
        l = l * alpha;
        o[0] *= alpha;
        o[1] *= alpha;
        uint64_t left = __ballot(visible);
        while (left) {
            const int i = __builtin_ctzll(left);
            left &= left - 1;
            const float pi = __shfl(e, i, kWave);
            const size_t vrow = (uint64_t(uint32_t(__shfl(int(row >> 32), i, kWave))) << 32) |
                                uint32_t(__shfl(int(uint32_t(row)), i, kWave));
            l += pi;
            if (lane < D) o[0] = __builtin_fmaf(pi, f16_to_f32(p.b.values[vrow + lane]), o[0]);
            if (D == 128) o[1] = __builtin_fmaf(pi, f16_to_f32(p.b.values[vrow + lane + 64]), o[1]);
        }
        m = top;
    }
}

// ---------------------------------------------------------------------- plan
// The chunks of 64 positions that a tile's queries, at positions pa .. pb,
// see: chunks 0 .. sink - 1, then `first` and on, `count` in all.
struct Span {
    int sink, first, count;
    __device__ __forceinline__ int chunk(int c) const { return c < sink ? c : first + (c - sink); }
};

__device__ __forceinline__ Span span_of(const PagedAttnParams& p, int pa, int pb)
{
    if (pb < 0) return Span{0, 0, 0};
    const int end = min(pb + 1, p.b.max_pages << p.b.shift);
    const int last = (end - 1) / kChunkKeys + 1;
    const int low = p.window > 0 && pa >= p.window ? pa - p.window + 1 : 0;
    const int first = low / kChunkKeys;
    const int sunk = min(p.sinks, low);
    const int sink = min(min(first, last), sunk / kChunkKeys + (sunk % kChunkKeys != 0));
    return Span{sink, first, sink + max(0, last - first)};
}

struct SequencePlan {
    int first, n;                // rows
    int length;                  // (a negative one counts as 0)
    // chunks: the last tile's.  Under a window a tile before it may have a few
    // more (it may be fuller, and lie across one more border of chunks): its
    // pieces are that much longer, and no bound relies on it.
    int tile_tokens, tiles, chunks;
    bool small;
    int cost;                    // of a chunk
};

template <bool TREE>
__device__ __forceinline__ SequencePlan sequence_plan(const PagedAttnParams& p, int b, bool* fall)
{
    SequencePlan s;
    s.first = b;
    s.n = 1;
    s.small = true;
    s.tile_tokens = s.tiles = 1;
    s.length = max(0, p.b.lengths[b]);
    if (TREE || p.b.starts) {
        const int a = p.b.starts[b], z = p.b.starts[b + 1];
        *fall |= a > z;
        s.first = a;
        s.n = a < 0 || a >= z || z > p.b.tokens ? 0 : z - a;
        s.small = s.n <= kStreamRows<TREE> / p.b.groups;
        s.tile_tokens = s.small ? max(1, s.n) : p.tile_tokens;
        s.tiles = s.small ? min(s.n, 1) : quotient(s.n + s.tile_tokens - 1, s.tile_tokens);
    }
    s.cost = s.small || TREE ? 1 : kLargeCost;
    const int origin = s.length - s.n;
    // (a tree's nodes may all be roots: their positions are at or past the base)
    s.chunks = s.n ? span_of(p, TREE ? origin : origin + (s.tiles - 1) * s.tile_tokens, s.length - 1).count : 0;
    if (TREE && p.narrow && s.chunks <= kWholeChunks && s.n > kSmallRows / p.b.groups && s.n <= kStreamNodes) {
        s.small = true;
        s.tile_tokens = kSmallRows / p.b.groups;
        s.tiles = quotient(s.n + s.tile_tokens - 1, s.tile_tokens);
    }
    return s;
}

// A block's piece: one tile (rows of one sequence and kv head), some of its chunks.
struct Piece {
    int b, head;
    int first, n;                // the tile's tokens
    int pos;                     // position (slot) of its first token (negative: before the sequence)
    int base;                    // of the sequence's first new token, which is row first - (pos - base)
    int length;
    int pieces, split, part;     // part: first partial row of this piece
    bool small;
    __device__ __forceinline__ int position(int i) const { return max(pos + i, -1); }
    // (TREE) what its i-th token, of depth `depth`, sees of the slots j0 .. j0 + 31; nodes: see tree_mask
    __device__ __forceinline__ uint32_t mask(const PagedAttnParams& p, int i, int depth, int j0, uint32_t nodes) const
    {
        return tree_mask(p, depth, first - (pos - base), base, position(i), j0, nodes);
    }
    __device__ __forceinline__ uint32_t bits(const PagedAttnParams& p, int i, int j0) const
    {
        return tree_bits(p, first + i, max(0, j0 - base));
    }
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Inclusive prefix sum over the wave (every lane active): row shifts, then the
// row totals broadcast to the rows above.
__device__ __forceinline__ int wave_prefix(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);    // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast 31 into rows 2 and 3
    return v;
}

// Pieces a sequence's tiles are cut in for pieces of about `target` chunks;
// tiles: of the whole batch (of one kv head).
template <bool TREE>
__device__ __forceinline__ int cuts_of(const PagedAttnParams& p, const SequencePlan& s, int target, int tiles)
{
    if (p.whole || (s.small && s.tiles > 1)) return 1;
    if (!s.small && s.chunks <= kLargeWhole && int64_t(tiles) * p.b.kv_heads >= kTarget / 2) return 1;
    const int size = max(target, s.small ? kSmallMin : kLargeMin * s.cost);
    return max(1, int(float(s.chunks * s.cost) / float(size) + 0.5f));
}

// Sequence b's piece number `local`, of `cuts` a tile; its partial rows start at first_part.
template <bool TREE>
__device__ __forceinline__ void place_piece(const PagedAttnParams& p, const SequencePlan& s, int b, int local, int cuts,
                                            int first_part, Piece& out)
{
    out.b = b;
    out.pieces = cuts;
    out.small = s.small;
    out.length = s.length;
    int rest, tile;
    if (out.small) {                                         // (one tile, but for narrow ones, of one piece each)
        rest = quotient(local, p.b.kv_heads);
        out.split = TREE && cuts == 1 ? 0 : rest;
        tile = TREE && cuts == 1 ? rest : 0;
    } else {
        // The longest first; and since blocks i and i + 256 share a CU, where
        // all have a place the second 256 the other way round (a prompt of
        // 1800 tokens: 82 us, 85.5 without; of 2048: 94, 97.5).
        const int all = s.tiles * cuts * p.b.kv_heads;
        if (all <= kTarget && local >= kTarget / 2) local = kTarget / 2 + all - 1 - local;
        rest = quotient(local, p.b.kv_heads);
        const int done = quotient(rest, out.pieces);
        out.split = rest - done * out.pieces;
        tile = s.tiles - 1 - done;
    }
    tile = uniform(tile);
    out.split = uniform(out.split);
    out.head = uniform(local - rest * p.b.kv_heads);
    out.first = s.first + tile * s.tile_tokens;
    out.n = min(s.tile_tokens, s.n - tile * s.tile_tokens);
    out.base = out.length - s.n;
    out.pos = out.base + tile * s.tile_tokens;
    out.part = first_part + (((tile * p.b.kv_heads + out.head) * out.pieces) + out.split) *
                                (out.small ? kStreamRows<TREE> : kTileRows);
}

// Chunks a piece should have, for all the batch's chunks (of one kv head).
__device__ __forceinline__ int piece_target(const PagedAttnParams& p, int64_t units)
{
    return int(min((units * p.b.kv_heads + kTarget - 1) / kTarget, int64_t(0x40000000)));
}

// The plan of many sequences, in one block: the sequences with rows in order,
// their first pieces and partial rows.
template <bool TREE>
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedAttnParams p)
{
    constexpr int WAVES = kPlanThreads / kWave;
    __shared__ unsigned long long all_units;
    __shared__ int falls, all_tiles;
    __shared__ int3 wave_sum[WAVES];
    const int t = threadIdx.x, lane = t & (kWave - 1), wave = t / kWave;
    if (t == 0) all_units = 0, falls = all_tiles = 0;
    __syncthreads();
    bool fall = false;
    int64_t units = 0;
    int sum = 0;
    SequencePlan mine{};
    for (int b = t; b < p.b.sequences; b += kPlanThreads) {
        mine = sequence_plan<TREE>(p, b, &fall);
        units += int64_t(mine.tiles) * mine.chunks * mine.cost;
        sum += mine.tiles;
    }
    if (sum) atomicAdd(&all_tiles, sum);
    if (units) atomicAdd(&all_units, static_cast<unsigned long long>(units));
    if (fall) falls = 1;
    __syncthreads();
    int count = 0, pieces = 0, rows = 0;
    if (!falls) {
        const int target = piece_target(p, int64_t(all_units)), tiles = all_tiles;
        for (int base = 0; base < p.b.sequences; base += kPlanThreads) {
            const int b = base + t;
            if (p.b.sequences > kPlanThreads && b < p.b.sequences) mine = sequence_plan<TREE>(p, b, &fall);
            if (b >= p.b.sequences) mine.tiles = 0;
            const int cuts = cuts_of<TREE>(p, mine, target, tiles);
            const int here = mine.tiles * cuts * p.b.kv_heads;
            const int part = cuts > 1 ? here * (mine.small ? kStreamRows<TREE> : kTileRows) : 0;
            const uint64_t has = __ballot(here > 0);
            const int incl = wave_prefix(here), part_incl = wave_prefix(part);
            __syncthreads();                   // (wave_sum's last readers)
            if (lane == kWave - 1) wave_sum[wave] = make_int3(int(__popcll(has)), incl, part_incl);
            __syncthreads();
            int3 before = make_int3(count, pieces, rows);
            for (int w = 0; w < WAVES; ++w) {
                const int3 v = wave_sum[w];
                if (w < wave) before.x += v.x, before.y += v.y, before.z += v.z;
                count += v.x;
                pieces += v.y;
                rows += v.z;
            }
            if (here > 0) {                    // (a sequence with rows: no more than there are tokens)
                const int at = before.x + int(__popcll(has & ((uint64_t(1) << lane) - 1)));
                p.plan_first[at] = before.y + incl - here;
                p.plan_item[at] = make_int4(b, cuts, before.z + part_incl - part, 0);
            }
        }
    }
    if (t == 0) {
        p.plan_first[count] = pieces;
        *p.plan_count = count;
        *p.cut = rows > 0;
    }
}

// The work of block `q`, the same in every wave; false: none.
template <bool TREE>
__device__ __forceinline__ bool plan_piece(const PagedAttnParams& p, int q, Piece& out)
{
    const int lane = threadIdx.x & (kWave - 1);
    if (!TREE && p.whole && !p.b.starts) {     // a tile a block: nothing to count
        out.b = uniform(quotient(q, p.b.kv_heads));
        out.head = q - out.b * p.b.kv_heads;
        out.first = out.b;
        out.n = 1;
        out.length = uniform(max(0, p.b.lengths[out.b]));
        out.pos = out.base = out.length - 1;
        out.pieces = 1;
        out.split = out.part = 0;
        out.small = true;
        return true;
    }
    bool fall = false;
    if (p.planned) {
        const int count = *p.plan_count;
        int first, next;
        const int i = wave_count_upto(p.plan_first, count, q, &first, &next);
        if (i >= count) return false;
        const int4 item = p.plan_item[i];
        const int b = uniform(item.x);
        place_piece<TREE>(p, sequence_plan<TREE>(p, b, &fall), b, q - first, uniform(item.y), uniform(item.z), out);
        return true;
    }
    int64_t units = 0;
    int tiles = 0;
    SequencePlan mine{};
    for (int base = 0; base < p.b.sequences; base += kWave) {
        if (base + lane < p.b.sequences) {
            mine = sequence_plan<TREE>(p, base + lane, &fall);
            units += int64_t(mine.tiles) * mine.chunks * mine.cost;
            tiles += mine.tiles;
        }
    }
    if (__any(fall)) {
        if (q == 0 && threadIdx.x == 0) *p.cut = 0;
        return false;
    }
    // (the sum of 64 in two parts that fit an int each)
    const int low = __builtin_amdgcn_readfirstlane(wave_isum64(int(units & 0xFFFFFF)));
    const int high = __builtin_amdgcn_readfirstlane(wave_isum64(int(min(units >> 24, int64_t(0xFFFFFF)))));
    int target = piece_target(p, (int64_t(high) << 24) + low);
    tiles = uniform(wave_isum64(tiles));
    // Rounded, they may be a few more pieces than places, and those run alone
    // at the end: larger ones that all have a place, if up to twice the size
    // gives such (800 tokens after 8200: 233 us, 273 without; 400 after 4600
    // 84, 108; 700 after 800 56, 63).  Of up to 64 sequences, whose plans the
    // lanes hold; more would be worked out anew for every size tried.  Where no
    // such size gives it (one long sequence among short ones that take most of
    // the places), the first stays, and the launch has the blocks: trees of 16
    // nodes on 46 chats of 300 and one of 40960 take 82 us so, 104 with sizes up
    // to four times the first and 1172 uncut (of 8 nodes 74, 70 and 564; 62 of
    // 3000 and one of 40960 207, 377 and 640).
    if (p.b.sequences <= kWave && !p.whole && int64_t(tiles) * p.b.kv_heads <= kTarget) {
        int larger = target;
        bool fits = false;
        for (int k = 0; k < 7 && !fits; ++k) {
            fits = uniform(wave_isum64(mine.tiles * cuts_of<TREE>(p, mine, larger, tiles))) * p.b.kv_heads <= kTarget;
            if (fits) target = larger;
            else larger += larger / 8 + 1;
        }
    }
    int pieces = 0, rows = 0;
    bool got = false;
    for (int base = 0; base < p.b.sequences; base += kWave) {
        const bool in = base + lane < p.b.sequences;
        if (p.b.sequences > kWave && in) mine = sequence_plan<TREE>(p, base + lane, &fall);
        if (!in) mine.tiles = 0;
        const int cuts = cuts_of<TREE>(p, mine, target, tiles);
        const int here = mine.tiles * cuts * p.b.kv_heads;
        const int part = cuts > 1 ? here * (mine.small ? kStreamRows<TREE> : kTileRows) : 0;
        const int incl = wave_prefix(here), part_incl = wave_prefix(part);
        const uint64_t found = __ballot(q >= pieces + incl - here && q < pieces + incl);
        got |= found != 0;
        if (found) {
            const int src = __builtin_ctzll(found);
            auto from = [&](int v) { return __builtin_amdgcn_readlane(v, src); };
            SequencePlan s;
            s.first = from(mine.first);
            s.n = from(mine.n);
            s.length = from(mine.length);
            s.tile_tokens = from(mine.tile_tokens);
            s.tiles = from(mine.tiles);
            s.small = from(mine.small);
            place_piece<TREE>(p, s, base + src, q - from(pieces + incl - here), from(cuts), from(rows + part_incl - part), out);
            if (q != 0) return true;
        }
        pieces += __builtin_amdgcn_readlane(incl, kWave - 1);
        rows += __builtin_amdgcn_readlane(part_incl, kWave - 1);
    }
    if (q == 0 && threadIdx.x == 0) *p.cut = rows > 0;     // (block 0 goes through all sequences)
    return got;
}

// ------------------------------------------------------------- query operands
// The exponent that takes values of at most `top` to below 2^10 (0 for a row of zeros or without a finite maximum).
__device__ __forceinline__ int row_exponent(float top)
{
    if (!(top > 0.0f) || top == __builtin_inff()) return 0;
    return max(-100, int(__builtin_amdgcn_frexp_expf(top)) - 10);   // (2^e / sqrt(D) stays a normal number)
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// What an fp16 pair leaves of the two values it was rounded from: a - h.lo and
// b - h.hi, one v_fma_mix_f32 each (it reads an fp16 half; the compiler makes
// a conversion and a subtraction).
__device__ __forceinline__ float2v residual(float a, float b, half2v h)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, h);
    float2v r;
    float x, y;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(x) : "v"(u), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y) : "v"(u), "v"(b));
    r[0] = x;
    r[1] = y;
    return r;
}

// Eight values within fp16's range as hi + lo.
__device__ __forceinline__ void split8(const float (&w)[8], half8& hi, half8& lo)
{
    uint4v a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2v x = {w[2 * i], w[2 * i + 1]};
        const half2v h = __builtin_convertvector(x, half2v);
        const float2v rest = residual(x[0], x[1], h);
        a[i] = __builtin_bit_cast(uint32_t, h);
        b[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, half2v));
    }
    hi = __builtin_bit_cast(half8, a);
    lo = __builtin_bit_cast(half8, b);
}

// Over the lanes 16, 32 and 48 away (the four that hold one row of a small tile), in every lane.
__device__ __forceinline__ float max_over_g(float v)
{
    unsigned a = __builtin_bit_cast(unsigned, v), b = a;
    swap32(a, b);
    v = fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    a = b = __builtin_bit_cast(unsigned, v);
    swap16(a, b);
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float sum_over_g(float v)
{
    unsigned a = __builtin_bit_cast(unsigned, v), b = a;
    swap32(a, b);
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    a = b = __builtin_bit_cast(unsigned, v);
    swap16(a, b);
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

__device__ __forceinline__ bool finite(float x) { return __builtin_fabsf(x) < __builtin_inff(); }

// The result of one row, by one wave in fp32 (see paged_row), as this piece's output or part.
template <int D, bool TREE>
__device__ void redo_row(const PagedAttnParams& p, const Piece& w, const Span& span, int c0, int c1, int r)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int token = row_token(p, r);
    const size_t row = size_t(w.first + token) * p.b.heads + w.head * p.b.groups + (r - token * p.b.groups);
    float m = -__builtin_inff(), l = 0.0f, o[2] = {0.0f, 0.0f};
    bool seen = false;
    const int64_t end = int64_t(p.b.max_pages) << p.b.shift;
    for (int c = c0; c < c1; ++c) {
        const int at = span.chunk(c) * kChunkKeys;
        paged_row<D>(p, p.query + row * D, w.b, w.head, at, int(min(end, int64_t(at) + kChunkKeys)),
                     [&](int j) {
                         if constexpr (!TREE) return paged_visible(w.position(token), j, p.window, p.sinks);
                         const int depth = p.tree.depths[w.first + token];
                         return (w.mask(p, token, depth, j, w.bits(p, token, j)) & 1u) != 0;
                     },
                     m, l, o, seen);
    }
    if (w.pieces == 1) {
        if (lane < D) p.out[row * D + lane] = seen ? o[0] / l : 0.0f;
        if (D == 128) p.out[row * D + lane + 64] = seen ? o[1] / l : 0.0f;
        return;
    }
    const size_t at = size_t(w.part + r);
    if (lane < D) p.part_o[at * D + lane] = o[0];
    if (D == 128) p.part_o[at * D + lane + 64] = o[1];
    // (a row whose scores are all -inf has no softmax: the join finds the NaN where nothing else counts)
    if (lane == 0) p.part_ml[at] = make_float2(m * kLog2e, seen && m == -__builtin_inff() ? __builtin_nanf("") : l);
}

// ---------------------------------------------------------------- small tiles
template <int D, bool TREE>
struct SmallShared {
    float o[4][kSmallRows][D + 4];             // (+ 4: the rows start in different banks)
    float m[4][kSmallRows], l[4][kSmallRows];
    int bad[kStreamRows<TREE>];
    // two sets' query parts, lane by lane, and factors (see small_tile)
    half8 q[TREE ? 2 : 1][TREE ? (D + 31) / 32 : 1][2][TREE ? kWave : 1];
    float c[2][kSmallRows];
};

// R sets of 16 rows on the same keys.
template <int D, bool TREE, int R>
__device__ void small_tile(const PagedAttnParams& p, const Piece& w, const Span& span, int c0, int c1,
                           SmallShared<D, TREE>& S)
{
    constexpr int STEPS = (D + 31) / 32;       // products over the dims
    constexpr int VEC = D / 16;                // dims a lane holds of a V row
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n = lane & 15, g = lane >> 4;
    const int G = p.b.groups;
    const int rows = w.n * G;
    const int ps = p.b.page_size;
    bool mine[R];
    int token[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = 16 * r + n;
        mine[r] = row < rows;
        token[r] = mine[r] ? row_token(p, row) : 0;
    }
    // (of a tree: no row sees less than all slots before the base, none more than those up to its own)
    const int pos_min = TREE ? w.base - 1 : w.position(0), pos_max = w.position(w.n - 1);
    float4v acc[R][VEC];
    float m[R], l[R];
    bool seen[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[r][i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
        m[r] = -__builtin_inff();
        l[r] = 0.0f;
        seen[r] = false;
    }

    // this wave's steps of 32 keys: wave, wave + 4, ...; pages of 32 of them at a time, two a step, in a register
    const int steps = 2 * (c1 - c0);
    const size_t head_stride = size_t(ps) * D;
    auto key_of = [&](int t) { return span.chunk(c0 + (t >> 1)) * kChunkKeys + (t & 1) * 32; };
    auto pages_of = [&](int k) {                       // k: the wave's k-th step, first of 32
        const int t = wave + 4 * (k + (lane >> 1));
        return t < steps ? paged_page(p.b, w.b, key_of(t) + 16 * (lane & 1)) : -1;
    };
    half8 kf[2][STEPS];
    uint32_t vf[8][VEC >= 2 ? VEC / 2 : 1];
    auto base_of = [&](int page, int j) {
        return (size_t(max(page, 0)) * p.b.kv_heads + w.head) * head_stride + size_t(j & (ps - 1)) * D;
    };
    auto load_k = [&](int pg0, int pg1, int j) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint16_t* k = p.b.keys + base_of(t ? pg1 : pg0, j + 16 * t);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int d = 32 * s + 8 * g;
                kf[t][s] = D >= 32 || d < D ? *reinterpret_cast<const half8*>(k + n * D + d) : half8{};
            }
        }
    };
    auto load_v = [&](int pg0, int pg1, int j) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint16_t* v = p.b.values + base_of(t ? pg1 : pg0, j + 16 * t);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t* a = v + (4 * g + i) * D + VEC * n;
                if constexpr (VEC == 8) {
                    const uint4v x = *reinterpret_cast<const uint4v*>(a);
#pragma unroll
                    for (int d = 0; d < 4; ++d) vf[4 * t + i][d] = x[d];
                } else if constexpr (VEC == 4) {
                    const uint2 x = *reinterpret_cast<const uint2*>(a);
                    vf[4 * t + i][0] = x.x;
                    vf[4 * t + i][1] = x.y;
                } else if constexpr (VEC == 2) {
                    vf[4 * t + i][0] = *reinterpret_cast<const uint32_t*>(a);
                } else {
                    vf[4 * t + i][0] = *a;
                }
            }
        }
    };
    const int own = steps > wave ? (steps - wave + 3) / 4 : 0;
    // (TREE) the rows' depths and ancestors: of at most kStreamNodes
    int depth[TREE ? R : 1];
    uint64_t bits[TREE ? R : 1];
    if constexpr (TREE) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            depth[r] = p.tree.depths[w.first + token[r]];
            bits[r] = *reinterpret_cast<const uint64_t*>(p.tree.ancestors + size_t(w.first + token[r]) * kTreeWords);
        }
    }
    // This lane's query row (n), dims 32 s + 8 g ..: its loads, the page
    // table's and then the first step's of K and V are under way together.
    // Of two sets wave 0 and 2 split the first for all, 1 and 3 the second.
    constexpr bool SHARED = R > 1;
    const int q_set = SHARED ? wave & 1 : 0;
    float4v x[STEPS][2];
    {
        const int i = SHARED && q_set ? 1 : 0, of = i ? token[R - 1] : token[0];
        const int head = (i ? mine[R - 1] : mine[0]) ? 16 * i + n - of * G : 0;
        const float* q = p.query + (size_t(w.first + of) * p.b.heads + w.head * G + head) * D;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int d = D >= 32 ? 32 * s + 8 * g : 8 * (g & 1);
            x[s][0] = *reinterpret_cast<const float4v*>(q + d);
            x[s][1] = *reinterpret_cast<const float4v*>(q + d + 4);
        }
    }
    int pg = own ? pages_of(0) : -1;
    int pg0 = __builtin_amdgcn_readlane(pg, 0), pg1 = __builtin_amdgcn_readlane(pg, 1);
    int j0 = own ? key_of(wave) : 0;
    if (own) {
        load_k(pg0, pg1, j0);
        load_v(pg0, pg1, j0);
    }
    half8 qhi[R][STEPS], qlo[SHARED ? 1 : R][STEPS];   // (of two sets the remainders stay in LDS)
    float c[R];
    {
        const bool used = D >= 32 || g < 2;   // (a lane of no row: the tile's first row, not stored)
        float top = 0.0f;
        float y[STEPS][8];
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[s][i] = used ? x[s][i >> 2][i & 3] : 0.0f;
                top = fmaxf(top, __builtin_fabsf(y[s][i]));
            }
        top = max_over_g(top);
        const int e = row_exponent(top);
        const float down = __builtin_ldexpf(1.0f, -e);
        c[0] = __builtin_ldexpf(kLog2e / __builtin_sqrtf(float(D)), e);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (SHARED && STEPS > 1 && (s & 1) != wave >> 1) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[s][i] *= down;
            half8 hi, lo;
            split8(y[s], hi, lo);
            if constexpr (SHARED) {
                S.q[q_set][s][0][lane] = hi;
                S.q[q_set][s][1][lane] = lo;
            } else {
                qhi[0][s] = hi;
                qlo[0][s] = lo;
            }
        }
    }
    if constexpr (SHARED) {
        if (g == 0 && wave < 2) S.c[q_set][n] = c[0];
        lds_sync();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            c[r] = S.c[r][n];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) qhi[r][s] = S.q[r][s][0][lane];
        }
    }
    for (int k = 0; k < own; ++k) {
        // the next step's pages
        const int kn = k + 1;
        int next0 = -1, next1 = -1, nj = 0;
        if (kn < own) {
            if ((kn & 31) == 0) pg = pages_of(kn);
            next0 = __builtin_amdgcn_readlane(pg, 2 * (kn & 31));
            next1 = __builtin_amdgcn_readlane(pg, 2 * (kn & 31) + 1);
            nj = key_of(wave + 4 * kn);
        }
        float4v s[R][2];
        if constexpr (SHARED) {
            uint32_t at = lane;                // (the compiler would read the remainders once for all steps)
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
            // (products that follow one another go to different sums)
#pragma unroll
            for (int d = 0; d < STEPS; ++d) {
                half8 q[R];
#pragma unroll
                for (int r = 0; r < R; ++r) q[r] = S.q[r][d][1][at];
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        s[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][d], q[r], s[r][t], 0, 0, 0);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        s[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][d], qhi[r][d], s[r][t], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                s[0][t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int d = 0; d < STEPS; ++d) {
                    s[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][d], qlo[0][d], s[0][t], 0, 0, 0);
                    s[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][d], qhi[0][d], s[0][t], 0, 0, 0);
                }
            }
        }
        if (kn < own) load_k(next0, next1, nj);
        // lane (n, g): row n, keys j0 + 16 t + 4 g + i
        const bool all = pg0 >= 0 && pg1 >= 0 && j0 + 31 <= pos_min &&
                         (p.window == 0 || j0 > pos_max - p.window || j0 + 32 <= p.sinks);
        half8 hi[R], lo[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (!all) {
                const int pos = w.position(token[r]);
                const int from = max(0, j0 - w.base);
                const uint32_t nodes = TREE && from < kStreamNodes ? uint32_t(bits[TREE ? r : 0] >> from) : 0u;
                const uint32_t mask = TREE ? w.mask(p, token[r], depth[TREE ? r : 0], j0, nodes) : 0u;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = j0 + 16 * t + 4 * g + i;
                        const bool there = (t ? pg1 : pg0) >= 0;
                        const bool visible = there && (TREE ? ((mask >> (16 * t + 4 * g + i)) & 1u) != 0
                                                            : paged_visible(pos, j, p.window, p.sinks));
                        s[r][t][i] = visible ? s[r][t][i] : -__builtin_inff();
                        seen[r] |= visible;
                        if (r == 0 && (!there || j >= w.length))
#pragma unroll
                            for (auto& x : vf[4 * t + i]) x = 0;
                    }
            } else {
                seen[r] = true;
            }
            float top = fmaxf(fmaxf(fmaxf(s[r][0][0], s[r][0][1]), fmaxf(s[r][0][2], s[r][0][3])),
                              fmaxf(fmaxf(s[r][1][0], s[r][1][1]), fmaxf(s[r][1][2], s[r][1][3])));
            top = max_over_g(top);
            top = fmaxf(m[r], top);
            const float safe = top == -__builtin_inff() ? 0.0f : top;
            if (__any(top > m[r])) {
                const float alpha = exp2_fast((m[r] - safe) * c[r]);
                l[r] *= alpha;
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[r][i] *= alpha;
                m[r] = top;
            }
            const float shift = 14.0f - safe * c[r];
            float e[8];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[4 * t + i] = exp2_fast(__builtin_fmaf(s[r][t][i], c[r], shift));
                    l[r] += e[4 * t + i];
                }
            split8(e, hi[r], lo[r]);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            // dims VEC n + i: half (i & 1) of word i / 2 of each key
            uint4v a;
#pragma unroll
            for (int d = 0; d < 4; ++d)
                a[d] = __builtin_amdgcn_perm(vf[2 * d + 1][i / 2], vf[2 * d][i / 2], (i & 1) ? 0x07060302u : 0x05040100u);
            const half8 v = __builtin_bit_cast(half8, a);
#pragma unroll
            for (int r = 0; r < R; ++r)
                acc[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo[r], acc[r][i], 0, 0, 0);
#pragma unroll
            for (int r = 0; r < R; ++r)
                acc[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi[r], acc[r][i], 0, 0, 0);
        }
        if (kn < own) load_v(next0, next1, nj);
        pg0 = next0;
        pg1 = next1;
        j0 = nj;
    }
    // join the four waves, a set of rows at a time: lane (n, g) holds row n, dims VEC (4 g + i) + v
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] = sum_over_g(l[r]);
        if (TREE && depth[TREE ? r : 0] < 0) seen[r] = false;                    // (of a tree that is none)
        const uint64_t any_seen = __ballot(seen[r]);
        const bool row_seen = ((any_seen | (any_seen >> 16) | (any_seen >> 32) | (any_seen >> 48)) >> n) & 1;
        if (r > 0) lds_sync();                                 // (the last set is joined)
        if (g == 0) {
            S.m[wave][n] = m[r] * c[r];
            S.l[wave][n] = row_seen ? l[r] : -1.0f;            // (-1: this wave saw nothing of the row)
            if (wave == 0) S.bad[16 * r + n] = 0;
        }
        if (mine[r]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float* to = &S.o[wave][n][VEC * (4 * g + i)];
                if constexpr (VEC >= 4) {
#pragma unroll
                    for (int v = 0; v < VEC; v += 4)
                        *reinterpret_cast<float4v*>(to + v) = float4v{acc[r][v][i], acc[r][v + 1][i], acc[r][v + 2][i],
                                                                      acc[r][v + 3][i]};
                } else {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) to[v] = acc[r][v][i];
                }
            }
        }
        lds_sync();
        for (int i = threadIdx.x; i < min(rows - 16 * r, 16) * (D / 4); i += kBlock) {
            const int in = i / (D / 4), d = 4 * (i % (D / 4)), tile_row = 16 * r + in;
            float sm[4], sl[4];
            float4v so[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                sm[v] = S.m[v][in];
                sl[v] = S.l[v][in];
                so[v] = *reinterpret_cast<const float4v*>(&S.o[v][in][d]);
            }
            const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
            float sum = 0.0f;
            float4v o = {0.0f, 0.0f, 0.0f, 0.0f};
            bool none = true;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float f = sm[v] == -__builtin_inff() ? 0.0f : exp2_fast(sm[v] - top);
                if (sl[v] != -1.0f) {
                    none = false;
                    sum += sl[v] * f;
                }
                o += so[v] * f;
            }
            const bool bad = !none && (!finite(sum) || sum == 0.0f || !finite(o[0]) || !finite(o[1]) || !finite(o[2]) ||
                                       !finite(o[3]));
            if (bad) S.bad[tile_row] = 1;
            const float f = none ? 0.0f : w.pieces == 1 ? 1.0f / sum : 1.0f / kWeightScale;
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = none ? 0.0f : o[k] * f;
            const int of = row_token(p, tile_row);
            const size_t row = size_t(w.first + of) * p.b.heads + w.head * G + (tile_row - of * G);
            if (w.pieces == 1) {
                *reinterpret_cast<float4v*>(p.out + row * D + d) = o;
            } else {
                const int part = w.part + tile_row;
                *reinterpret_cast<float4v*>(p.part_o + size_t(part) * D + d) = o;
                if (d == 0) p.part_ml[part] = none ? make_float2(-__builtin_inff(), 0.0f) : make_float2(top, sum * f);
            }
        }
    }
    wait_all_memory();                         // (a row done again is stored again, by another wave)
    __syncthreads();
    for (int r = wave; r < rows; r += 4)
        if (S.bad[r]) redo_row<D, TREE>(p, w, span, c0, c1, r);
}

// ---------------------------------------------------------------- large tiles
// Two groups of 16 lanes read four pieces of four rows of V at a time: 16 of
// the 16 places of 256 bytes (a row of D = 128, two of D = 64, ...).
template <int D>
__host__ __device__ constexpr int v_flip(int key)
{
    return D == 128 ? 4 * (key & 3) : D == 64 ? 4 * ((key >> 1) & 1) : 0;
}

template <int D>
struct LargeShared {
    // [key][dim], the 16-byte pieces of a row permuted by the key: piece i of K in place i ^ (key & 15), of V in
    // i ^ v_flip(key) (both within the row), so that the rows a product reads together lie in different banks
    alignas(256) uint16_t k[2][kChunkKeys * D];
    alignas(256) uint16_t v[2][kChunkKeys * D];
};

typedef short short4v __attribute__((ext_vector_type(4)));

// Four keys of one dim a lane from V rows in LDS: lane i of 16 gives the
// address of row i / 4, dims 4 (i % 4) .. + 3 and receives dim i of the four.
__device__ __forceinline__ short4v read_transposed(uint32_t lds)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(uintptr_t(lds)));
}

template <int D, bool TREE>
__device__ void large_tile(const PagedAttnParams& p, const Piece& w, const Span& span, int c0, int c1,
                           LargeShared<D>& S)
{
    constexpr int STEPS = D / 16;
    constexpr int DT = D < 32 ? 1 : D / 32;
    constexpr int PIECES = D / 8;              // 16-byte pieces of a K row
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n = lane & 31, g = lane >> 5;
    const int G = p.b.groups;
    const int ps = p.b.page_size;
    const int rows = w.n * G;
    const int r = 32 * wave + n;               // this lane's row
    const bool mine = r < rows;
    const int token = mine ? row_token(p, r) : 0;
    const size_t out_row = size_t(w.first + token) * p.b.heads + w.head * G + (mine ? r - token * G : 0);
    half8 qhi[STEPS], qlo[STEPS];
    float c = 0.0f;
    auto split_query = [&] {
        const float* q = p.query + out_row * D;
        float top = 0.0f;
        float x[STEPS][8];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const float4v a = *reinterpret_cast<const float4v*>(q + 16 * s + 8 * g);
            const float4v b = *reinterpret_cast<const float4v*>(q + 16 * s + 8 * g + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {      // (a lane of no row: the tile's first row, not stored)
                x[s][i] = a[i];
                x[s][4 + i] = b[i];
                top = fmaxf(top, fmaxf(__builtin_fabsf(x[s][i]), __builtin_fabsf(x[s][4 + i])));
            }
        }
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const int e = row_exponent(top);
        const float down = __builtin_ldexpf(1.0f, -e);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[s][i] *= down;
            split8(x[s], qhi[s], qlo[s]);
        }
        c = __builtin_ldexpf(kLog2e / __builtin_sqrtf(float(D)), e);
    };
    if constexpr (!TREE) split_query();
    const int depth = TREE ? p.tree.depths[w.first + token] : 0;
    const bool active = 32 * wave < rows;      // (wave-uniform)
    const int pos_min = TREE ? w.base - 1 : uniform(w.position(row_token(p, min(32 * wave, rows - 1))));
    const int pos_max = uniform(w.position(row_token(p, min(32 * wave + 31, rows - 1))));

    float16v acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[i][k] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f, shift = kLargeShift;
    bool seen = false;

    const size_t head_stride = size_t(ps) * D;
    auto base_of = [&](int page, int j) {
        return (size_t(max(page, 0)) * p.b.kv_heads + w.head) * head_stride + size_t(j & (ps - 1)) * D;
    };
    // pages of 16 chunks at a time, 4 parts of 16 keys each, in a register:
    // of chunks pg_first ..; a chunk's are taken when its values are fetched
    int pg = -1, pg_first = c0;
    auto pages_of = [&](int cc) {
        const int at = cc + (lane >> 2);
        return at < c1 ? paged_page(p.b, w.b, span.chunk(at) * kChunkKeys + 16 * (lane & 3)) : -1;
    };
    auto opaque = [](uint32_t v) {             // (the compiler would keep everything made from it in registers)
        asm volatile("" : "+v"(v));
        return v;
    };
    // Rows 16 wave .. + 15 of chunk cc (from position `at`), contiguous in their page, to LDS: copy
    // i takes PER rows, lane (row, place) the piece that belongs in that place.
    // The permutations work bit by bit, so copy i's piece is copy 0's with
    // bits of the row 16 i / COPIES flipped.
    constexpr int PER = 64 / PIECES < 16 ? 64 / PIECES : 16, COPIES = 16 / PER;
    auto copy_k = [&](int page, int at, int cc) {
        const uint16_t* k = p.b.keys + base_of(page, at + 16 * wave);
        const uint32_t to = lds_addr(&S.k[cc & 1][16 * wave * D]);
        const uint32_t x = opaque(lane), row = x / PIECES, place = x % PIECES;
        const uint32_t from = (row * PIECES + (place ^ (row & (PIECES - 1)))) * 16;
#pragma unroll
        for (int i = 0; i < COPIES; ++i)
            if (D >= 32 || row < 16)
                dma16(k, (from ^ (16 * ((i * PER) & (PIECES - 1)))) + 1024 * i, to + 1024 * i);
    };
    auto copy_v = [&](int page, int at, int cc) {
        const int j0 = at + 16 * wave;
        const uint16_t* v = p.b.values + base_of(page, j0);
        uint16_t* to = &S.v[cc & 1][16 * wave * D];
        const int there = page < 0 ? 0 : w.length - j0;                  // rows of the 16; the others are zeros
        const uint32_t x = opaque(lane), copy_row = x / PIECES;
        const uint32_t from = (copy_row * PIECES + ((x % PIECES) ^ v_flip<D>(copy_row))) * 16;
        if (there >= 16) {
#pragma unroll
            for (int i = 0; i < COPIES; ++i)
                if (D >= 32 || copy_row < 16)
                    dma16(v, (from ^ (16 * v_flip<D>(i * PER))) + 1024 * i, lds_addr(to) + 1024 * i);
        } else {
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                if (D < 32 && copy_row >= 16) continue;
                if (int(copy_row) < there - i * PER) {
                    dma16(v, (from ^ (16 * v_flip<D>(i * PER))) + 1024 * i, lds_addr(to) + 1024 * i);
                } else {
                    const uint32_t z = opaque(0);
                    *reinterpret_cast<uint4v*>(to + 512 * i + 8 * lane) = uint4v{z, z, z, z};
                }
            }
        }
    };
    // Operands from LDS: unit i of the scores of half t (dims 16 i ..), unit i
    // of the products with V of half t (16 keys and 32 dims).  The addresses
    // are a lane's base with bits of the piece flipped; the bases are made
    // anew for every step (opaque to the compiler, which would keep all of
    // them in registers).
    typedef __attribute__((address_space(3))) const half8* lds_half8;
    constexpr uint32_t kBufBytes = kChunkKeys * D * 2;
    const int lane16 = lane & 15;
    const uint32_t k_lane = lds_addr(&S.k[0][0]) + n * 2 * D + ((g ^ (n & (PIECES - 1))) & (PIECES - 1)) * 16;
    const int v_key = 4 * g + (lane16 >> 2);
    const uint32_t v_lane = lds_addr(&S.v[0][0]) + v_key * 2 * D + 8 * (lane16 & 1) +
                            (((2 * ((lane >> 4) & 1) + ((lane16 & 3) >> 1)) & (PIECES - 1)) ^ v_flip<D>(v_key)) * 16;
    auto k_unit = [&](uint32_t base, int i) { return *lds_half8(uintptr_t(base ^ (32 * i))); };
    auto v_unit = [&](uint32_t base, int i) {
        const uint32_t at = (base ^ ((64 * (i % DT)) & (2 * D - 1))) + (i / DT) * 32 * D;
        // (the rows 8 keys on have the same permutation)
        struct { short4v a, b; } both = {read_transposed(at), read_transposed(at + 16 * D)};
        return __builtin_bit_cast(half8, both);
    };
    struct Weights {
        uint4v hi[2], lo[2];                   // [16 keys], two fp16 a word
    };
    // The weights `now` of the scores `cur` side by side with the scores
    // `next` of half kt in K buffer kbuf (matrix instructions of one and the
    // arithmetic of the other overlap only where they alternate in the
    // program), then O += V P of half vt in buffer vbuf.  Lane (n, g) of the
    // scores: row n, keys 32 t + 8 (i / 4) + 4 g + i % 4.
    constexpr int VUNITS = 2 * DT;
    auto weigh = [&](const float16v& cur, int pair, Weights& now) {
        const int at = 2 * pair;
        const float2v e = {exp2_fast(__builtin_fmaf(cur[at], c, shift)),
                           exp2_fast(__builtin_fmaf(cur[at + 1], c, shift))};
        l += e[0];
        l += e[1];
        asm volatile("" : "+v"(l));            // (summed here: the compiler would keep all of e for later)
        const half2v h = __builtin_convertvector(e, half2v);
        const float2v rest = residual(e[0], e[1], h);
        const half2v f = __builtin_convertvector(rest, half2v);
        now.hi[at / 8][at % 8 / 2] = __builtin_bit_cast(uint32_t, h);
        now.lo[at / 8][at % 8 / 2] = __builtin_bit_cast(uint32_t, f);
    };
    auto step = [&](auto with_scores, int kbuf, int kt, float16v& next, auto with_weights, const float16v& cur,
                    int vbuf, int vt) {
        constexpr bool SC = decltype(with_scores)::value, WE = decltype(with_weights)::value;
        constexpr int UNITS = SC ? STEPS : 1;
        constexpr int PAIRS = 8 / UNITS;
        // (a wave at its matrix instructions goes before one at its masks and
        // maxima: the SIMD's two waves then fall out of step, and overlap)
        __builtin_amdgcn_s_setprio(1);
        constexpr int AHEAD = 2, V_AHEAD = 3, VSET = V_AHEAD + 1;      // units whose operands are read ahead
        Weights now{};
        half8 ka[AHEAD + 1], va[VSET];
        uint32_t kb = 0, vb = 0;
        if constexpr (SC) {
            kb = opaque(k_lane + kbuf * kBufBytes + kt * 64 * D);
            unrolled<(AHEAD < UNITS ? AHEAD : UNITS)>([&](auto u) { ka[decltype(u)::value] = k_unit(kb, decltype(u)::value); });
#pragma unroll
            for (int i = 0; i < 16; ++i) next[i] = 0.0f;
        }
        unrolled<UNITS>([&](auto u) {
            constexpr int i = decltype(u)::value;
            if constexpr (SC) __builtin_amdgcn_sched_barrier(0);
            if constexpr (SC && i + AHEAD < UNITS) ka[(i + AHEAD) % (AHEAD + 1)] = k_unit(kb, i + AHEAD);
            if constexpr (WE && i == UNITS - 1) {
                vb = opaque(v_lane + vbuf * kBufBytes + vt * 64 * D);
                unrolled<(V_AHEAD < VUNITS ? V_AHEAD : VUNITS)>([&](auto q) { va[decltype(q)::value] = v_unit(vb, decltype(q)::value); });
            }
            const half8 k = ka[i % (AHEAD + 1)];
            if constexpr (SC) next = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qlo[i], next, 0, 0, 0);
            if constexpr (WE)
                unrolled<PAIRS>([&](auto q) {
                    if constexpr (2 * decltype(q)::value < PAIRS) weigh(cur, i * PAIRS + decltype(q)::value, now);
                });
            if constexpr (SC) next = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qhi[i], next, 0, 0, 0);
            if constexpr (WE)
                unrolled<PAIRS>([&](auto q) {
                    if constexpr (2 * decltype(q)::value >= PAIRS) weigh(cur, i * PAIRS + decltype(q)::value, now);
                });
        });
        if constexpr (WE) {
            unrolled<VUNITS>([&](auto u) {
                constexpr int i = decltype(u)::value;
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (i + V_AHEAD < VUNITS) va[(i + V_AHEAD) % VSET] = v_unit(vb, i + V_AHEAD);
                const half8 v = va[i % VSET];
                acc[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, __builtin_bit_cast(half8, now.lo[i / DT]), acc[i % DT], 0, 0, 0);
                acc[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, __builtin_bit_cast(half8, now.hi[i / DT]), acc[i % DT], 0, 0, 0);
            });
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    // masks, and a new maximum where the old one is left too far behind
    auto settle = [&](int at, int t, uint32_t there, float16v& s) {
        const int j0 = at + 32 * t;
        const uint32_t both = (there >> (2 * t)) & 3u;
        const bool all = both == 3u && j0 + 31 <= pos_min &&
                         (p.window == 0 || j0 > pos_max - p.window || j0 + 32 <= p.sinks);
        if (!all) {
            // of the lane's first key; its others lie 8 (i / 4) + i % 4 further
            const int x = int(opaque(lane)), g = x >> 5;
            const int row = 32 * wave + (x & 31);
            if constexpr (TREE) {
                const int i = row < rows ? row_token(p, row) : 0;
                const uint32_t nodes = j0 + 32 > w.base ? w.bits(p, i, j0) : 0u;
                const uint32_t mask = w.mask(p, i, depth, j0, nodes) >> (4 * g);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const bool visible = ((both >> (i >> 3)) & 1u) & ((mask >> (8 * (i >> 2) + (i & 3))) & 1u);
                    s[i] = visible ? s[i] : -__builtin_inff();
                    seen |= visible;
                }
            } else {
                const int pos = w.position(row < rows ? row_token(p, row) : 0);
                const int low = p.window > 0 ? max(0, pos - p.window + 1) : 0;     // first position of the row's window
                const int to_pos = int(opaque(pos - j0 - 4 * g)), to_low = int(opaque(low - j0 - 4 * g));
                const int to_sinks = int(opaque(p.sinks - j0 - 4 * g));
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int at = 8 * (i >> 2) + (i & 3);
                    const bool visible = ((both >> (i >> 3)) & 1u) & (at <= to_pos) & ((at >= to_low) | (at < to_sinks));
                    s[i] = visible ? s[i] : -__builtin_inff();
                    seen |= visible;
                }
            }
        } else {
            seen = true;
        }
        float top = fmaxf(fmaxf(s[0], s[1]), s[2]);
#pragma unroll
        for (int i = 3; i < 15; i += 2) top = fmaxf(fmaxf(top, s[i]), s[i + 1]);
        top = fmaxf(top, s[15]);
        unsigned a = __builtin_bit_cast(unsigned, top), b = a;
        swap32(a, b);
        top = fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
        // (m = -inf: the first that is seen; both -inf: NaN, not taken)
        if (__any((top - m) * c > kLargeSlack)) {
            top = fmaxf(m, top);
            const float safe = top == -__builtin_inff() ? 0.0f : top;
            const float alpha = exp2_fast((m - safe) * c);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] *= alpha;
            m = top;
            shift = kLargeShift - safe * c;
        }
    };
    auto there_of = [&](int cc) { return uint32_t(__ballot(pg >= 0) >> (4 * (cc - pg_first))) & 15u; };

    if (c0 < c1) {
        // The scores run half a chunk (32 keys) ahead of the weights.  Two
        // barriers a chunk: one lets K of chunk cc + 2 take cc's place, one V.
        pg = pages_of(c0);
        uint32_t there = there_of(c0);
        int page = __builtin_amdgcn_readlane(pg, wave);        // of chunk c0, then of cc + 1
        // positions of chunks cc and cc + 1
        int at = span.chunk(c0) * kChunkKeys, at_next = span.chunk(c0 + 1) * kChunkKeys;
        copy_k(page, at, c0);
        copy_v(page, at, c0);
        page = __builtin_amdgcn_readlane(pg, 4 + wave);
        if (c0 + 1 < c1) copy_k(page, at_next, c0 + 1);
        if constexpr (TREE) split_query();     // (beside the first copies)
        wait_all_memory();
        lds_sync();
        // copies of chunk cc + 1's V, and (once K of cc is read) of cc + 2's K
        auto stage_v = [&](int cc) { copy_v(page, at_next, cc + 1); };
        auto stage_k = [&](int cc) {
            lds_sync();                        // K of cc is read
            there = there_of(cc + 1);
            at = at_next;
            at_next = span.chunk(cc + 2) * kChunkKeys;
            if (cc + 2 < c1) {
                if (cc + 2 - pg_first == 16) {
                    pg_first = cc + 2;
                    pg = pages_of(pg_first);
                }
                page = __builtin_amdgcn_readlane(pg, 4 * (cc + 2 - pg_first) + wave);
                copy_k(page, at_next, cc + 2);
            }
        };
        auto arrived = [&] {
            // (waiting for V of cc + 1 alone, with K of cc + 2 on its way, gained nothing)
            wait_all_memory();
            lds_sync();
        };
        if (active) {
            float16v sa, sb;
            step(yes, c0 & 1, 0, sa, no, sa, 0, 0);
            settle(at, 0, there, sa);
            for (int cc = c0; cc < c1 - 1; ++cc) {
                // here: sa the scores of cc's first half; K of cc and cc + 1, V of cc in LDS
                stage_v(cc);
                step(yes, cc & 1, 1, sb, yes, sa, cc & 1, 0);
                settle(at, 1, there, sb);
                stage_k(cc);
                step(yes, (cc + 1) & 1, 0, sa, yes, sb, cc & 1, 1);
                settle(at, 0, there, sa);
                arrived();
            }
            step(yes, (c1 - 1) & 1, 1, sb, yes, sa, (c1 - 1) & 1, 0);
            settle(at, 1, there, sb);
            step(no, 0, 0, sa, yes, sb, (c1 - 1) & 1, 1);
        } else {                               // rows of no token: only the wave's share of the copies
            for (int cc = c0; cc < c1 - 1; ++cc) {
                stage_v(cc);
                stage_k(cc);
                arrived();
            }
        }
    }
    l += __shfl_xor(l, 32, kWave);
    // lane (n, g): row n, dims 32 dt + 8 (i / 4) + 4 g + i % 4
    const int x = int(opaque(lane)), n_end = x & 31, g_end = x >> 5, r_end = 32 * wave + n_end;
    const bool mine_end = r_end < rows;
    const int token_end = mine_end ? row_token(p, r_end) : 0;
    const size_t row_end = size_t(w.first + token_end) * p.b.heads + w.head * G + (mine_end ? r_end - token_end * G : 0);
    float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // NaN where an output is not finite
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (32 * dt + 8 * (i >> 2) < D) zero[i & 3] = __builtin_fmaf(acc[dt][i], 0.0f, zero[i & 3]);
    const uint64_t was_seen = __ballot(seen);
    bool none = (((was_seen | (was_seen >> 32)) >> n_end) & 1) == 0;
    if (TREE) none |= depth < 0;               // (of a tree that is none)
    // (a row that sees nothing has zeros, unless its tile holds something not finite)
    const bool ok = (zero[0] + zero[1]) + (zero[2] + zero[3]) == 0.0f && (none || (finite(l) && l != 0.0f));
    const uint64_t wrong = __ballot(mine_end && !ok);
    const uint32_t again = uint32_t(wrong | (wrong >> 32));
    if (mine_end && ((again >> n_end) & 1) == 0) {
        const bool direct = w.pieces == 1;
        float* to = direct ? p.out + row_end * D : p.part_o + size_t(w.part + r_end) * D;
        const float f = none ? 0.0f : direct ? 1.0f / l : 1.0f / kLargeScale;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int dim = 32 * dt + 8 * i + 4 * g_end;
                if (dim < D) {
                    float4v x;
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = acc[dt][4 * i + k] * f;
                    *reinterpret_cast<float4v*>(to + dim) = x;
                }
            }
        if (!direct && g_end == 0)
            p.part_ml[w.part + r_end] = none ? make_float2(-__builtin_inff(), 0.0f)
                                         : make_float2(m * c, l * (1.0f / kLargeScale));
    }
    for (uint32_t left = again; left; left &= left - 1)
        redo_row<D, TREE>(p, w, span, c0, c1, 32 * wave + __builtin_ctz(left));
}

template <int D, bool LARGE, bool TREE>
struct AttnShared {
    SmallShared<D, TREE> small;
};
template <int D, bool TREE>
struct AttnShared<D, true, TREE> {
    union {
        SmallShared<D, TREE> small;
        LargeShared<D> large;
    };
};

template <int D, bool LARGE, bool TREE>
__global__ __launch_bounds__(kBlock, 2) void paged_attention_kernel(PagedAttnParams p)
{
    __shared__ AttnShared<D, LARGE, TREE> S;
    Piece w;
    if (!plan_piece<TREE>(p, blockIdx.x, w)) return;
    // the join's directory: which rows have parts, and where
    if (w.split == 0 && !p.whole)
        for (int i = threadIdx.x; i < w.n; i += kBlock)
            p.desc[size_t(w.first + i) * p.b.kv_heads + w.head] =
                make_int2(2 * w.pieces + (w.small ? 1 : 0), w.part + i * p.b.groups);
    Span span = span_of(p, TREE ? w.base : w.pos, w.position(w.n - 1));
    // (the same in every lane: kept where the compiler knows it)
    span.sink = uniform(span.sink);
    span.first = uniform(span.first);
    int c0 = 0, c1 = uniform(span.count);
    if (w.pieces > 1) {                        // count / pieces chunks each, the first ones one more
        const int each = uniform(int(unsigned(c1) / unsigned(w.pieces))), more = c1 - each * w.pieces;
        c0 = each * w.split + min(w.split, more);
        c1 = c0 + each + (w.split < more ? 1 : 0);
    }
    if constexpr (TREE) {
        if (w.small && w.n * p.b.groups <= kSmallRows) small_tile<D, true, 1>(p, w, span, c0, c1, S.small);
        else if (w.small) small_tile<D, true, 2>(p, w, span, c0, c1, S.small);
        else if constexpr (LARGE) large_tile<D, true>(p, w, span, c0, c1, S.large);
    } else {
        if (w.small) small_tile<D, false, 1>(p, w, span, c0, c1, S.small);
        else if constexpr (LARGE) large_tile<D, false>(p, w, span, c0, c1, S.large);
    }
}

// The join's threads are sets of groups * D / 4, one thread for four values of
// the output; what 256 leaves over is no whole set.  Set 0 stores.
__host__ __device__ constexpr int join_set(int thread, int quads) { return thread / quads; }
__host__ __device__ constexpr int join_quad(int thread, int quads) { return thread % quads; }
__host__ __device__ constexpr bool join_stores(int thread, int quads) { return join_set(thread, quads) == 0; }

// Whether every four values have one thread that stores them, for each head size and group.
constexpr bool join_has_one_writer()
{
    for (int D = 16; D <= 128; D *= 2)
        for (int groups = 1; groups <= 8; ++groups) {
            int writers[kJoinThreads] = {};
            const int quads = groups * D / 4;
            for (int t = 0; t < kJoinThreads; ++t)
                if (join_stores(t, quads)) ++writers[join_quad(t, quads)];
            for (int q = 0; q < quads; ++q)
                if (writers[q] != 1) return false;
        }
    return true;
}
static_assert(join_has_one_writer());

// Join the parts of one token's heads of one kv head: thread (set of parts,
// four values), the parts' loads four at a time ahead of their use.  Bound by
// latency where the parts are few (32 chats: 4.9 us) and by the L2 and HBM
// where they are many (501 tokens of 32 heads in 4 parts, 34 MB: 12 us).
// Blocks of 512 threads take 5 us longer for the latter.
template <int D, bool TREE>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(PagedAttnParams p)
{
    __shared__ float4v so[kJoinThreads];
    __shared__ float sl[kJoinThreads], sm[kJoinThreads];
    const int cut = *p.cut;                               // (waited for beside the first row's loads)
    const int quads = p.b.groups * D / 4;                 // at most 256
    const int sets = kJoinThreads / quads;
    const int set = join_set(threadIdx.x, quads), quad = join_quad(threadIdx.x, quads);
    const int r = quad / (D / 4), at = quad % (D / 4);
    const unsigned all = unsigned(p.b.tokens) * unsigned(p.b.kv_heads);
    for (unsigned i = blockIdx.x; i < all; i += gridDim.x) {
        const int t = int(i / unsigned(p.b.kv_heads)), h = int(i - unsigned(t) * unsigned(p.b.kv_heads));
        const int2 d = p.desc[i];                         // (of any contents where the row is nobody's)
        int first = 0, count = 0;
        const int b = paged_sequence(p.b, t, &first, &count);
        if (cut == 0) return;
        if (b < 0) continue;
        const int pieces = d.x >> 1, stride = (d.x & 1) ? kStreamRows<TREE> : kTileRows;
        if (pieces < 2 || d.y < 0 || int64_t(d.y) + int64_t(pieces - 1) * stride + p.b.groups > p.part_rows) continue;
        float m = -__builtin_inff(), l = 0.0f;
        float4v o = {0.0f, 0.0f, 0.0f, 0.0f};
        float lost = 0.0f;                                // NaN where a part saw only scores of -inf
        auto add = [&](float pm, float pl, const float4v& po) {
            if (pm == -__builtin_inff()) {
                lost += pl;
                return;
            }
            const float top = fmaxf(m, pm);
            const float a = exp2_fast(m - top), b = exp2_fast(pm - top);
            l = l * a + pl * b;
            o = o * a + po * b;
            m = top;
        };
        if (set < sets) {
            for (int i0 = set; i0 < pieces; i0 += 4 * sets) {
                float2 ml[4];
                float4v x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int j = i0 + k * sets;
                    const size_t row = size_t(d.y) + size_t(j < pieces ? j : i0) * stride + r;
                    ml[k] = p.part_ml[row];
                    x[k] = reinterpret_cast<const float4v*>(p.part_o + row * D)[at];
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i0 + k * sets < pieces) add(ml[k].x, ml[k].y, x[k]);
            }
        }
        if (sets > 1) {
            __syncthreads();                              // (the last row's readers)
            sm[threadIdx.x] = m;
            sl[threadIdx.x] = m == -__builtin_inff() ? lost : l;
            so[threadIdx.x] = o;
            __syncthreads();
        }
        // (of one set and threads left over too: groups of 5 to 7 heads of 128)
        if (!join_stores(threadIdx.x, quads)) continue;
        if (sets > 1) {
            for (int k = 1; k < sets; ++k) add(sm[k * quads + quad], sl[k * quads + quad], so[k * quads + quad]);
        }
        const float f = 1.0f / l;
        float4v y = {o[0] * f, o[1] * f, o[2] * f, o[3] * f};
        if (m == -__builtin_inff()) y = float4v{lost, lost, lost, lost};   // nothing seen: 0; only scores of -inf: NaN
        const size_t row = size_t(t) * p.b.heads + h * p.b.groups + r;
        reinterpret_cast<float4v*>(p.out + row * D)[at] = y;
    }
}

// The join of a tree's batch of many rows (a token's heads of one kv head), whose
// parts are few: quads of a multiple of 64 threads, so that a wave has one row,
// as many rows a block as fit, and no exchange between threads (6 heads of 128
// are 192 threads: one row, and a wave left over).  382 tokens of 32 heads in 2
// parts: 6.4 us, 9.1 by paged_join_kernel; 96 in 16 parts 10.3 and 9.1: where
// rows are few, their parts are many.  Where both are (46 chats of 300 positions
// in one part, one of 40960 in 46, trees of 16 nodes) the call takes 83 us, 79 by
// paged_join_kernel.
constexpr int kJoinRows = 2048;

template <int D>
__global__ __launch_bounds__(kJoinThreads) void tree_join_kernel(PagedAttnParams p)
{
    const int cut = *p.cut;
    const int quads = p.b.groups * D / 4;                 // 64, 128, 192 or 256
    const int slots = kJoinThreads / quads;
    const int slot = uniform(threadIdx.x / unsigned(quads)), quad = threadIdx.x - slot * quads;
    if (slot >= slots) return;                            // (left over: the row after is another block's)
    const int r = quad / (D / 4), at = quad % (D / 4);
    const unsigned all = unsigned(p.b.tokens) * unsigned(p.b.kv_heads);
    for (unsigned i = blockIdx.x * slots + slot; i < all; i += gridDim.x * slots) {
        const int t = int(i / unsigned(p.b.kv_heads)), h = int(i - unsigned(t) * unsigned(p.b.kv_heads));
        const int2 d = p.desc[i];                         // (of any contents where the row is nobody's)
        int first = 0, count = 0;
        const int b = paged_sequence(p.b, t, &first, &count);
        if (cut == 0) return;
        if (b < 0) continue;
        const int pieces = d.x >> 1, stride = (d.x & 1) ? kStreamRows<true> : kTileRows;
        if (pieces < 2 || d.y < 0 || int64_t(d.y) + int64_t(pieces - 1) * stride + p.b.groups > p.part_rows) continue;
        float m = -__builtin_inff(), l = 0.0f, lost = 0.0f;
        float4v o = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int AHEAD = 4;
        for (int i0 = 0; i0 < pieces; i0 += AHEAD) {
            float2 ml[AHEAD];
            float4v x[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                if (i0 + k >= pieces) break;
                const size_t row = size_t(d.y) + size_t(i0 + k) * stride + r;
                ml[k] = p.part_ml[row];
                x[k] = reinterpret_cast<const float4v*>(p.part_o + row * D)[at];
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                if (i0 + k >= pieces) break;
                if (ml[k].x == -__builtin_inff()) {
                    lost += ml[k].y;
                    continue;
                }
                const float top = fmaxf(m, ml[k].x);
                const float a = exp2_fast(m - top), b = exp2_fast(ml[k].x - top);
                l = l * a + ml[k].y * b;
                o = o * a + x[k] * b;
                m = top;
            }
        }
        const float f = 1.0f / l;
        float4v y = {o[0] * f, o[1] * f, o[2] * f, o[3] * f};
        if (m == -__builtin_inff()) y = float4v{lost, lost, lost, lost};   // nothing seen: 0; only scores of -inf: NaN
        const size_t row = size_t(t) * p.b.heads + h * p.b.groups + r;
        reinterpret_cast<float4v*>(p.out + row * D)[at] = y;
    }
}

// -------------------------------------------------------------------- host
struct AttnLayout {
    size_t first, item, desc, ml, o, total;
    int part_rows;
};

// Rows of partial results: pieces are of T >= work / kTarget chunks, and a
// sequence of S > 1 pieces a tile has at least 1.5 T chunks a tile, so S <=
// chunks / T + 1/2 < 2 chunks / T, and over all of them fewer than 2 kTarget.
template <bool TREE>
AttnLayout attn_layout(int tokens, int kv_heads, int head_dim, bool large)
{
    AttnLayout L;
    auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
    L.part_rows = 2 * kTarget * (large ? kTileRows : kStreamRows<TREE>);
    L.first = 256;                             // (the plan's, of sequences with rows)
    L.item = L.first + up((size_t(tokens) + 1) * sizeof(int32_t));
    L.desc = L.item + up(size_t(tokens) * sizeof(int4));
    L.ml = L.desc + up(size_t(tokens) * kv_heads * sizeof(int2));
    L.o = L.ml + up(size_t(L.part_rows) * sizeof(float2));
    L.total = L.o + up(size_t(L.part_rows) * head_dim * sizeof(float));
    return L;
}

// Whether a batch may hold a tile of more rows than stream to registers.
template <bool TREE>
bool attn_large(int tokens, int groups, bool single)
{
    return !single && int64_t(tokens) * groups > kStreamRows<TREE>;
}

template <int D, bool TREE>
void launch_attention(const PagedAttnParams& p, bool large, int64_t blocks, hipStream_t s)
{
    if (p.planned) hipLaunchKernelGGL(paged_plan_kernel<TREE>, dim3(1), dim3(kPlanThreads), 0, s, p);
    if (large) hipLaunchKernelGGL((paged_attention_kernel<D, true, TREE>), dim3(unsigned(blocks)), dim3(kBlock), 0, s, p);
    else hipLaunchKernelGGL((paged_attention_kernel<D, false, TREE>), dim3(unsigned(blocks)), dim3(kBlock), 0, s, p);
    if (p.whole) return;
    const int64_t rows = int64_t(p.b.tokens) * p.b.kv_heads;
    if constexpr (TREE) {
        const int quads = p.b.groups * D / 4;
        if (quads % kWave == 0 && rows >= kJoinRows) {
            const int64_t blocks = (rows * quads + kJoinThreads - 1) / kJoinThreads;
            hipLaunchKernelGGL(tree_join_kernel<D>, dim3(unsigned(std::min<int64_t>(kJoinBlocks, blocks))),
                               dim3(kJoinThreads), 0, s, p);
            return;
        }
    }
    hipLaunchKernelGGL((paged_join_kernel<D, TREE>), dim3(unsigned(std::min<int64_t>(kJoinBlocks, rows))),
                       dim3(kJoinThreads), 0, s, p);
}

// The launches of a checked call (its batch is p.b already).
template <bool TREE>
int run_attention(PagedAttnParams& p, const hq_pages* cache, const float* query, int window, int sinks, float* output,
                  void* workspace, hipStream_t s)
{
    const int32_t* starts = p.b.starts;
    const int tokens = p.b.tokens;
    p.query = query;
    p.out = output;
    p.window = window;
    p.sinks = sinks;
    p.tile_tokens = kTileRows / p.b.groups;
    p.by_group = 65536 / p.b.groups + 1;
    const bool large = attn_large<TREE>(tokens, p.b.groups, starts == nullptr);
    const AttnLayout L = attn_layout<TREE>(tokens, p.b.kv_heads, cache->head_dim, large);
    char* ws = static_cast<char*>(workspace);
    p.part_rows = L.part_rows;
    p.cut = reinterpret_cast<int32_t*>(ws);
    p.plan_count = p.cut + 1;
    p.plan_first = reinterpret_cast<int32_t*>(ws + L.first);
    p.plan_item = reinterpret_cast<int4*>(ws + L.item);
    p.desc = reinterpret_cast<int2*>(ws + L.desc);
    p.part_ml = reinterpret_cast<float2*>(ws + L.ml);
    p.part_o = reinterpret_cast<float*>(ws + L.o);
    // chunks / T + 1 pieces a tile and kv head at most, so `target` and one of each in all; nor more than the
    // table's width allows.  A block without a piece ends at once.
    const int64_t narrow = int64_t(tokens) / std::max(1, kSmallRows / p.b.groups) + std::min(tokens, p.b.sequences);
    p.narrow = TREE && narrow * p.b.kv_heads <= kTarget / 2;
    const int64_t tiles = p.narrow ? narrow
                          : large  ? int64_t(tokens) / p.tile_tokens + (tokens < p.b.sequences ? tokens : p.b.sequences)
                                   : std::min(tokens, p.b.sequences);
    const int64_t widest = (int64_t(cache->max_pages) * cache->page_size + kChunkKeys - 1) / kChunkKeys;
    p.whole = widest <= kWholeChunks;
    const int64_t blocks = p.whole ? tiles * p.b.kv_heads
                                   : std::min(kTarget + tiles * p.b.kv_heads,
                                              tiles * p.b.kv_heads * ((widest + kSmallMin - 1) / kSmallMin));
    p.planned = cache->sequences >= kPlanSequences && !(p.whole && !starts);
    if (blocks > kMaxBlocks || int64_t(tokens) * p.b.kv_heads > 0x7fffffff) return HQ_ERR_ARG;
    switch (cache->head_dim) {
    case 16: launch_attention<16, TREE>(p, large, blocks, s); break;
    case 32: launch_attention<32, TREE>(p, large, blocks, s); break;
    case 64: launch_attention<64, TREE>(p, large, blocks, s); break;
    default: launch_attention<128, TREE>(p, large, blocks, s); break;
    }
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}

}  // namespace hq
