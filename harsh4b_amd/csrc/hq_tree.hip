// hq_tree.hip - drafted trees over the paged cache on gfx950: their plan
// (hq_tree_plan) and the path that the model's choices follow
// (hq_pages_accept).  No reference counterpart.
#include <algorithm>

#include "hq_device.h"
#include "hq_internal.h"
#include "hq_paged.h"

namespace hq {

constexpr int kTreeLanes = kTreeNodes / kWave;   // nodes a lane holds: lane, lane + 64, ..
constexpr int kTreeWaves = kBlock / kWave;

// A sequence's rows; false: its starts are no range of the batch's rows.
__device__ __forceinline__ bool tree_rows(const int32_t* starts, int b, int tokens, int* first, int* count)
{
    const int a = starts[b], z = starts[b + 1];
    const bool bad = a < 0 || a > z || z > tokens;
    *first = bad ? 0 : a;
    *count = bad ? 0 : z - a;
    return !bad;
}

// -------------------------------------------------------------------- plan
// A wave a sequence: its parents in LDS, and each lane walks up from its node.
__global__ __launch_bounds__(kBlock) void tree_plan_kernel(hq_tree t, int sequences, int32_t* status)
{
    __shared__ int parent_of[kTreeWaves][kTreeNodes];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int b = blockIdx.x * kTreeWaves + wave;
    if (b >= sequences) return;
    int first, n;
    if (!tree_rows(t.starts, b, t.tokens, &first, &n)) {
        if (lane == 0) atomicOr(status, HQ_PAGES_BAD);
        return;
    }
    bool bad = n > kTreeNodes;
    for (int i = lane; i < n && i < kTreeNodes; i += kWave) {
        const int p = t.parents[first + i];
        bad |= p < -1 || p >= i;
        parent_of[wave][i] = p;
    }
    bad = __any(bad);
    if (bad && lane == 0) atomicOr(status, HQ_PAGES_BAD);
    for (int i = lane; i < n; i += kWave) {
        uint32_t words[kTreeWords] = {};
        int depth = -1;
        if (!bad) {
            // (a parent stands before its node: the walk ends)
            for (int at = i; at >= 0; at = parent_of[wave][at]) {
                ++depth;
#pragma unroll
                for (int w = 0; w < kTreeWords; ++w) words[w] |= at >> 5 == w ? 1u << (at & 31) : 0u;
            }
        }
        t.depths[first + i] = depth;
        uint4* to = reinterpret_cast<uint4*>(t.ancestors + size_t(first + i) * kTreeWords);
        to[0] = make_uint4(words[0], words[1], words[2], words[3]);
        to[1] = make_uint4(words[4], words[5], words[6], words[7]);
    }
}

// ------------------------------------------------------------------ accept
struct Best {
    float v;
    int i;
};

struct AcceptParams {
    hq_pages c;
    hq_tree t;
    const int32_t* drafted;
    const int32_t* choices;      // or
    const float* logits;         // [tokens, vocab]
    int vocab, levels, shift;
    int splits;                  // parts of a row of logits
    Best* best;                  // [tokens, splits], by levels [2, sequences, splits]
    int32_t* nodes;              // by levels: [levels, sequences] the path's node, or -1
    int32_t* last;               // by levels: [sequences] the choice where the path ended
    int32_t* kept;
    int32_t* path;
    int32_t* next;
};

__device__ __forceinline__ Best better(Best a, Best b) { return argmax_better(b.v, b.i, a.v, a.i) ? b : a; }

__device__ __forceinline__ Best wave_best(Best x)
{
#pragma unroll
    for (int o = kWave / 2; o >= 1; o >>= 1)
        x = better(x, Best{__shfl_xor(x.v, o, kWave), __shfl_xor(x.i, o, kWave)});
    return x;
}

// The best of part `part` of a row of logits, by a block; valid in thread 0.
__device__ Best row_part_best(const float* row, int vocab, int part, int splits, Best* red)
{
    const int each = (vocab + splits - 1) / splits;
    const int from = min(part * each, vocab), to = min(from + each, vocab);
    Best x{-__builtin_inff(), 0x7fffffff};
    for (int i = from + int(threadIdx.x); i < to; i += kBlock) {
        const float v = row[i];
        if (argmax_better(v, i, x.v, x.i)) x = Best{v, i};
    }
    x = wave_best(x);
    const int wave = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) red[wave] = x;
    __syncthreads();
    for (int w = 0; w < kTreeWaves; ++w) x = better(x, red[w]);
    return x;
}

// The choice that a row's parts give (wave-uniform; every lane calls it).
__device__ __forceinline__ int choice_of(const Best* parts, int splits)
{
    const int lane = threadIdx.x & (kWave - 1);
    Best x{-__builtin_inff(), 0x7fffffff};
    if (lane < splits) x = parts[lane];
    return __builtin_amdgcn_readfirstlane(wave_best(x).i);
}

// Whether a sequence takes part (wave-uniform): its rows, and slot of the root.
__device__ __forceinline__ bool accept_rows(const AcceptParams& p, int b, int* first, int* n, int* base, bool* bad)
{
    *bad = !tree_rows(p.t.starts, b, p.t.tokens, first, n);
    *base = 0;
    if (*n == 0) return false;
    *base = p.c.lengths[b] - *n;
    *bad = p.t.depths[*first] < 0 || *n > kTreeNodes || *base < 0;
    return !*bad && (*p.c.status & (HQ_PAGES_FULL | HQ_PAGES_REFUSED)) == 0;
}

// A sequence's nodes in the lanes of a wave.
struct Nodes {
    int parent[kTreeLanes], token[kTreeLanes];
    __device__ __forceinline__ void load(const AcceptParams& p, int first, int n)
    {
        const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
        for (int k = 0; k < kTreeLanes; ++k) {
            const int i = lane + k * kWave;
            parent[k] = i < n ? p.t.parents[first + i] : -2;
            token[k] = i < n ? p.drafted[first + i] : 0;
        }
    }
    // The first child of node u that holds `choice`, or -1.
    __device__ __forceinline__ int child(int u, int choice) const
    {
        const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
        for (int k = 0; k < kTreeLanes; ++k) {
            const uint64_t m = __ballot(parent[k] == u && token[k] == choice && lane + k * kWave > u);
            if (m) return k * kWave + __builtin_ctzll(m);
        }
        return -1;
    }
};

// Every row's choice, a block a part.
__global__ __launch_bounds__(kBlock) void accept_rows_kernel(AcceptParams p)
{
    __shared__ Best red[kTreeWaves];
    const int row = blockIdx.x;
    const Best x = row_part_best(p.logits + size_t(row) * p.vocab, p.vocab, blockIdx.y, p.splits, red);
    if (threadIdx.x == 0) p.best[size_t(row) * p.splits + blockIdx.y] = x;
}

// The path's node of level `level` (from the choice at the one above), or -1: for every block of a sequence.
__device__ __forceinline__ int step_down(const AcceptParams& p, int b, int level, bool writes)
{
    const int lane = threadIdx.x & (kWave - 1);
    int first, n, base, v = -1;
    bool bad;
    if (level == 0) {
        if (accept_rows(p, b, &first, &n, &base, &bad)) v = 0;
    } else {
        const int u = p.nodes[size_t(level - 1) * p.c.sequences + b];
        if (u >= 0) {
            const Best* parts = p.best + (size_t((level - 1) & 1) * p.c.sequences + b) * p.splits;
            const int choice = choice_of(parts, p.splits);
            if (level < p.levels) {
                accept_rows(p, b, &first, &n, &base, &bad);
                Nodes nodes;
                nodes.load(p, first, n);
                v = nodes.child(u, choice);
            }
            if (v < 0 && writes && lane == 0) p.last[b] = choice;
        }
    }
    if (writes && lane == 0 && level < p.levels) p.nodes[size_t(level) * p.c.sequences + b] = v;
    return v;
}

// One level of the paths: the node, and the parts of its row of logits.
__global__ __launch_bounds__(kBlock) void accept_level_kernel(AcceptParams p, int level)
{
    __shared__ Best red[kTreeWaves];
    const int b = blockIdx.x;
    const int v = step_down(p, b, level, blockIdx.y == 0 && threadIdx.x < kWave);
    if (v < 0) return;
    const size_t row = size_t(p.t.starts[b]) + v;
    const Best x = row_part_best(p.logits + row * p.vocab, p.vocab, blockIdx.y, p.splits, red);
    if (threadIdx.x == 0) p.best[(size_t(level & 1) * p.c.sequences + b) * p.splits + blockIdx.y] = x;
}

// The end of a path walked by levels.
__global__ __launch_bounds__(kBlock) void accept_last_kernel(AcceptParams p)
{
    const int b = blockIdx.x * kTreeWaves + threadIdx.x / kWave;
    if (b < p.c.sequences) step_down(p, b, p.levels, true);
}

// The path, and its K and V to their slots: blocks (sequence, slice of the
// layers' heads); each wave walks the path by itself.
constexpr int kMoveItems = 4;          // a wave's rows of (layer, K or V, kv head)

template <int D, bool LEVELS>
__global__ __launch_bounds__(kBlock) void accept_move_kernel(AcceptParams p)
{
    constexpr int PIECES = D / 8, ROWS = kWave / PIECES;   // 16-byte pieces of a K row, rows a wave moves at a time
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int b = blockIdx.x;
    int first, n, base;
    bool bad;
    const bool takes_part = accept_rows(p, b, &first, &n, &base, &bad);
    const bool writes = blockIdx.y == 0 && wave == 0;
    int path[kTreeLanes];
#pragma unroll
    for (int k = 0; k < kTreeLanes; ++k) path[k] = -1;
    int count = 0, choice = -1;
    if (takes_part) {
        if constexpr (LEVELS) {
#pragma unroll
            for (int k = 0; k < kTreeLanes; ++k) {
                const int level = lane + k * kWave;
                if (level < p.levels) path[k] = p.nodes[size_t(level) * p.c.sequences + b];
                count += __popcll(__ballot(path[k] >= 0));
            }
            choice = p.last[b];
        } else {
            Nodes nodes;
            nodes.load(p, first, n);
            int mine[kTreeLanes];
            if (!p.logits) {
#pragma unroll
                for (int k = 0; k < kTreeLanes; ++k) mine[k] = lane + k * kWave < n ? p.choices[first + lane + k * kWave] : 0;
            }
            for (int u = 0; u >= 0; u = count < p.levels ? nodes.child(u, choice) : -1) {
#pragma unroll
                for (int k = 0; k < kTreeLanes; ++k)
                    if (lane + k * kWave == count) path[k] = u;
                ++count;
                if (p.logits) {
                    choice = choice_of(p.best + size_t(first + u) * p.splits, p.splits);
                } else {
#pragma unroll
                    for (int k = 0; k < kTreeLanes; ++k)
                        if (u >> 6 == k) choice = __builtin_amdgcn_readlane(mine[k], u & (kWave - 1));
                }
            }
        }
    }
    if (writes) {
        if (lane == 0) {
            p.kept[b] = takes_part ? base + count : -1;
            p.next[b] = choice;
            if (bad) atomicOr(p.c.status, HQ_PAGES_BAD);
        }
        for (int i = lane; i < n; i += kWave) {
            int v = -1;
#pragma unroll
            for (int k = 0; k < kTreeLanes; ++k)
                if (i >> 6 == k) v = path[k];
            p.path[first + i] = v;
        }
    }
    // Rows in the path's order, ROWS at a time, all read before the first is
    // written: node i of the path stands at or behind place i, so what is
    // written is no later one's source.
    const int heads = p.c.kv_heads, items = 2 * p.c.layers * heads;
    const size_t head = size_t(p.c.page_size) * D;
    for (int from = 0; from < count; from += ROWS) {
        const int i = from + lane / PIECES;
        int v = -1;
#pragma unroll
        for (int k = 0; k < kTreeLanes; ++k)
            if (from >> 6 == k) v = __shfl(path[k], i & (kWave - 1), kWave);
        bool moves = i < count && v != i;
        if (!__any(moves)) continue;
        auto page_of = [&](int slot) {
            const int e = slot >> p.shift;
            const int page = e < p.c.max_pages ? p.c.table[size_t(b) * p.c.max_pages + e] : -1;
            return page < p.c.pages ? page : -1;
        };
        const int to = moves ? page_of(base + i) : 0, of = moves ? page_of(base + v) : 0;
        if (to < 0 || of < 0) {
            moves = false;
            if (writes) atomicOr(p.c.status, HQ_PAGES_BAD);
        }
        const size_t place = (lane % PIECES) * 8;
        const size_t dst = size_t(max(to, 0)) * heads * head + size_t((base + i) & (p.c.page_size - 1)) * D + place;
        const size_t src = size_t(max(of, 0)) * heads * head + size_t((base + max(v, 0)) & (p.c.page_size - 1)) * D + place;
        for (int item = (blockIdx.y * kTreeWaves + wave) * kMoveItems; item < items;
             item += gridDim.y * kTreeWaves * kMoveItems) {
            uint4 x[kMoveItems];
            uint16_t* at[kMoveItems];
#pragma unroll
            for (int k = 0; k < kMoveItems; ++k) {
                const int it = min(item + k, items - 1);
                const int h = it % heads, rest = it / heads;
                at[k] = ((rest & 1) ? p.c.values : p.c.keys) + (size_t(rest >> 1) * p.c.pages * heads + h) * head;
                if (moves) x[k] = *reinterpret_cast<const uint4*>(at[k] + src);
            }
#pragma unroll
            for (int k = 0; k < kMoveItems; ++k)
                if (moves && item + k < items) *reinterpret_cast<uint4*>(at[k] + dst) = x[k];
        }
    }
}

// -------------------------------------------------------------------- host
// How the choices are found: each row's of the batch in one launch, or a launch
// for each level of the paths that reads its nodes' rows alone.
struct AcceptPlan {
    bool by_levels;
    int splits;
    size_t nodes, last, total;   // (best is at 0)
};

static AcceptPlan accept_plan(int tokens, int sequences, int vocab, int levels)
{
    AcceptPlan a{};
    auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
    const double row_us = vocab * 4.0 / 5e6;
    a.by_levels = vocab > 0 && tokens * row_us > levels * (3.0 + sequences * row_us);
    const int64_t rows = std::max(1, a.by_levels ? sequences : tokens);
    a.splits = vocab ? int(std::max<int64_t>(1, std::min<int64_t>({64, (1024 + rows - 1) / rows, (vocab + 2047) / 2048}))) : 0;
    a.nodes = up((a.by_levels ? 2 * rows : rows) * a.splits * sizeof(Best));
    a.last = a.nodes + (a.by_levels ? up(size_t(levels) * sequences * 4) : 0);
    a.total = a.last + (a.by_levels ? up(size_t(sequences) * 4) : 0);
    return a;
}

template <bool LEVELS>
static void launch_move(const AcceptParams& p, dim3 grid, hipStream_t s)
{
    switch (p.c.head_dim) {
    case 16: hipLaunchKernelGGL((accept_move_kernel<16, LEVELS>), grid, dim3(kBlock), 0, s, p); break;
    case 32: hipLaunchKernelGGL((accept_move_kernel<32, LEVELS>), grid, dim3(kBlock), 0, s, p); break;
    case 64: hipLaunchKernelGGL((accept_move_kernel<64, LEVELS>), grid, dim3(kBlock), 0, s, p); break;
    default: hipLaunchKernelGGL((accept_move_kernel<128, LEVELS>), grid, dim3(kBlock), 0, s, p); break;
    }
}

}  // namespace hq

using namespace hq;

extern "C" int hq_tree_plan(const hq_tree* tree, int sequences, int32_t* status, void* stream)
{
    const int bad = tree_check(tree);
    if (bad) return bad;
    if (sequences < 1 || sequences > kMaxBlocks || tree->tokens > kMaxBlocks || !status) return HQ_ERR_ARG;
    hipLaunchKernelGGL(tree_plan_kernel, dim3((sequences + kTreeWaves - 1) / kTreeWaves), dim3(kBlock), 0,
                       static_cast<hipStream_t>(stream), *tree, sequences, status);
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}

extern "C" size_t hq_pages_accept_workspace_bytes(int tokens, int sequences, int vocab, int levels)
{
    if (tokens < 0 || sequences < 1 || vocab < 0 || levels < 1 || levels > kTreeNodes) return 0;
    return std::max<size_t>(256, accept_plan(tokens, sequences, vocab, levels).total);
}

extern "C" int hq_pages_accept(const hq_pages* cache, const hq_tree* tree, const int32_t* drafted, const int32_t* choices,
                               const float* logits, int vocab, int levels, int32_t* kept, int32_t* path, int32_t* next,
                               void* workspace, void* stream)
{
    const int bad = tree_check(tree);
    if (bad) return bad;
    PagedBatch batch;
    const int err = paged_check(cache, cache ? cache->keys : nullptr, tree->starts, tree->tokens, cache ? cache->kv_heads : 0,
                                cache ? cache->values : nullptr, &batch);
    if (err) return err;
    if (cache->layers < 1 || !cache->status || !kept || !next || !workspace || levels < 1 || levels > kTreeNodes)
        return HQ_ERR_ARG;
    if (tree->tokens && (!drafted || !path || !choices == !logits)) return HQ_ERR_ARG;
    if (logits ? vocab < 1 : vocab != 0) return HQ_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return HQ_ERR_ALIGN;
    for (const void* q : {static_cast<const void*>(drafted), static_cast<const void*>(choices),
                          static_cast<const void*>(logits), static_cast<const void*>(kept),
                          static_cast<const void*>(path), static_cast<const void*>(next)})
        if (reinterpret_cast<uintptr_t>(q) & 3u) return HQ_ERR_ALIGN;
    const AcceptPlan a = accept_plan(tree->tokens, cache->sequences, vocab, levels);
    char* ws = static_cast<char*>(workspace);
    AcceptParams p{*cache, *tree, drafted, choices, logits, vocab, levels, batch.shift, a.splits,
                   reinterpret_cast<Best*>(ws), reinterpret_cast<int32_t*>(ws + a.nodes),
                   reinterpret_cast<int32_t*>(ws + a.last), kept, path, next};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t items = int64_t(2) * cache->layers * cache->kv_heads;
    if (items > 0x7fffffff) return HQ_ERR_ARG;
    const int per_block = kTreeWaves * kMoveItems;
    const int slices = int(std::min({(items + per_block - 1) / per_block, kMaxBlocks / cache->sequences, int64_t(4096)}));
    if (a.by_levels) {
        for (int level = 0; level < levels; ++level)
            hipLaunchKernelGGL(accept_level_kernel, dim3(cache->sequences, a.splits), dim3(kBlock), 0, s, p, level);
        hipLaunchKernelGGL(accept_last_kernel, dim3((cache->sequences + kTreeWaves - 1) / kTreeWaves), dim3(kBlock), 0, s, p);
        launch_move<true>(p, dim3(cache->sequences, slices), s);
    } else {
        if (logits && tree->tokens)
            hipLaunchKernelGGL(accept_rows_kernel, dim3(tree->tokens, a.splits), dim3(kBlock), 0, s, p);
        launch_move<false>(p, dim3(cache->sequences, slices), s);
    }
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}
