// hq_tree.hip - drafted trees over the paged cache on gfx950: their plan
// (hq_tree_plan) and the path that the model's choices follow
// (hq_pages_accept).  No reference counterpart.
#include <algorithm>

#include "hq_device.h"
#include "hq_internal.h"
#include "hq_paged.h"

namespace hq {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr int kTreeLanes = kTreeNodes / kWave;   // nodes a lane holds: lane, lane + 64, ..
constexpr int kTreeWaves = kBlock / kWave;
constexpr int kTreePages = kTreeNodes / 16 + 1;  // a tree may lie in

// A sequence's rows; false: its starts are no range of the batch's rows.
__device__ __forceinline__ bool tree_rows(const int32_t* starts, int b, int tokens, int* first, int* count)
{
    const int a = starts[b], z = starts[b + 1];
    const bool bad = a < 0 || a > z || z > tokens;
    *first = bad ? 0 : a;
    *count = bad ? 0 : z - a;
    return !bad;
}

// What the lanes of a wave wrote to LDS before is what they read after: a wave's
// LDS accesses take effect in their order, and the fences keep the compiler from
// another one (no instruction; to it the lanes' addresses may well be apart).
__device__ __forceinline__ void wave_lds_order()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// -------------------------------------------------------------------- plan
// A wave a sequence.  Each node holds the bits of the nodes up to some above it
// and which one comes next; a round takes over that one's, so that after k
// rounds 2^k nodes are covered: a chain of 256 has 8 rounds (6.0 us; walking up
// node by node, 255 steps, 65).  A node's depth is the number of its bits, less its
// own.  Bound by latency, a launch and three dependent reads (one tree of 8
// nodes 2.5 us, 64 of 60 4.0).
__global__ __launch_bounds__(kBlock) void tree_plan_kernel(hq_tree t, int sequences, int32_t* status)
{
    __shared__ uint4v seen_of[kTreeWaves][kTreeNodes][2];
    __shared__ int next_of[kTreeWaves][kTreeNodes];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int b = blockIdx.x * kTreeWaves + wave;
    if (b >= sequences) return;
    int first, n;
    if (!tree_rows(t.starts, b, t.tokens, &first, &n)) {
        if (lane == 0) atomicOr(status, HQ_PAGES_BAD);
        return;
    }
    first = __builtin_amdgcn_readfirstlane(first);
    n = __builtin_amdgcn_readfirstlane(n);
    uint4v seen[kTreeLanes][2];
    int next[kTreeLanes];
    bool bad = n > kTreeNodes;
#pragma unroll
    for (int k = 0; k < kTreeLanes; ++k) {
        const int i = lane + k * kWave;
        next[k] = i < n ? t.parents[first + i] : -1;
        bad |= next[k] < -1 || next[k] >= i;
        seen[k][0] = seen[k][1] = uint4v{0, 0, 0, 0};
        const uint32_t bit = 1u << (lane & 31);
        seen[k][k / 2][2 * (k % 2)] = lane < 32 ? bit : 0u;
        seen[k][k / 2][2 * (k % 2) + 1] = lane < 32 ? 0u : bit;
    }
    bad = __any(bad);
    if (bad) {
        if (lane == 0) atomicOr(status, HQ_PAGES_BAD);
        for (int i = lane; i < n; i += kWave) {
            t.depths[first + i] = -1;
            uint4v* const to = reinterpret_cast<uint4v*>(t.ancestors + size_t(first + i) * kTreeWords);
            to[0] = to[1] = uint4v{0, 0, 0, 0};
        }
        return;
    }
    while (true) {
        bool more = false;
        unrolled<kTreeLanes>([&](auto lanes) {
            constexpr int k = decltype(lanes)::value;
            if (k * kWave >= n) return;
            seen_of[wave][lane + k * kWave][0] = seen[k][0];
            seen_of[wave][lane + k * kWave][1] = seen[k][1];
            next_of[wave][lane + k * kWave] = next[k];
            more |= next[k] >= 0;
        });
        if (!__any(more)) break;
        wave_lds_order();
        unrolled<kTreeLanes>([&](auto lanes) {
            constexpr int k = decltype(lanes)::value;
            if (k * kWave >= n || next[k] < 0) return;
            seen[k][0] |= seen_of[wave][next[k]][0];
            seen[k][1] |= seen_of[wave][next[k]][1];
            next[k] = next_of[wave][next[k]];
        });
        wave_lds_order();                      // (all of a round's reads come before the next one's writes)
    }
#pragma unroll
    for (int k = 0; k < kTreeLanes; ++k) {
        const int i = lane + k * kWave;
        if (i >= n) continue;
        int depth = -1;
#pragma unroll
        for (int w = 0; w < 4; ++w) depth += __popc(seen[k][0][w]) + __popc(seen[k][1][w]);
        t.depths[first + i] = depth;
        uint4v* const to = reinterpret_cast<uint4v*>(t.ancestors + size_t(first + i) * kTreeWords);
        to[0] = seen[k][0];
        to[1] = seen[k][1];
    }
}

// ------------------------------------------------------------------ accept
// Greedy choices: a node's choice can be the token of one of its children
// alone, of the one with the largest logit there (in argmax's order).  So the
// path is the beginning of a chain that a look at the children's logits gives,
// from the root to a leaf: one launch finds the argmax of the chain's rows, and
// no others are read.  The next walks the path and moves K and V.
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
    int slots;                   // levels of a chain looked at side by side
    int splits;                  // parts of a row of logits
    Best* best;                  // [tokens, splits] of the chain's node at level l in a sequence's row l
    int32_t* kept;
    int32_t* path;
    int32_t* next;
};

__device__ __forceinline__ Best better(Best a, Best b) { return argmax_better(b.v, b.i, a.v, a.i) ? b : a; }

// The least of the wave's values, in every lane (levels as in wave_max64_all).
__device__ __forceinline__ int wave_imin64_all(int v)
{
    unsigned x = unsigned(v), y = x;
    swap32(x, y);
    v = min(int(x), int(y));
    x = y = unsigned(v);
    swap16(x, y);
    v = min(int(x), int(y));
    v = min(v, dpp_i<kRowShl8>(v));
    v = min(v, dpp_i<kRowShl4>(v));
    v = min(v, dpp_i<kRowShl2>(v));
    v = min(v, dpp_i<kRowShl1>(v));
    return __builtin_amdgcn_readfirstlane(v);
}

// The best of the wave's, in every lane (no shuffles through LDS: a chain's
// levels follow one another).
__device__ __forceinline__ Best wave_best(Best x)
{
    const uint64_t nans = __ballot(x.v != x.v);
    const float top = wave_max64_all(x.v);             // (of the numbers)
    const bool leads = nans ? x.v != x.v : x.v == top;
    const int i = wave_imin64_all(leads ? x.i : 0x7fffffff);
    return Best{nans ? __builtin_nanf("") : top, i};
}

// A sequence, its nodes in the lanes of a wave; n = 0: it takes no part
// (wave-uniform).
struct Sequence {
    int first, n, base;
    int rows;                    // its rows of the batch (whether it takes part or not)
    bool bad;
    int parent[kTreeLanes], token[kTreeLanes], choice[kTreeLanes], depth[kTreeLanes];
    int status;

    // Two round trips, the second under way when this returns: the sequence's
    // numbers, then its nodes' together.
    __device__ __forceinline__ void load(const AcceptParams& p, int b)
    {
        const int lane = threadIdx.x & (kWave - 1);
        const int length = p.c.lengths[b];
        status = *p.c.status;
        bad = !tree_rows(p.t.starts, b, p.t.tokens, &first, &rows);
        first = __builtin_amdgcn_readfirstlane(first);
        rows = __builtin_amdgcn_readfirstlane(rows);
        // (a length near -2^31: in 32 bits the difference would wrap round to a slot past any table)
        base = int(max(int64_t(__builtin_amdgcn_readfirstlane(length)) - rows, int64_t(-1)));
        n = 0;
        if (rows == 0) return;
#pragma unroll
        for (int k = 0; k < kTreeLanes; ++k) {
            const int i = lane + k * kWave;
            parent[k] = i < rows ? p.t.parents[first + i] : -2;
            token[k] = i < rows ? p.drafted[first + i] : 0;
            choice[k] = i < rows && p.choices ? p.choices[first + i] : 0;
            depth[k] = i < rows ? p.t.depths[first + i] : -1;
        }
    }
    // Whether it takes part.
    __device__ __forceinline__ bool settle()
    {
        if (rows == 0) return false;
        bad = __builtin_amdgcn_readfirstlane(depth[0]) < 0 || rows > kTreeNodes || base < 0;
        if (!bad && (__builtin_amdgcn_readfirstlane(status) & (HQ_PAGES_FULL | HQ_PAGES_REFUSED)) == 0) n = rows;
        return n != 0;
    }
    __device__ __forceinline__ bool below(int k, int u) const      // whether the lane's k-th node is a child of u
    {
        return parent[k] == u && int(threadIdx.x & (kWave - 1)) + k * kWave > u;
    }
    // The first child of node u that holds `choice`, or -1.
    __device__ __forceinline__ int child(int u, int choice) const
    {
#pragma unroll
        for (int k = 0; k < kTreeLanes; ++k) {
            if (k * kWave >= n) break;
            const uint64_t m = __ballot(below(k, u) && token[k] == choice);
            if (m) return k * kWave + __builtin_ctzll(m);
        }
        return -1;
    }
};

constexpr int kRowAhead = 8;           // fours of logits a thread has on their way

// The best of part `part` of a row of logits, by a block; valid in thread 0.
// The row in fours from its first 16-byte border on; what lies before it goes
// to part 0, the rest behind the fours to the last part.
__device__ Best row_part_best(const float* row, int vocab, int part, int splits, Best* red)
{
    const int t = threadIdx.x;
    const int head = min(int(-(reinterpret_cast<uintptr_t>(row) >> 2) & 3), vocab);
    const int quads = (vocab - head) / 4, each = (quads + splits - 1) / splits;
    const int from = min(part * each, quads), to = min(from + each, quads);
    const float4v* body = reinterpret_cast<const float4v*>(row + head);
    Best x{-__builtin_inff(), 0x7fffffff};
    // (a thread's indices rise: a later value has to be larger, or the first NaN)
    auto take = [&](float v, int i) {
        if (x.i == 0x7fffffff || (!(v <= x.v) && x.v == x.v)) x = Best{v, i};
    };
    if (part == 0 && t < head) take(row[t], t);
    // (the last ones' places taken again rather than one at a time: a round trip each)
    constexpr int AHEAD = kRowAhead;
    for (int q = from + t; q < to; q += AHEAD * kBlock) {
        float4v v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) v[k] = body[min(q + k * kBlock, to - 1)];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (q + k * kBlock >= to) continue;
            const int i = head + 4 * (q + k * kBlock);
#pragma unroll
            for (int e = 0; e < 4; ++e) take(v[k][e], i + e);
        }
    }
    const int tail = head + 4 * quads + t;
    if (part == splits - 1 && tail < vocab) take(row[tail], tail);
    x = wave_best(x);
    const int wave = t / kWave;
    __syncthreads();                   // (red's last readers)
    if ((t & (kWave - 1)) == 0) red[wave] = x;
    __syncthreads();
    for (int w = 0; w < kTreeWaves; ++w) x = better(x, red[w]);
    return x;
}

// The argmax of the chains' rows: blocks (sequence, part of its rows, first of
// the chain's levels that the block takes, every slots-th).  A block's first
// wave works the chain out, from three round trips: the sequence's numbers, its
// nodes', and the nodes' logits at their parents, which lie scattered over the
// rows; the root is known without, so its row is on its way meanwhile (24.7 us
// for the below, 26.6 if it waits too).  Then the rows are bound by HBM: 32
// chats' chains of 138 rows of 151936 (84 MB, 17.8 us at the rate of a copy);
// every row of the batch takes 124, and a launch for each level would be seven.
// A block that takes the levels one after another (no slots) 45: the longest
// chain sets the time.
__global__ __launch_bounds__(kBlock) void accept_chain_kernel(AcceptParams p)
{
    __shared__ Best red[kTreeWaves];
    __shared__ int node[kTreeNodes], nodes, first;
    if (blockIdx.z == 0) {
        int root, rows;
        tree_rows(p.t.starts, blockIdx.x, p.t.tokens, &root, &rows);
        if (rows == 0) return;
        const size_t at = __builtin_amdgcn_readfirstlane(root);
        const Best x = row_part_best(p.logits + at * p.vocab, p.vocab, blockIdx.y, p.splits, red);
        if (threadIdx.x == 0) p.best[at * p.splits + blockIdx.y] = x;
        if (p.levels <= p.slots) return;
    }
    if (threadIdx.x < kWave) {
        const int lane = threadIdx.x;
        int taken = 0;
        Sequence s;
        s.load(p, blockIdx.x);
        if (s.settle()) {
            Best own[kTreeLanes];              // a node's logit at its parent
#pragma unroll
            for (int k = 0; k < kTreeLanes; ++k) {
                const int u = s.parent[k], i = s.token[k];
                own[k] = Best{-__builtin_inff(), 0x7fffffff};
                if (u >= 0 && i >= 0 && i < p.vocab && s.below(k, u))
                    own[k] = Best{p.logits[size_t(s.first + u) * p.vocab + i], i};
            }
            if (lane == 0) first = s.first;
            int u = 0;
            for (int level = 0; u >= 0 && level < p.levels; ++level) {
                if (level && level % p.slots == int(blockIdx.z)) {
                    if (lane == 0) node[taken] = u;
                    ++taken;
                }
                Best x{-__builtin_inff(), 0x7fffffff};
#pragma unroll
                for (int k = 0; k < kTreeLanes; ++k)
                    if (s.below(k, u)) x = better(x, own[k]);
                const int choice = __builtin_amdgcn_readfirstlane(wave_best(x).i);
                u = choice == 0x7fffffff ? -1 : s.child(u, choice);
            }
        }
        if (lane == 0) nodes = taken;
    }
    lds_sync();
    const int taken = __builtin_amdgcn_readfirstlane(nodes);
    if (taken == 0) return;
    const size_t from = __builtin_amdgcn_readfirstlane(first);
    for (int k = 0; k < taken; ++k) {
        const float* row = p.logits + (from + __builtin_amdgcn_readfirstlane(node[k])) * p.vocab;
        const Best x = row_part_best(row, p.vocab, blockIdx.y, p.splits, red);
        const size_t level = blockIdx.z + size_t(k + (blockIdx.z == 0)) * p.slots;
        if (threadIdx.x == 0) p.best[(from + level) * p.splits + blockIdx.y] = x;
    }
}

// The choices at the levels of a sequence's chain, into LDS, by a wave: splits
// lanes (a power of two) a level, 64 / splits levels at a time.  Returns the
// levels that it has: those of the plan's depths, which the walk may not leave
// (a chain follows the parents, and goes on past them where the plan was made
// of others).  What lies past the chain's end is of any contents, and the walk,
// which ends there, does not come to it.
__device__ __forceinline__ int chain_choices(const AcceptParams& p, const Sequence& s, int* level_choice)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int part = lane & (p.splits - 1), each = kWave / p.splits;
    int deepest = 0;
#pragma unroll
    for (int k = 0; k < kTreeLanes; ++k) deepest = max(deepest, s.depth[k]);
    deepest = -wave_imin64_all(-deepest);
    const int levels = min(min(p.levels, s.n), min(deepest, kTreeNodes - 1) + 1);
    for (int from = 0; from < levels; from += each) {
        const int level = from + lane / p.splits;
        Best x = p.best[size_t(s.first + min(level, levels - 1)) * p.splits + part];
        for (int o = p.splits / 2; o >= 1; o >>= 1)
            x = better(x, Best{__shfl_xor(x.v, o, kWave), __shfl_xor(x.i, o, kWave)});
        if (level < levels && part == 0) level_choice[level] = x.i;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    return levels;
}

// The path, and its K and V to their slots: blocks (sequence, slice of the
// layers' heads).  A block's first wave walks the path; with all four walking
// for themselves the walks are most of the time.  Bound by latency, four or five
// dependent reads (one chat 4.2 us, of 36 layers and 8 kv heads), and where many
// move by rows of 256 bytes that lie apart (32 chats, 12 MB: 8.3 to 9.3 us).
// Of a wave's rows (layer, K or V, kv head) four: 8.6 us, 12.6 with two, 8.6
// with eight (one chat 5.1), 10.6 with sixteen.
constexpr int kMoveItems = 4;

template <int D>
__global__ __launch_bounds__(kBlock) void accept_move_kernel(AcceptParams p)
{
    constexpr int PIECES = D / 8, ROWS = kWave / PIECES;   // 16-byte pieces of a K row, rows a wave moves at a time
    __shared__ int level_choice[kTreeNodes], path[kTreeNodes], page_at[kTreePages];
    __shared__ int shared_count, shared_base;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int b = blockIdx.x;
    const bool writes = blockIdx.y == 0;
    if (wave == 0) {
        Sequence s;
        s.load(p, b);
        if (lane < kTreePages) {               // the pages of the tree's slots
            const int e = (s.base >> p.shift) + lane;
            const int page = s.rows && s.base >= 0 && e < p.c.max_pages ? p.c.table[size_t(b) * p.c.max_pages + e] : -1;
            page_at[lane] = page < p.c.pages ? page : -1;
        }
        int count = 0, choice = -1;
        if (s.settle()) {
            const int levels = p.logits ? chain_choices(p, s, level_choice) : p.levels;
            int u = 0;
            for (; u >= 0 && count < levels; u = count < p.levels ? s.child(u, choice) : -1) {
                if (lane == 0) path[count] = u;
                if (p.logits) {
                    choice = __builtin_amdgcn_readfirstlane(level_choice[count]);
                } else {
#pragma unroll
                    for (int k = 0; k < kTreeLanes; ++k)
                        if (u >> 6 == k) choice = __builtin_amdgcn_readlane(s.choice[k], u & (kWave - 1));
                }
                ++count;
            }
            s.bad = u >= 0;                    // (the path goes on where the plan has no level)
        }
        if (lane == 0) {
            shared_count = count;
            shared_base = s.base;
            if (writes) {
                p.kept[b] = s.n ? s.base + count : -1;
                p.next[b] = choice;
                if (s.bad) atomicOr(p.c.status, HQ_PAGES_BAD);
            }
        }
        if (writes) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            for (int i = lane; i < s.rows; i += kWave) p.path[s.first + i] = i < count ? path[i] : -1;
        }
    }
    lds_sync();
    const int count = __builtin_amdgcn_readfirstlane(shared_count), base = __builtin_amdgcn_readfirstlane(shared_base);
    // Rows in the path's order, ROWS at a time, all read before the first is
    // written: node i of the path stands at or behind place i, so what is
    // written is no later one's source.
    const int heads = p.c.kv_heads, items = 2 * p.c.layers * heads;
    const size_t head = size_t(p.c.page_size) * D;
    for (int from = 0; from < count; from += ROWS) {
        const int i = from + lane / PIECES;
        const int v = i < count ? path[i] : -1;
        bool moves = i < count && v != i;
        if (!__any(moves)) continue;
        auto page_of = [&](int slot) { return page_at[(slot >> p.shift) - (base >> p.shift)]; };
        const int to = moves ? page_of(base + i) : 0, of = moves ? page_of(base + v) : 0;
        if (to < 0 || of < 0) {
            moves = false;
            if (writes) atomicOr(p.c.status, HQ_PAGES_BAD);
        }
        const size_t place = (lane % PIECES) * 8;
        auto offset = [&](int page, int slot) {
            return size_t(max(page, 0)) * heads * head + size_t(slot & (p.c.page_size - 1)) * D + place;
        };
        const size_t dst = offset(to, base + i), src = offset(of, base + max(v, 0));
        for (int item = (blockIdx.y * kTreeWaves + wave) * kMoveItems; item < items;
             item += gridDim.y * kTreeWaves * kMoveItems) {
            uint4v x[kMoveItems];
            uint16_t* at[kMoveItems];
            int rest = item / heads, h = item - rest * heads;
#pragma unroll
            for (int k = 0; k < kMoveItems; ++k) {
                at[k] = ((rest & 1) ? p.c.values : p.c.keys) + (size_t(rest >> 1) * p.c.pages * heads + h) * head;
                x[k] = uint4v{0, 0, 0, 0};
                if (moves && item + k < items) x[k] = *reinterpret_cast<const uint4v*>(at[k] + src);
                if (++h == heads) {
                    h = 0;
                    ++rest;
                }
            }
#pragma unroll
            for (int k = 0; k < kMoveItems; ++k)
                if (moves && item + k < items) *reinterpret_cast<uint4v*>(at[k] + dst) = x[k];
        }
    }
}

// -------------------------------------------------------------------- host
struct AcceptPlan {
    int slots, splits;
    size_t bytes;
};

// Blocks aimed at for the rows of the chains' levels, many of which no chain
// reaches (32 chats of 16 nodes, the root's too waiting: 26 us, 28 with 512, 30 with 2048).
constexpr int kChainBlocks = 1024;
// Parts of a row at most: the rows of one chat of 16 nodes take 6.8 us (6.1 with
// up to 64 parts), and the move, each of whose blocks joins them, 6.3 (12.5).
constexpr int kMostParts = 16;
// Values of a row of logits: the places of its last block's threads, up to 255 past its end, are ints.
constexpr int kMostVocab = 1 << 30;

static AcceptPlan accept_plan(int tokens, int sequences, int vocab, int levels)
{
    AcceptPlan a{};
    if (vocab) {                                       // (a power of two: see chain_choices)
        a.slots = int(std::max<int64_t>(1, std::min<int64_t>({levels, tokens, 16, kMaxBlocks / sequences})));
        a.splits = 1;
        const int64_t rows = int64_t(sequences) * a.slots;
        while (a.splits < kMostParts && a.splits * rows < kChainBlocks && a.splits * 2048 < vocab) a.splits *= 2;
    }
    a.bytes = size_t(tokens) * a.splits * sizeof(Best);
    return a;
}

static void launch_move(const AcceptParams& p, dim3 grid, hipStream_t s)
{
    switch (p.c.head_dim) {
    case 16: hipLaunchKernelGGL(accept_move_kernel<16>, grid, dim3(kBlock), 0, s, p); break;
    case 32: hipLaunchKernelGGL(accept_move_kernel<32>, grid, dim3(kBlock), 0, s, p); break;
    case 64: hipLaunchKernelGGL(accept_move_kernel<64>, grid, dim3(kBlock), 0, s, p); break;
    default: hipLaunchKernelGGL(accept_move_kernel<128>, grid, dim3(kBlock), 0, s, p); break;
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
    if (tokens < 0 || sequences < 1 || vocab < 0 || vocab > kMostVocab || levels < 1 || levels > kTreeNodes) return 0;
    return std::max<size_t>(256, accept_plan(tokens, sequences, vocab, levels).bytes);
}

extern "C" int hq_pages_accept(const hq_pages* cache, const hq_tree* tree, const int32_t* drafted,
                               const int32_t* choices, const float* logits, int vocab, int levels, int32_t* kept,
                               int32_t* path, int32_t* next, void* workspace, void* stream)
{
    const int bad = tree_check(tree);
    if (bad) return bad;
    PagedBatch batch;
    if (!cache) return HQ_ERR_ARG;
    const int err = paged_check(cache, cache->keys, tree->starts, tree->tokens, cache->kv_heads, cache->values, &batch);
    if (err) return err;
    if (cache->layers < 1 || !cache->status || !kept || !next || !workspace || levels < 1 || levels > kTreeNodes)
        return HQ_ERR_ARG;
    if (tree->tokens && (!drafted || !path || !choices == !logits)) return HQ_ERR_ARG;
    if (logits ? vocab < 1 || vocab > kMostVocab : vocab != 0) return HQ_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return HQ_ERR_ALIGN;
    for (const void* q : {static_cast<const void*>(drafted), static_cast<const void*>(choices),
                          static_cast<const void*>(logits), static_cast<const void*>(kept),
                          static_cast<const void*>(path), static_cast<const void*>(next)})
        if (reinterpret_cast<uintptr_t>(q) & 3u) return HQ_ERR_ALIGN;
    const AcceptPlan a = accept_plan(tree->tokens, cache->sequences, vocab, levels);
    AcceptParams p{*cache, *tree, drafted, choices, logits, vocab, levels, batch.shift, a.slots, a.splits,
                   static_cast<Best*>(workspace), kept, path, next};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t items = int64_t(2) * cache->layers * cache->kv_heads;
    if (items > 0x7fffffff) return HQ_ERR_ARG;
    const int per_block = kTreeWaves * kMoveItems;
    const int slices = int(std::min({(items + per_block - 1) / per_block, kMaxBlocks / cache->sequences,
                                     int64_t(4096)}));
    if (logits && tree->tokens) {
        hipLaunchKernelGGL(accept_chain_kernel, dim3(cache->sequences, a.splits, a.slots), dim3(kBlock), 0, s, p);
    }
    launch_move(p, dim3(cache->sequences, slices), s);
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}
