// hq_pages.hip - management of the paged K/V cache on gfx950: growth and
// release of sequences (hq_pages_resize), forks (hq_pages_fork) and
// compaction (hq_pages_compact).  No reference counterpart.
//
// All of it runs on the device, so that a captured step can cross a page
// border without the host.  A page is free while no table entry holds it
// (refs = 0) and allocation takes the lowest free pages, so every call's
// outcome is a function of the tables alone, whatever order its atomics run
// in.  Each call is two launches (a fork of a small table one):
//   plan    one block (resize, compact): counts, prefix sums, the list of free
//           pages; decides whether the call can be done at all
//   apply   many blocks: table rows, reference counts and the page copies
// A copy's source may be released by the same call and its target was free
// before it, so copies and releases need no order between them.
#include <algorithm>

#include "hq_device.h"
#include "hq_internal.h"
#include "hq_paged.h"

namespace hq {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;
constexpr int kPlanSlots = 2 * kPlanThreads;   // (half of them free at least)
constexpr int kPlanStep = 16;          // pages a lane looks at per round of the free-page search

struct PagesParams {
    hq_pages c;
    int32_t shift;                     // log2(page_size)
    const int32_t* want;               // resize: new lengths; fork: parents
    int window, sinks;                 // resize
    int32_t* live;                     // compact (nullable)
    int32_t* head;                     // workspace: [0] go, [1] copies, [2] pages in use
    int32_t* a;                        // resize: first new page's rank per row; compact: sources
    int32_t* b;                        // resize: copy flags per row; compact: targets
    int32_t* free_list;                // resize
    int32_t* owner;                    // resize: per page, the first row growing in it
    int32_t* count;                    // resize: per page, the rows growing in it
    int32_t* items;                    // resize: per copy the source, the target's rank, the positions filled
    int32_t* snapshot;                 // fork: the table, then the lengths
};

// Block-wide exclusive prefix sum over 1024 threads; total in *total.
__device__ __forceinline__ int plan_scan(int v, int* wave_sum, int* total)
{
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int incl = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int y = __shfl_up(incl, o, kWave);
        if (lane >= o) incl += y;
    }
    __syncthreads();                   // wave_sum's last readers
    if (lane == kWave - 1) wave_sum[wave] = incl;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        before += w < wave ? wave_sum[w] : 0;
        sum += wave_sum[w];
    }
    *total = sum;
    return before + incl - v;
}

// What hq_pages_resize does to one row.
struct ResizeRow {
    int old_len, new_len;
    int old_entries, new_entries;      // table entries the two lengths need
    int source;                        // page the growth goes on writing to, or -1
    bool bad;
};

__device__ __forceinline__ ResizeRow resize_row(const PagesParams& p, int r)
{
    ResizeRow d;
    const int ps = p.c.page_size;
    d.old_len = p.c.lengths[r];
    const int want = p.want[r];
    d.new_len = want < 0 ? d.old_len : want;
    d.bad = d.old_len < 0 || int64_t(d.old_len) > int64_t(p.c.max_pages) * ps;
    d.old_entries = int((int64_t(d.old_len) + ps - 1) >> p.shift);
    d.new_entries = int((int64_t(d.new_len) + ps - 1) >> p.shift);
    d.source = -1;
    if (!d.bad && d.new_len > d.old_len && (d.old_len & (ps - 1))) {
        const int e = d.old_len >> p.shift;
        const int page = p.c.table[size_t(r) * p.c.max_pages + e];
        if (page >= 0 && page < p.c.pages) d.source = page;
        else d.bad = true;             // (another in its place would hold some other sequence's rows)
    }
    return d;
}

// The pages free in round `base` of the search: bit `lane` of is_free[k] for
// page base + 1024 wave + 64 k + lane.
__device__ __forceinline__ void free_pages(const PagesParams& p, uint32_t at, uint64_t (&is_free)[kPlanStep])
{
    const uint32_t pages = p.c.pages;
    int refs[kPlanStep];
#pragma unroll
    for (int k = 0; k < kPlanStep; ++k) refs[k] = p.c.refs[min(at + k * kWave, pages - 1)];
#pragma unroll
    for (int k = 0; k < kPlanStep; ++k) is_free[k] = __ballot(at + k * kWave < pages && refs[k] == 0);
}

// Bound by latency: three dependent reads (lengths, table, refs), the first
// 16384 pages' refs beside them, and the block's barriers.  32 rows: 4.0 us
// where nothing is copied, 7.0 with 21 copies.
__global__ __launch_bounds__(kPlanThreads) void resize_plan_kernel(PagesParams p)
{
    __shared__ int wave_sum[kPlanWaves];
    __shared__ int refuse, copies;
    // pages that rows grow in, by open addressing: the page, its rows, the first of them
    __shared__ int page_of[kPlanSlots], grows[kPlanSlots], first_of[kPlanSlots];
    const int t = threadIdx.x;
    const int lane = t & (kWave - 1), wave = t / kWave;
    const int rows = p.c.sequences;
    // up to 1024 rows: a thread keeps its row, and the rows that grow in one page find each other in LDS (1024 forks'
    // growth 24 us; 52 with a search of the rows by each)
    const bool few = rows <= kPlanThreads;
    uint64_t is_free[kPlanStep];
    free_pages(p, wave * kWave * kPlanStep + lane, is_free);
    ResizeRow mine{};
    mine.source = -1;
    int slot = 0;
    for (int i = t; i < kPlanSlots; i += kPlanThreads) {
        page_of[i] = -1;
        grows[i] = 0;
        first_of[i] = rows;
    }
    if (t == 0) refuse = copies = 0;
    __syncthreads();
    for (int r = t; r < rows; r += kPlanThreads) {
        mine = resize_row(p, r);
        if (mine.bad) atomicOr(&refuse, HQ_PAGES_BAD);
        else if (mine.new_entries > p.c.max_pages) atomicOr(&refuse, HQ_PAGES_FULL);
        if (!few && mine.source >= 0) {
            publish_i(p.count + mine.source, 0);
            publish_i(p.owner + mine.source, 0x7fffffff);
        }
    }
    if (few && mine.source >= 0) {
        slot = mine.source & (kPlanSlots - 1);
        while (true) {
            const int held = atomicCAS(&page_of[slot], -1, mine.source);
            if (held == -1 || held == mine.source) break;
            slot = (slot + 1) & (kPlanSlots - 1);
        }
        atomicAdd(&grows[slot], 1);
        atomicMin(&first_of[slot], t);
    }
    if (!few) wait_all_memory();
    __syncthreads();
    if (refuse) {
        if (t == 0) {
            atomicOr(p.c.status, refuse | (refuse & HQ_PAGES_BAD ? HQ_PAGES_REFUSED : 0));
            p.head[0] = 0;
        }
        return;
    }
    if (!few) {
        for (int r = t; r < rows; r += kPlanThreads) {
            const ResizeRow d = resize_row(p, r);
            if (d.source >= 0) {
                atomicAdd(p.count + d.source, 1);
                atomicMin(p.owner + d.source, r);
            }
        }
        wait_all_memory();
        __syncthreads();
    }
    // new pages of each row, in the order of the table's entries
    int need = 0;
    for (int base = 0; base < rows; base += kPlanThreads) {
        const int r = base + t;
        int new_pages = 0;
        bool copied = false;
        if (r < rows) {
            if (!few) mine = resize_row(p, r);
            if (mine.source >= 0) {
                const int held = p.c.refs[mine.source];
                if (held > 1) {
                    const int first = few ? first_of[slot] : read_i(p.owner + mine.source);
                    const int grow = few ? grows[slot] : read_i(p.count + mine.source);
                    copied = !(first == r && grow == held);
                }
            }
            new_pages = max(0, mine.new_entries - mine.old_entries) + (copied ? 1 : 0);
            p.b[r] = copied;
        }
        int total;
        const int rank = plan_scan(new_pages, wave_sum, &total);
        if (r < rows) p.a[r] = need + rank;
        if (copied) {
            int32_t* item = p.items + 3 * atomicAdd(&copies, 1);
            item[0] = mine.source;
            item[1] = need + rank;
            item[2] = mine.old_len & (p.c.page_size - 1);
        }
        // (rows x entries fits the table; past the pool the call is refused)
        need = need > p.c.pages ? need : need + total;
    }
    // the first `need` free pages: a wave looks at 1024 pages a round
    int found = 0;
    for (uint32_t base = 0; base < uint32_t(p.c.pages) && found < need; base += kPlanThreads * kPlanStep) {
        const uint32_t at = base + wave * kWave * kPlanStep + lane;
        if (base > 0) free_pages(p, at, is_free);
        int n = 0;
#pragma unroll
        for (int k = 0; k < kPlanStep; ++k) n += __popcll(is_free[k]);
        int total;
        int rank = found + plan_scan(lane == 0 ? n : 0, wave_sum, &total);
        rank = __builtin_amdgcn_readfirstlane(rank);
#pragma unroll
        for (int k = 0; k < kPlanStep; ++k) {
            const int at_rank = rank + __popcll(is_free[k] & ((uint64_t(1) << lane) - 1));
            if (((is_free[k] >> lane) & 1) && at_rank < need) p.free_list[at_rank] = int(at + k * kWave);
            rank += __popcll(is_free[k]);
        }
        found += total;
    }
    if (t == 0) {
        const bool go = found >= need;
        if (!go) atomicOr(p.c.status, HQ_PAGES_FULL);
        p.head[0] = go;
        p.head[1] = copies;
    }
}

// Copy the first `fill` positions of page `src` to page `dst`, one kv head of
// K or V of one layer a wave: segment s of layers * 2 * kv_heads.
__device__ __forceinline__ void copy_segment(const hq_pages& c, int src, int dst, int fill, int s)
{
    const int h = s % c.kv_heads;
    const int lw = s / c.kv_heads;
    uint16_t* pool = (lw & 1) ? c.values : c.keys;
    const size_t layer = size_t(lw >> 1) * c.pages;
    const size_t head = size_t(c.page_size) * c.head_dim;
    typedef uint32_t piece __attribute__((ext_vector_type(4)));
    const piece* from = reinterpret_cast<const piece*>(pool + ((layer + src) * c.kv_heads + h) * head);
    piece* to = reinterpret_cast<piece*>(pool + ((layer + dst) * c.kv_heads + h) * head);
    const int n = fill * c.head_dim / 8;             // 16-byte pieces (head_dim is a multiple of 16)
    int i = threadIdx.x & (kWave - 1);
    for (; i + 3 * kWave < n; i += 4 * kWave) {      // four loads under way, then the stores
        const piece x0 = from[i], x1 = from[i + kWave], x2 = from[i + 2 * kWave], x3 = from[i + 3 * kWave];
        to[i] = x0;
        to[i + kWave] = x1;
        to[i + 2 * kWave] = x2;
        to[i + 3 * kWave] = x3;
    }
    for (; i < n; i += kWave) to[i] = from[i];
}

// 32 rows without a copy 3.8 us; with 21 copies in 36 layers (24 MB each way, of
// pages that the last-level cache holds) 7.1.
__global__ __launch_bounds__(kBlock) void resize_apply_kernel(PagesParams p)
{
    if (p.head[0] == 0) return;
    const hq_pages& c = p.c;
    for (int r = blockIdx.x; r < c.sequences; r += gridDim.x) {
        const ResizeRow d = resize_row(p, r);
        const int rank = p.a[r];
        const bool fresh_source = p.b[r] != 0;
        const int e0 = d.old_len >> p.shift;             // the partly filled page's entry
        // positions no query from here on sees: [sinks, low)
        const int64_t low = p.window > 0 ? int64_t(min(d.old_len, d.new_len)) - p.window + 1 : 0;
        __syncthreads();                                 // every thread has read the row
        for (int e = threadIdx.x; e < c.max_pages; e += kBlock) {
            int32_t* entry = c.table + size_t(r) * c.max_pages + e;
            const int page = *entry;
            const bool held = page >= 0 && page < c.pages;
            const bool replaced = fresh_source && e == e0;
            const bool added = e >= d.old_entries && e < d.new_entries;
            int now = page;
            if (replaced) now = p.free_list[rank];
            else if (added) now = p.free_list[rank + (fresh_source ? 1 : 0) + e - d.old_entries];
            else if (e >= d.new_entries) now = -1;
            else if ((int64_t(e) + 1) << p.shift <= low && int64_t(e) << p.shift >= p.sinks) now = -1;
            if (now != page) {
                if (held) atomicSub(c.refs + page, 1);
                if (replaced || added) atomicAdd(c.refs + now, 1);
                *entry = now;
            }
        }
        if (threadIdx.x == 0) c.lengths[r] = d.new_len;
    }
    // page copies, spread over all the launch's waves
    const int waves = gridDim.x * (kBlock / kWave);
    const int segments = c.layers * 2 * c.kv_heads;
    const int64_t all = int64_t(p.head[1]) * segments;
    for (int64_t s = int64_t(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave; s < all; s += waves) {
        const int32_t* item = p.items + 3 * (s / segments);
        copy_segment(c, item[0], p.free_list[item[1]], item[2], int(s % segments));
    }
}

// ------------------------------------------------------------------ forks
__device__ __forceinline__ bool parents_ok(const PagesParams& p)
{
    // every block looks at all of them: all or nothing
    int bad = 0;
    for (int r = threadIdx.x; r < p.c.sequences; r += kBlock) bad |= p.want[r] >= p.c.sequences;
    return !__syncthreads_or(bad);
}

// Tables of up to kForkEntries entries: one block, which holds all that the
// rows take over before it writes any (32 rows: 3.7 to 4.2 us).
constexpr int kForkPer = 16, kForkEntries = kForkPer * kPlanThreads;

__global__ __launch_bounds__(kPlanThreads) void fork_small_kernel(PagesParams p)
{
    const hq_pages& c = p.c;
    const int t = threadIdx.x, entries = c.sequences * c.max_pages;
    int now[kForkPer], was[kForkPer], bad = 0;
#pragma unroll
    for (int k = 0; k < kForkPer; ++k) {
        const int i = t + k * kPlanThreads;
        now[k] = was[k] = 0;
        if (i < entries) {
            const int r = i / c.max_pages;
            const int parent = p.want[r];
            bad |= parent >= c.sequences;
            was[k] = c.table[i];
            now[k] = parent < 0 || parent >= c.sequences ? was[k] : c.table[i + (parent - r) * c.max_pages];
        }
    }
    // (at most as many rows as entries: a row's length to the thread of its number, several rows a thread)
    int lengths[kForkPer];
#pragma unroll
    for (int k = 0; k < kForkPer; ++k) {
        const int r = t + k * kPlanThreads;
        lengths[k] = 0;
        if (r < c.sequences) {
            const int parent = p.want[r];
            lengths[k] = c.lengths[parent < 0 || parent >= c.sequences ? r : parent];
        }
    }
    if (__syncthreads_or(bad)) {
        if (t == 0) atomicOr(c.status, HQ_PAGES_BAD | HQ_PAGES_REFUSED);
        return;
    }
#pragma unroll
    for (int k = 0; k < kForkPer; ++k) {
        const int i = t + k * kPlanThreads;
        if (i < entries && was[k] != now[k]) {
            if (was[k] >= 0 && was[k] < c.pages) atomicSub(c.refs + was[k], 1);
            if (now[k] >= 0 && now[k] < c.pages) atomicAdd(c.refs + now[k], 1);
            c.table[i] = now[k];
        }
        if (i < c.sequences) c.lengths[i] = lengths[k];
    }
}

__global__ __launch_bounds__(kBlock) void fork_snapshot_kernel(PagesParams p)
{
    const int r = blockIdx.x;
    const size_t row = size_t(r) * p.c.max_pages;
    for (int e = threadIdx.x; e < p.c.max_pages; e += kBlock) p.snapshot[row + e] = p.c.table[row + e];
    if (threadIdx.x == 0) p.snapshot[size_t(p.c.sequences) * p.c.max_pages + r] = p.c.lengths[r];
}

__global__ __launch_bounds__(kBlock) void fork_rows_kernel(PagesParams p)
{
    const hq_pages& c = p.c;
    const int r = blockIdx.x;
    if (!parents_ok(p)) {
        if (r == 0 && threadIdx.x == 0) atomicOr(c.status, HQ_PAGES_BAD | HQ_PAGES_REFUSED);
        return;
    }
    const int parent = p.want[r];
    if (parent < 0 || parent == r) return;
    const size_t row = size_t(r) * c.max_pages, from = size_t(parent) * c.max_pages;
    for (int e = threadIdx.x; e < c.max_pages; e += kBlock) {
        const int was = p.snapshot[row + e], now = p.snapshot[from + e];
        if (was == now) continue;
        if (was >= 0 && was < c.pages) atomicSub(c.refs + was, 1);
        if (now >= 0 && now < c.pages) atomicAdd(c.refs + now, 1);
        c.table[row + e] = now;
    }
    if (threadIdx.x == 0) c.lengths[r] = p.snapshot[size_t(c.sequences) * c.max_pages + parent];
}

// ------------------------------------------------------------- compaction
// The pages to move (in use, at `live` and above) to a[], the free places below
// `live` to b[], both ascending: a[i] goes to b[i].
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(PagesParams p)
{
    __shared__ int wave_sum[kPlanWaves];
    const int t = threadIdx.x;
    const int lane = t & (kWave - 1), wave = t / kWave;
    const uint32_t pages = p.c.pages;
    const uint32_t round = kPlanThreads * kPlanStep;
    uint64_t used[kPlanStep];              // of the round looked at last
    auto look = [&](uint32_t at) {
        int refs[kPlanStep];
#pragma unroll
        for (int k = 0; k < kPlanStep; ++k) refs[k] = p.c.refs[min(at + k * kWave, pages - 1)];
#pragma unroll
        for (int k = 0; k < kPlanStep; ++k) used[k] = __ballot(at + k * kWave < pages && refs[k] > 0);
    };
    int n = 0;
    for (uint32_t base = 0; base < pages; base += round) {
        look(base + wave * kWave * kPlanStep + lane);
#pragma unroll
        for (int k = 0; k < kPlanStep; ++k) n += __popcll(used[k]);
    }
    int live;
    plan_scan(lane == 0 ? n : 0, wave_sum, &live);
    int sources = 0, targets = 0;
    for (uint32_t base = 0; base < pages; base += round) {
        const uint32_t at = base + wave * kWave * kPlanStep + lane;
        if (pages > round) look(at);
        int above = 0, below = 0;
#pragma unroll
        for (int k = 0; k < kPlanStep; ++k) {
            const uint32_t page = at + k * kWave;
            above += __popcll(used[k] & __ballot(page >= uint32_t(live)));
            below += __popcll(~used[k] & __ballot(page < uint32_t(live)));
        }
        // (both fit 15 bits a round: one sum for the two)
        int total;
        const int ranks = plan_scan(lane == 0 ? above << 16 | below : 0, wave_sum, &total);
        int rank_above = sources + (__builtin_amdgcn_readfirstlane(ranks) >> 16);
        int rank_below = targets + (__builtin_amdgcn_readfirstlane(ranks) & 0xFFFF);
        const uint64_t under = (uint64_t(1) << lane) - 1;
#pragma unroll
        for (int k = 0; k < kPlanStep; ++k) {
            const uint32_t page = at + k * kWave;
            const uint64_t up = used[k] & __ballot(page >= uint32_t(live));
            const uint64_t down = ~used[k] & __ballot(page < uint32_t(live));
            if ((up >> lane) & 1) p.a[rank_above + __popcll(up & under)] = int(page);
            if ((down >> lane) & 1) p.b[rank_below + __popcll(down & under)] = int(page);
            rank_above += __popcll(up);
            rank_below += __popcll(down);
        }
        sources += total >> 16;
        targets += total & 0xFFFF;
    }
    if (t == 0) {
        p.head[1] = sources;
        p.head[2] = live;
        if (p.live) *p.live = live;
    }
}

// Bound by HBM: 89 pages of 16 positions in 36 layers, 420 MB read and written
// in 84 us, 5.0 TB/s.
__global__ __launch_bounds__(kBlock) void compact_apply_kernel(PagesParams p)
{
    const hq_pages& c = p.c;
    const int moves = p.head[1], live = p.head[2];
    if (moves == 0) return;
    const int64_t threads = int64_t(gridDim.x) * kBlock;
    const int64_t first = int64_t(blockIdx.x) * kBlock + threadIdx.x;
    for (int64_t i = first; i < int64_t(c.sequences) * c.max_pages; i += threads) {
        const int page = c.table[i];
        if (page < live || page >= c.pages) continue;
        int lo = 0, hi = moves;            // its place among the pages that move
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (p.a[mid] < page) lo = mid + 1;
            else hi = mid;
        }
        if (lo < moves && p.a[lo] == page) c.table[i] = p.b[lo];
    }
    for (int64_t i = first; i < moves; i += threads) {
        c.refs[p.b[i]] = c.refs[p.a[i]];
        c.refs[p.a[i]] = 0;
    }
    const int waves = gridDim.x * (kBlock / kWave);
    const int segments = c.layers * 2 * c.kv_heads;
    for (int64_t s = first / kWave; s < int64_t(moves) * segments; s += waves) {
        const int i = int(s / segments);
        copy_segment(c, p.a[i], p.b[i], c.page_size, int(s % segments));
    }
}

// ------------------------------------------------------------------- host
static size_t al256g(size_t v) { return (v + 255) & ~size_t(255); }

static bool pages_shape_ok(const hq_pages* c)
{
    if (!c || c->layers < 1 || c->pages < 1 || c->kv_heads < 1 || c->sequences < 1 || c->max_pages < 1) return false;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return false;
    if (c->head_dim != 16 && c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return false;
    // (a fork of a large table has a block a sequence)
    if (c->sequences > kMaxBlocks) return false;
    // a length is an int, and so is a table's size
    return int64_t(c->max_pages) * c->page_size <= kMaxPositions && int64_t(c->sequences) * c->max_pages <= 0x7fffffff;
}

static PagesParams pages_params(const hq_pages* c, void* workspace)
{
    PagesParams p{};
    p.c = *c;
    p.shift = __builtin_ctz(unsigned(c->page_size));
    char* at = static_cast<char*>(workspace);
    auto take = [&](size_t ints) {
        int32_t* here = reinterpret_cast<int32_t*>(at);
        at += al256g(ints * 4);
        return here;
    };
    const size_t wide = std::max(c->sequences, c->pages);
    p.head = take(64);
    p.a = take(wide);
    p.b = take(wide);
    p.count = take(c->pages);
    p.owner = take(c->pages);
    p.free_list = take(c->pages);
    p.items = take(size_t(3) * c->sequences);
    p.snapshot = take(size_t(c->sequences) * c->max_pages + c->sequences);
    return p;
}

// blocks of 256 threads for page copies: 16 a CU (1024 to 8192 blocks differ by 2 %)
constexpr int kCopyBlocks = 4096;

}  // namespace hq

using namespace hq;

extern "C" size_t hq_pages_workspace_bytes(const hq_pages* cache)
{
    if (!pages_shape_ok(cache)) return 0;
    const PagesParams p = pages_params(cache, nullptr);
    return size_t(reinterpret_cast<uintptr_t>(p.snapshot)) +
           al256g((size_t(cache->sequences) * cache->max_pages + cache->sequences) * 4);
}

extern "C" int hq_pages_resize(const hq_pages* cache, const int32_t* new_lengths, int window, int sinks,
                               void* workspace, void* stream)
{
    if (!pages_shape_ok(cache) || !new_lengths || !workspace || window < 0 || sinks < 0) return HQ_ERR_ARG;
    if (!cache->keys || !cache->values || !cache->table || !cache->lengths || !cache->refs || !cache->status)
        return HQ_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(workspace) & 255u) || (reinterpret_cast<uintptr_t>(cache->keys) & 15u) ||
        (reinterpret_cast<uintptr_t>(cache->values) & 15u))
        return HQ_ERR_ALIGN;
    hipStream_t s = static_cast<hipStream_t>(stream);
    PagesParams p = pages_params(cache, workspace);
    p.want = new_lengths;
    p.window = window;
    p.sinks = sinks;
    hipLaunchKernelGGL(resize_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
    hipLaunchKernelGGL(resize_apply_kernel, dim3(kCopyBlocks), dim3(kBlock), 0, s, p);
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}

extern "C" int hq_pages_fork(const hq_pages* cache, const int32_t* parents, void* workspace, void* stream)
{
    if (!pages_shape_ok(cache) || !parents || !workspace) return HQ_ERR_ARG;
    if (!cache->table || !cache->lengths || !cache->refs || !cache->status) return HQ_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return HQ_ERR_ALIGN;
    hipStream_t s = static_cast<hipStream_t>(stream);
    PagesParams p = pages_params(cache, workspace);
    p.want = parents;
    if (int64_t(cache->sequences) * cache->max_pages <= kForkEntries) {
        hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
    } else {
        hipLaunchKernelGGL(fork_snapshot_kernel, dim3(cache->sequences), dim3(kBlock), 0, s, p);
        hipLaunchKernelGGL(fork_rows_kernel, dim3(cache->sequences), dim3(kBlock), 0, s, p);
    }
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}

extern "C" int hq_pages_compact(const hq_pages* cache, int32_t* live, void* workspace, void* stream)
{
    if (!pages_shape_ok(cache) || !workspace) return HQ_ERR_ARG;
    if (!cache->keys || !cache->values || !cache->table || !cache->refs) return HQ_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(workspace) & 255u) || (reinterpret_cast<uintptr_t>(cache->keys) & 15u) ||
        (reinterpret_cast<uintptr_t>(cache->values) & 15u))
        return HQ_ERR_ALIGN;
    hipStream_t s = static_cast<hipStream_t>(stream);
    PagesParams p = pages_params(cache, workspace);
    p.live = live;
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
    hipLaunchKernelGGL(compact_apply_kernel, dim3(kCopyBlocks), dim3(kBlock), 0, s, p);
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}
