// hq_paged.hip - append to the paged K/V cache on gfx950 (hq_paged_append).
// No reference counterpart: the reference writes one contiguous cache per
// session (cpu_lightspark.py:435-440), token by token.
#include <algorithm>

#include "hq_device.h"
#include "hq_internal.h"
#include "hq_paged.h"

namespace hq {

// ------------------------------------------------------------------ append
struct AppendParams {
    PagedBatch b;
    const float* qkv;            // [tokens, (heads + 2 kv_heads) * D]
    const float* q_norm;
    const float* k_norm;
    const float* rope_cos;       // [rope_positions, D/2]
    const float* rope_sin;
    float eps;
    int rope_positions;
    int looks;                   // the first blocks, which look at the starts
    float* query;                // [tokens, heads, D]
};

// A token's heads (q, k, v) over the waves of gridDim.y blocks, PER at a time:
// their loads together, then the spec's norm (64 fmaf partials, halving tree)
// and rotation as the decode step's, so that K, V and q have its bits.  Bound
// by HBM (2000 tokens of 48 heads, 91 MB: 17.0 us, 5.3 TB/s) or latency (32
// single tokens: 3.2 us).
constexpr int kAppendPer = 2;
constexpr int kAppendWide = 1024;      // tokens from which on a block does a whole token

// Starts that are no ranges of the batch's rows are reported, by the launch's
// first blocks, `looks` of them: they cost nothing there (2000 tokens 17.9 us,
// 18.0 without them; behind the rows' blocks 18.3, by the rows' own 18.5).
constexpr int kLookBlocks = 64;

__device__ __forceinline__ void look_at_starts(const PagedBatch& p, int i, int n)
{
    for (int b = i * kBlock + threadIdx.x; b < p.sequences; b += n * kBlock) {
        const int from = p.starts[b], to = p.starts[b + 1];
        if (from < 0 || from > to || to > p.tokens) atomicOr(p.status, HQ_PAGES_BAD);
    }
}

template <int D>
__global__ __launch_bounds__(kBlock) void paged_append_kernel(AppendParams p)
{
    constexpr int VALUES = D == 128 ? 2 : 1;       // a lane holds of a row
    const int t = int(blockIdx.x) - p.looks;
    const int lane = threadIdx.x & (kWave - 1);
    const int heads = p.b.heads, kv_heads = p.b.kv_heads;
    const int total = heads + 2 * kv_heads;
    const bool in = lane < D;
    const int step = gridDim.y * (kBlock / kWave) * kAppendPer;
    int slot0 = (blockIdx.y * (kBlock / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)) * kAppendPer;
    if (slot0 >= total || t < 0) {
        if (t < 0 && blockIdx.y == 0) look_at_starts(p.b, blockIdx.x, p.looks);
        return;
    }
    float x0[kAppendPer], x1[kAppendPer];
    auto load = [&](int from) {
#pragma unroll
        for (int i = 0; i < kAppendPer; ++i) {
            const float* src = p.qkv + (size_t(t) * total + min(from + i, total - 1)) * D;
            x0[i] = in ? src[lane] : 0.0f;
            x1[i] = VALUES == 2 ? src[lane + 64] : 0.0f;
        }
    };
    load(slot0);
    int first = 0, count = 0;
    const int b = paged_sequence(p.b, t, &first, &count);
    if (b < 0) return;
    const int pos = paged_position(p.b, b, count, t - first);
    const int page = paged_page(p.b, b, pos);
    const bool placed = pos >= 0 && pos < p.rope_positions && page >= 0;
    const bool held = (*p.b.status & (HQ_PAGES_FULL | HQ_PAGES_REFUSED)) != 0;
    if (!placed && lane == 0) atomicOr(p.b.status, HQ_PAGES_BAD);
    // pairs (i, i + D/2): of D = 128 in one lane, else in lanes D/2 apart
    const int pair = VALUES == 2 ? lane : lane & (D / 2 - 1);
    const size_t rope = size_t(placed ? pos : 0) * (D / 2) + pair;
    const float cos = p.rope_cos[rope], sin = p.rope_sin[rope];
    const float qw0 = in ? p.q_norm[lane] : 0.0f, kw0 = in ? p.k_norm[lane] : 0.0f;
    const float qw1 = VALUES == 2 ? p.q_norm[lane + 64] : 0.0f, kw1 = VALUES == 2 ? p.k_norm[lane + 64] : 0.0f;
    // this position's K and V rows of kv head 0
    const size_t head = size_t(p.b.page_size) * D;
    const size_t at = size_t(max(page, 0)) * kv_heads * head + size_t(pos & (p.b.page_size - 1)) * D;
    uint16_t* const krow = const_cast<uint16_t*>(p.b.keys) + at;
    uint16_t* const vrow = const_cast<uint16_t*>(p.b.values) + at;
    while (true) {
        float y0[kAppendPer], y1[kAppendPer];
#pragma unroll
        for (int i = 0; i < kAppendPer; ++i) {
            const int slot = slot0 + i;
            if (slot >= heads + kv_heads) {        // v: as it is
                y0[i] = x0[i];
                y1[i] = x1[i];
                continue;
            }
            const bool is_q = slot < heads;
            float s = __builtin_fmaf(x0[i], x0[i], 0.0f);
            if (VALUES == 2) s = __builtin_fmaf(x1[i], x1[i], s);
            const float ss = wave_tree_sum64_all(s);
            const float r = __builtin_sqrtf(ss / float(D) + p.eps);
            const float a = (x0[i] / r) * (is_q ? qw0 : kw0);
            if (VALUES == 2) {
                const float c = (x1[i] / r) * (is_q ? qw1 : kw1);
                y0[i] = a * cos - c * sin;
                y1[i] = c * cos + a * sin;
            } else {
                const float z = in ? a : 0.0f;
                const float other = __shfl_xor(z, D / 2, kWave);
                y0[i] = lane < D / 2 ? z * cos - other * sin : z * cos + other * sin;
                y1[i] = 0.0f;
            }
        }
        const int done = slot0;
        slot0 += step;
        const bool more = slot0 < total;
        if (more) load(slot0);
#pragma unroll
        for (int i = 0; i < kAppendPer; ++i) {
            const int slot = done + i;
            if (slot < heads) {
                float* to = p.query + (size_t(t) * heads + slot) * D;
                if (in) to[lane] = placed ? y0[i] : 0.0f;
                if (VALUES == 2) to[lane + 64] = placed ? y1[i] : 0.0f;
            } else if (slot < total && placed && !held) {
                uint16_t* to = slot < heads + kv_heads ? krow + (slot - heads) * head
                                                       : vrow + (slot - heads - kv_heads) * head;
                if (in) to[lane] = f32_to_f16(y0[i]);
                if (VALUES == 2) to[lane + 64] = f32_to_f16(y1[i]);
            }
        }
        if (!more) return;
    }
}

}  // namespace hq

using namespace hq;

static void launch_append(int head_dim, dim3 grid, hipStream_t s, const AppendParams& p)
{
    switch (head_dim) {
    case 16: hipLaunchKernelGGL(paged_append_kernel<16>, grid, dim3(kBlock), 0, s, p); break;
    case 32: hipLaunchKernelGGL(paged_append_kernel<32>, grid, dim3(kBlock), 0, s, p); break;
    case 64: hipLaunchKernelGGL(paged_append_kernel<64>, grid, dim3(kBlock), 0, s, p); break;
    default: hipLaunchKernelGGL(paged_append_kernel<128>, grid, dim3(kBlock), 0, s, p); break;
    }
}

extern "C" int hq_paged_append(const hq_pages* cache, const float* qkv, const int32_t* starts, int tokens, int heads,
                               const float* q_norm, const float* k_norm, float eps, const float* rope_cos,
                               const float* rope_sin, int rope_positions, float* query, void* stream)
{
    AppendParams p;
    const int err = paged_check(cache, qkv, starts, tokens, heads, query, &p.b);
    if (err) return err;
    if (!q_norm || !k_norm || !rope_cos || !rope_sin || rope_positions < 1 || !cache->status) return HQ_ERR_ARG;
    if (tokens == 0) return HQ_OK;
    p.qkv = qkv;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.rope_cos = rope_cos;
    p.rope_sin = rope_sin;
    p.eps = eps;
    p.rope_positions = rope_positions;
    p.query = query;
    // few tokens: kAppendPer heads a wave; many: a block a token, whose waves look its place up once for all their
    // heads (2000 tokens 17.9 us; with kAppendPer heads a wave 23.1)
    const int slots = heads + 2 * cache->kv_heads;
    const int per_block = kAppendPer * (kBlock / kWave);
    p.looks = starts ? std::min((cache->sequences + kBlock - 1) / kBlock, kLookBlocks) : 0;
    const int y = tokens < kAppendWide ? (slots + per_block - 1) / per_block : 1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (int64_t(tokens) + p.looks > kMaxBlocks) {  // (a launch of their own)
        launch_append(cache->head_dim, dim3(p.looks), s, p);
        p.looks = 0;
    }
    launch_append(cache->head_dim, dim3(tokens + p.looks, y), s, p);
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}
