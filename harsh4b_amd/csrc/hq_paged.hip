// hq_paged.hip - append to the paged K/V cache on gfx950 (hq_paged_append).
// No reference counterpart: the reference writes one contiguous cache per
// session (cpu_lightspark.py:435-440), token by token.
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
    float* query;                // [tokens, heads, D]
};

// One head's row of one token a wave, as prefill_qk_kernel: the spec's norm
// (64 fmaf partials, halving tree) and rotation, so that K, V and q have the
// decode step's bits.  Bound by HBM (a prompt) or latency (a token a sequence).
template <int D>
__global__ __launch_bounds__(kBlock) void paged_append_kernel(AppendParams p)
{
    constexpr int PER = D == 128 ? 2 : 1;          // values a lane holds
    const int t = blockIdx.x;
    const int slot = blockIdx.y * (kBlock / kWave) + threadIdx.x / kWave;
    const int lane = threadIdx.x & (kWave - 1);
    const int heads = p.b.heads, kv_heads = p.b.kv_heads;
    const int total = heads + 2 * kv_heads;
    if (slot >= total) return;
    const bool in = lane < D;
    const float* src = p.qkv + (size_t(t) * total + slot) * D;
    const float x0 = in ? src[lane] : 0.0f;
    const float x1 = PER == 2 ? src[lane + 64] : 0.0f;
    int first = 0, count = 0;
    const int b = paged_sequence(p.b, t, &first, &count);
    if (b < 0) return;
    const int pos = paged_position(p.b, b, count, t - first);
    const int page = paged_page(p.b, b, pos);
    const bool is_q = slot < heads;
    const bool placed = pos >= 0 && pos < p.rope_positions && page >= 0;
    if (!placed) {
        if (lane == 0) atomicOr(p.b.status, HQ_PAGES_BAD);
        if (is_q && in) {
            float* qd = p.query + (size_t(t) * heads + slot) * D;
            qd[lane] = 0.0f;
            if (PER == 2) qd[lane + 64] = 0.0f;
        }
        return;
    }
    if (!is_q && (*p.b.status & HQ_PAGES_FULL)) return;
    const size_t at = size_t(pos & (p.b.page_size - 1)) * D;
    const size_t head = size_t(p.b.page_size) * D;
    if (slot >= heads + kv_heads) {
        uint16_t* vd = const_cast<uint16_t*>(p.b.values) +
                       (size_t(page) * kv_heads + (slot - heads - kv_heads)) * head + at;
        if (in) vd[lane] = f32_to_f16(x0);
        if (PER == 2) vd[lane + 64] = f32_to_f16(x1);
        return;
    }
    const float* w = is_q ? p.q_norm : p.k_norm;
    float s = __builtin_fmaf(x0, x0, 0.0f);
    if (PER == 2) s = __builtin_fmaf(x1, x1, s);
    const float ss = wave_tree_sum64_all(s);
    const float r = __builtin_sqrtf(ss / float(D) + p.eps);
    // pairs (i, i + D/2): of D = 128 in one lane, else in lanes D/2 apart
    const int i = PER == 2 ? lane : lane & (D / 2 - 1);
    const float c0 = p.rope_cos[size_t(pos) * (D / 2) + i];
    const float s0 = p.rope_sin[size_t(pos) * (D / 2) + i];
    const float y0 = in ? (x0 / r) * w[lane] : 0.0f;
    float a, b2 = 0.0f;
    if (PER == 2) {
        const float y1 = (x1 / r) * w[lane + 64];
        a = y0 * c0 - y1 * s0;
        b2 = y1 * c0 + y0 * s0;
    } else {
        const float other = __shfl_xor(y0, D / 2, kWave);
        a = lane < D / 2 ? y0 * c0 - other * s0 : y0 * c0 + other * s0;
    }
    if (is_q) {
        float* qd = p.query + (size_t(t) * heads + slot) * D;
        if (in) qd[lane] = a;
        if (PER == 2) qd[lane + 64] = b2;
    } else {
        uint16_t* kd = const_cast<uint16_t*>(p.b.keys) + (size_t(page) * kv_heads + (slot - heads)) * head + at;
        if (in) kd[lane] = f32_to_f16(a);
        if (PER == 2) kd[lane + 64] = f32_to_f16(b2);
    }
}

}  // namespace hq

using namespace hq;

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
    const int slots = heads + 2 * cache->kv_heads;
    const dim3 grid(tokens, (slots + 3) / 4);
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (cache->head_dim) {
    case 16: hipLaunchKernelGGL(paged_append_kernel<16>, grid, dim3(kBlock), 0, s, p); break;
    case 32: hipLaunchKernelGGL(paged_append_kernel<32>, grid, dim3(kBlock), 0, s, p); break;
    case 64: hipLaunchKernelGGL(paged_append_kernel<64>, grid, dim3(kBlock), 0, s, p); break;
    default: hipLaunchKernelGGL(paged_append_kernel<128>, grid, dim3(kBlock), 0, s, p); break;
    }
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}
