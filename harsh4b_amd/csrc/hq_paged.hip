// hq_paged.hip - append to and attention over the paged K/V cache on gfx950
// (hq_paged_append, hq_paged_attention).  No reference counterpart: the
// reference attends one contiguous cache per session
// (cpu_lightspark.py:389-422), token by token.
//
// Row t of a batch belongs to the sequence b with starts[b] <= t <
// starts[b+1]; its position is lengths[b] - n_b + (t - starts[b]).
#include "hq_device.h"
#include "hq_internal.h"

namespace hq {

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

// The sequence of a batch row (wave-uniform; every lane calls it), or -1; its first row and its rows.
__device__ __forceinline__ int paged_sequence(const PagedBatch& p, int t, int* first, int* count)
{
    if (!p.starts) {
        *first = t;
        *count = 1;
        return t < p.sequences ? t : -1;
    }
    // sequences whose rows all lie at or before t
    const int lane = threadIdx.x & (kWave - 1);
    int b = 0;
    for (int base = 1; base <= p.sequences; base += kWave) {
        const int i = base + lane;
        const int past = __popcll(__ballot(i <= p.sequences && p.starts[i <= p.sequences ? i : 0] <= t));
        b += past;
        if (past < kWave) break;
    }
    if (b >= p.sequences) return -1;
    const int a = p.starts[b], z = p.starts[b + 1];
    *first = a;
    *count = z - a;
    return a < 0 || a > t || z <= t || z > p.tokens ? -1 : b;
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

// --------------------------------------------------------------- attention
struct PagedAttnParams {
    PagedBatch b;
    const float* query;          // [tokens, heads, D]
    float* out;
    int window, sinks;           // window 0: none
};

// Whether the query at position `pos` sees position j (pages aside).
__device__ __forceinline__ bool paged_visible(int pos, int j, int window, int sinks)
{
    return j <= pos && (window == 0 || j > pos - window || j < sinks);
}

// One query row over positions [lo, hi) of sequence b, kv head h, in fp32 and
// one wave: a lane scores one position of 64 at a time, and holds D/64 of the
// output's values.  Online softmax: m the running maximum, l the sum, o the
// weighted values; `seen` whether anything was visible.
template <int D>
__device__ void paged_row(const PagedAttnParams& p, const float* q, int b, int h, int pos, int lo, int hi,
                          float& m, float& l, float (&o)[2], bool& seen)
{
    const int lane = threadIdx.x & (kWave - 1);
    const float scale = 1.0f / __builtin_sqrtf(float(D));
    const size_t head = size_t(p.b.page_size) * D;
    for (int base = lo; base < hi; base += kWave) {
        const int j = base + lane;
        const int page = j < hi ? paged_page(p.b, b, j) : -1;
        const bool visible = page >= 0 && paged_visible(pos, j, p.window, p.sinks);
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

template <int D>
__global__ __launch_bounds__(kBlock) void paged_attention_kernel(PagedAttnParams p)
{
    __shared__ float qs[kBlock / kWave][D];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int t = blockIdx.x;
    const int head = blockIdx.y * (kBlock / kWave) + wave;
    if (head >= p.b.heads) return;
    int first = 0, count = 0;
    const int b = paged_sequence(p.b, t, &first, &count);
    if (b < 0) return;
    const int pos = paged_position(p.b, b, count, t - first);
    const size_t row = (size_t(t) * p.b.heads + head) * D;
    for (int i = lane; i < D; i += kWave) qs[wave][i] = p.query[row + i];
    float m = -__builtin_inff(), l = 0.0f, o[2] = {0.0f, 0.0f};
    bool seen = false;
    const int end = int(min(int64_t(pos) + 1, int64_t(p.b.max_pages) * p.b.page_size));
    const int low = p.window > 0 ? int(max(int64_t(0), int64_t(pos) - p.window + 1)) : 0;
    const int h = head / p.b.groups;
    if (low > 0 && p.sinks > 0) paged_row<D>(p, qs[wave], b, h, pos, 0, min(low, p.sinks), m, l, o, seen);
    paged_row<D>(p, qs[wave], b, h, pos, low, end, m, l, o, seen);
    if (lane < D) p.out[row + lane] = seen ? o[0] / l : 0.0f;
    if (D == 128) p.out[row + lane + 64] = seen ? o[1] / l : 0.0f;
}

// -------------------------------------------------------------------- host
static int paged_check(const hq_pages* c, const void* rows, const int32_t* starts, int tokens, int heads, const void* out,
                       PagedBatch* b)
{
    if (!c || !rows || !out || !c->keys || !c->values || !c->table || !c->lengths) return HQ_ERR_ARG;
    if (c->pages < 1 || c->kv_heads < 1 || c->sequences < 1 || c->max_pages < 1 || tokens < 0) return HQ_ERR_ARG;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return HQ_ERR_ARG;
    if (int64_t(c->max_pages) * c->page_size > 0x7fffffff || int64_t(c->sequences) * c->max_pages > 0x7fffffff)
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

extern "C" size_t hq_paged_attention_workspace_bytes(int tokens, int sequences, int heads, int kv_heads, int head_dim)
{
    if (tokens < 0 || sequences < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1) return 0;
    return 256;
}

extern "C" int hq_paged_attention(const hq_pages* cache, const float* query, const int32_t* starts, int tokens,
                                  int heads, int window, int sinks, float* output, void* workspace, void* stream)
{
    PagedAttnParams p;
    const int err = paged_check(cache, query, starts, tokens, heads, output, &p.b);
    if (err) return err;
    if (window < 0 || sinks < 0 || !workspace) return HQ_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return HQ_ERR_ALIGN;
    if (tokens == 0) return HQ_OK;
    p.query = query;
    p.out = output;
    p.window = window;
    p.sinks = sinks;
    const dim3 grid(tokens, (heads + 3) / 4);
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (cache->head_dim) {
    case 16: hipLaunchKernelGGL(paged_attention_kernel<16>, grid, dim3(kBlock), 0, s, p); break;
    case 32: hipLaunchKernelGGL(paged_attention_kernel<32>, grid, dim3(kBlock), 0, s, p); break;
    case 64: hipLaunchKernelGGL(paged_attention_kernel<64>, grid, dim3(kBlock), 0, s, p); break;
    default: hipLaunchKernelGGL(paged_attention_kernel<128>, grid, dim3(kBlock), 0, s, p); break;
    }
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}
