// hq_norm.hip - residual addition, RMSNorm and int8 quantization of a batch's
// rows (hq_add_rmsnorm_quant): what stands between the int4 products of a batch
// of tokens, in one launch, with the bits of hq_rmsnorm and
// hq_quantize_activation.
#include "hq_device.h"
#include "hq_internal.h"

namespace hq {

struct NormParams {
    const float* x;
    const float* delta;          // nullable
    const float* gamma;
    float* sum;                  // nullable where delta is
    int8_t* q;
    float* act;
    int rows, n;
    float eps;
};

// Longer rows: a block a row, which is read three times, a value a thread at a
// time (the second and third from the caches).  Bound by the latency of its 3 n
// / 256 reads one after another where rows are few (8 rows of 12288 29 us, of
// 16384 40), and by the same beside HBM where they are many (2048 of 12288 111
// us, 3.0 TB/s, of 16384 154; 2048 of 10240 in registers 44, 6.2 TB/s).
__global__ __launch_bounds__(kBlock) void norm_quant_long_kernel(NormParams p)
{
    __shared__ float red[kBlock];
    const size_t at = size_t(blockIdx.x) * p.n;
    const float* src = p.delta ? p.sum : p.x;
    float ss = 0.0f;
    for (int i = threadIdx.x; i < p.n; i += kBlock) {
        float v = p.x[at + i];
        if (p.delta) v = v + p.delta[at + i];
        if (p.sum) p.sum[at + i] = v;
        ss = __builtin_fmaf(v, v, ss);
    }
    const float total = block_tree_sum256(ss, red);
    const float r = __builtin_sqrtf(total / float(p.n) + p.eps);
    float amax = 0.0f;
    for (int i = threadIdx.x; i < p.n; i += kBlock) amax = fmaxf(amax, fabsf((src[at + i] / r) * p.gamma[i]));
    amax = fmaxf(block_max_nonneg(amax, red), 1e-5f);
    const float inv = 127.0f / amax;
    for (int i = threadIdx.x; i < p.n; i += kBlock) p.q[at + i] = quant_i8((src[at + i] / r) * p.gamma[i], inv);
    if (threadIdx.x == 0) p.act[blockIdx.x] = amax / 127.0f;
}

// Up to 256 NPT values a row: a block a row, held in registers, thread t its
// values t, t + 256, .. (partial t of the spec's sum), so that every array is
// read or written once and all of a row's loads are on their way together.
// Bound by HBM for many rows of 2560 (2048: 68 MB in 16.1 us, 4.2 TB/s; 8192:
// 48 us, 5.7 TB/s) and by latency for few (8 rows: 3.8 us, a launch, a round
// trip and three reductions).  A wave a row with its values in fours, whose
// loads and stores are wider and need no barrier, takes longer at every size (8
// rows 5.6 us, 2048 18.5, 8192 58): a wave then has the divisions of a whole row
// to itself, and fewer are on a CU.
template <int NPT>
__global__ __launch_bounds__(kBlock) void norm_quant_kernel(NormParams p)
{
    __shared__ float red[kBlock];
    const int t = threadIdx.x, n = p.n;
    const size_t at = size_t(blockIdx.x) * n;
    // (a row as a buffer: what lies past it reads as zero, which changes neither sum nor maximum, and is not written)
    const auto x = raw_rsrc(p.x + at, 4 * n), gamma = raw_rsrc(p.gamma, 4 * n);
    auto load = [&](__amdgpu_buffer_rsrc_t from, int k) {
        return bits_f32(__builtin_amdgcn_raw_buffer_load_b32(from, 4 * (t + kBlock * k), 0, 0));
    };
    float v[NPT], gam[NPT];
#pragma unroll
    for (int k = 0; k < NPT; ++k) v[k] = load(x, k);
    if (p.delta) {
        const auto delta = raw_rsrc(p.delta + at, 4 * n);
        float d[NPT];
#pragma unroll
        for (int k = 0; k < NPT; ++k) d[k] = load(delta, k);
#pragma unroll
        for (int k = 0; k < NPT; ++k) gam[k] = load(gamma, k);
#pragma unroll
        for (int k = 0; k < NPT; ++k) v[k] = v[k] + d[k];
    } else {
#pragma unroll
        for (int k = 0; k < NPT; ++k) gam[k] = load(gamma, k);
    }
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NPT; ++k) ss = __builtin_fmaf(v[k], v[k], ss);
    const float total = block_tree_sum256(ss, red);
    if (p.sum) {
        const auto sum = raw_rsrc(p.sum + at, 4 * n);
#pragma unroll
        for (int k = 0; k < NPT; ++k)
            __builtin_amdgcn_raw_buffer_store_b32(f32_bits(v[k]), sum, 4 * (t + kBlock * k), 0, 0);
    }
    const float r = __builtin_sqrtf(total / float(n) + p.eps);
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
        v[k] = (v[k] / r) * gam[k];
        amax = fmaxf(amax, fabsf(v[k]));               // (past n: 0, or a NaN, which does not count)
    }
    amax = fmaxf(block_max_nonneg(amax, red), 1e-5f);
    const float inv = 127.0f / amax;
    const auto q = raw_rsrc(p.q + at, n);
#pragma unroll
    for (int k = 0; k < NPT; ++k)
        __builtin_amdgcn_raw_buffer_store_b8(uint8_t(quant_i8(v[k], inv)), q, t + kBlock * k, 0, 0);
    if (t == 0) p.act[blockIdx.x] = amax / 127.0f;
}

}  // namespace hq

using namespace hq;

extern "C" int hq_add_rmsnorm_quant(const float* x, const float* delta, const float* gamma, float* sum, int8_t* q,
                                    float* act_scales, int rows, int n, float eps, void* stream)
{
    if (!x || !gamma || !q || !act_scales || (delta && !sum) || rows < 0 || rows > 0xffffff || n < 1 || n > 1 << 30)
        return HQ_ERR_ARG;
    for (const void* f : {static_cast<const void*>(x), static_cast<const void*>(delta), static_cast<const void*>(gamma),
                          static_cast<const void*>(sum), static_cast<const void*>(act_scales)})
        if (reinterpret_cast<uintptr_t>(f) & 3u) return HQ_ERR_ALIGN;
    if (rows == 0) return HQ_OK;
    const NormParams p{x, delta, gamma, sum, q, act_scales, rows, n, eps};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n <= kBlock * 4) hipLaunchKernelGGL(norm_quant_kernel<4>, dim3(rows), dim3(kBlock), 0, s, p);
    else if (n <= kBlock * 16) hipLaunchKernelGGL(norm_quant_kernel<16>, dim3(rows), dim3(kBlock), 0, s, p);
    else if (n <= kBlock * 40) hipLaunchKernelGGL(norm_quant_kernel<40>, dim3(rows), dim3(kBlock), 0, s, p);
    else hipLaunchKernelGGL(norm_quant_long_kernel, dim3(rows), dim3(kBlock), 0, s, p);
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}
