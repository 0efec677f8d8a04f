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

// Rows of any length: a block a row, which is read three times (the second
// and third from the caches).
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
// values t, t + 256, .. (partial t of the spec's sum).
template <int NPT>
__global__ __launch_bounds__(kBlock) void norm_quant_block_kernel(NormParams p)
{
    __shared__ float red[kBlock];
    const int t = threadIdx.x, n = p.n;
    const size_t at = size_t(blockIdx.x) * n;
    float v[NPT], gam[NPT];
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
        const int i = min(t + kBlock * k, n - 1);
        v[k] = p.x[at + i];
        gam[k] = p.gamma[i];
    }
    if (p.delta) {
        float d[NPT];
#pragma unroll
        for (int k = 0; k < NPT; ++k) d[k] = p.delta[at + min(t + kBlock * k, n - 1)];
#pragma unroll
        for (int k = 0; k < NPT; ++k) v[k] = v[k] + d[k];
    }
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NPT; ++k)
        if (t + kBlock * k < n) ss = __builtin_fmaf(v[k], v[k], ss);
    const float total = block_tree_sum256(ss, red);
    const float r = __builtin_sqrtf(total / float(n) + p.eps);
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
        if (p.sum && t + kBlock * k < n) p.sum[at + t + kBlock * k] = v[k];
        v[k] = (v[k] / r) * gam[k];
        amax = fmaxf(amax, fabsf(v[k]));               // (past n: the last value again)
    }
    amax = fmaxf(block_max_nonneg(amax, red), 1e-5f);
    const float inv = 127.0f / amax;
#pragma unroll
    for (int k = 0; k < NPT; ++k)
        if (t + kBlock * k < n) p.q[at + t + kBlock * k] = quant_i8(v[k], inv);
    if (t == 0) p.act[blockIdx.x] = amax / 127.0f;
}

// Up to 256 QUADS values a row, in fours: a wave a row, lane L its values
// 4 L + j + 256 k, partials 4 L + j of the spec's sum: the tree's levels 128 to
// 4 lie across the lanes, 2 and 1 within one.
template <int QUADS>
__global__ __launch_bounds__(kBlock) void norm_quant_wave_kernel(NormParams p)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int row = blockIdx.x * (kBlock / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (row >= p.rows) return;
    const int quads = p.n / 4;
    const size_t at = size_t(row) * p.n;
    const float4* x = reinterpret_cast<const float4*>(p.x + at);
    float4 v[QUADS];
#pragma unroll
    for (int k = 0; k < QUADS; ++k)
        if (lane + kWave * k < quads) v[k] = x[lane + kWave * k];
        else v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (p.delta) {
        const float4* delta = reinterpret_cast<const float4*>(p.delta + at);
        float4 d[QUADS];
#pragma unroll
        for (int k = 0; k < QUADS; ++k)
            if (lane + kWave * k < quads) d[k] = delta[lane + kWave * k];
#pragma unroll
        for (int k = 0; k < QUADS; ++k)
            if (lane + kWave * k < quads)
                v[k] = make_float4(v[k].x + d[k].x, v[k].y + d[k].y, v[k].z + d[k].z, v[k].w + d[k].w);
    }
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < QUADS; ++k) {                  // (zeros past n change nothing)
        s[0] = __builtin_fmaf(v[k].x, v[k].x, s[0]);
        s[1] = __builtin_fmaf(v[k].y, v[k].y, s[1]);
        s[2] = __builtin_fmaf(v[k].z, v[k].z, s[2]);
        s[3] = __builtin_fmaf(v[k].w, v[k].w, s[3]);
    }
    const float total = (wave_tree_sum64_all(s[0]) + wave_tree_sum64_all(s[2])) +
                        (wave_tree_sum64_all(s[1]) + wave_tree_sum64_all(s[3]));
    const float r = __builtin_sqrtf(total / float(p.n) + p.eps);
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < QUADS; ++k) {
        if (lane + kWave * k >= quads) continue;
        if (p.sum) reinterpret_cast<float4*>(p.sum + at)[lane + kWave * k] = v[k];
        const float4 g = reinterpret_cast<const float4*>(p.gamma)[lane + kWave * k];
        v[k] = make_float4((v[k].x / r) * g.x, (v[k].y / r) * g.y, (v[k].z / r) * g.z, (v[k].w / r) * g.w);
        amax = fmaxf(fmaxf(amax, fabsf(v[k].x)), fmaxf(fabsf(v[k].y), fmaxf(fabsf(v[k].z), fabsf(v[k].w))));
    }
    amax = fmaxf(wave_max64_all(amax), 1e-5f);
    const float inv = 127.0f / amax;
#pragma unroll
    for (int k = 0; k < QUADS; ++k) {
        if (lane + kWave * k >= quads) continue;
        const uint32_t q = uint32_t(uint8_t(quant_i8(v[k].x, inv))) | uint32_t(uint8_t(quant_i8(v[k].y, inv))) << 8 |
                           uint32_t(uint8_t(quant_i8(v[k].z, inv))) << 16 | uint32_t(uint8_t(quant_i8(v[k].w, inv))) << 24;
        reinterpret_cast<uint32_t*>(p.q + at)[lane + kWave * k] = q;
    }
    if (lane == 0) p.act[row] = amax / 127.0f;
}

constexpr int kWaveRows = 512;         // rows from which on a wave takes a row

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
    const bool quads = n % 4 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(delta) |
                                       reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(sum)) & 15u) == 0 &&
                       (reinterpret_cast<uintptr_t>(q) & 3u) == 0;
    if (quads && rows >= kWaveRows && n <= 256 * 16) {
        const dim3 grid((rows + kBlock / kWave - 1) / (kBlock / kWave));
        if (n <= 256 * 4) hipLaunchKernelGGL(norm_quant_wave_kernel<4>, grid, dim3(kBlock), 0, s, p);
        else if (n <= 256 * 8) hipLaunchKernelGGL(norm_quant_wave_kernel<8>, grid, dim3(kBlock), 0, s, p);
        else hipLaunchKernelGGL(norm_quant_wave_kernel<16>, grid, dim3(kBlock), 0, s, p);
    } else if (n <= kBlock * 4) {
        hipLaunchKernelGGL(norm_quant_block_kernel<4>, dim3(rows), dim3(kBlock), 0, s, p);
    } else if (n <= kBlock * 16) {
        hipLaunchKernelGGL(norm_quant_block_kernel<16>, dim3(rows), dim3(kBlock), 0, s, p);
    } else if (n <= kBlock * 40) {
        hipLaunchKernelGGL(norm_quant_block_kernel<40>, dim3(rows), dim3(kBlock), 0, s, p);
    } else {
        hipLaunchKernelGGL(norm_quant_long_kernel, dim3(rows), dim3(kBlock), 0, s, p);
    }
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}
