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

// A block a row, one value a thread at a time.
__global__ __launch_bounds__(kBlock) void norm_quant_kernel(NormParams p)
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
    hipLaunchKernelGGL(norm_quant_kernel, dim3(rows), dim3(kBlock), 0, static_cast<hipStream_t>(stream), p);
    return hipGetLastError() == hipSuccess ? HQ_OK : HQ_ERR_LAUNCH;
}
