// hq_paged_attn.hip - hq_paged_attention (hq_paged_attn.h has the kernels).
#include "hq_paged_attn.h"

using namespace hq;

extern "C" size_t hq_paged_attention_workspace_bytes(int tokens, int heads, int kv_heads, int head_dim, int single)
{
    if (tokens < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1) return 0;
    return attn_layout<false>(tokens, kv_heads, head_dim, attn_large<false>(tokens, heads / kv_heads, single != 0)).total;
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
    return run_attention<false>(p, cache, query, window, sinks, output, workspace, static_cast<hipStream_t>(stream));
}
