// hq_tree_attn.hip - hq_paged_attention_tree: the attention of drafted trees'
// nodes over the paged cache (hq_paged_attn.h has the kernels).  No reference
// counterpart.
#include "hq_paged_attn.h"

using namespace hq;

extern "C" size_t hq_paged_attention_tree_workspace_bytes(int tokens, int heads, int kv_heads, int head_dim)
{
    if (tokens < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1) return 0;
    return attn_layout<true>(tokens, kv_heads, head_dim, attn_large<true>(tokens, heads / kv_heads, false)).total;
}

extern "C" int hq_paged_attention_tree(const hq_pages* cache, const float* query, const hq_tree* tree, int heads,
                                       int window, int sinks, float* output, void* workspace, void* stream)
{
    const int bad = tree_check(tree);
    if (bad) return bad;
    PagedAttnParams p;
    const int err = paged_check(cache, query, tree->starts, tree->tokens, heads, output, &p.b);
    if (err) return err;
    if (window < 0 || sinks < 0 || !workspace) return HQ_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return HQ_ERR_ALIGN;
    if (tree->tokens == 0) return HQ_OK;
    p.tree = TreeBatch{tree->depths, tree->ancestors};
    return run_attention<true>(p, cache, query, window, sinks, output, workspace, static_cast<hipStream_t>(stream));
}
