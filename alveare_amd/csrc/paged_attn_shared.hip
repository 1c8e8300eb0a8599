// Attention of sequences that share their first pages: the entry, and bf16 pages.
#include "paged_attn_shared.h"

using namespace alv;

extern "C" uint64_t alv_attention_shared_workspace(int heads, int kv_heads, int D, int B, int T, int max_q, int groups) {
    if (heads < 1 || heads > kMaxHeads || kv_heads < 1 || heads % kv_heads || D < 1 || D > 512 || B < 1 || T < 1 || max_q < 0 ||
        groups < 0)
        return 0;
    if (groups == 0)
        return std::max(alv_attention_paged_workspace(heads, kv_heads, D, B, T, max_q),
                        alv_attention_paged8_workspace(heads, kv_heads, D, B, T, max_q));
    return std::max(shared_plan(heads, kv_heads, D, B, T, max_q, groups, false).bytes,
                    shared_plan(heads, kv_heads, D, B, T, max_q, groups, true).bytes);
}

extern "C" int alv_attention_shared(const uint16_t* q, int64_t ld_q, const void* kpages, const void* vpages, int64_t k_stride,
                                    int64_t v_stride, const uint8_t* scales, int64_t s_stride, int pages, int page_size,
                                    const int32_t* page_table, int64_t ld_table, int max_pages, const int32_t* q_start,
                                    const int32_t* kv_len, int B, int T, int max_q, const int32_t* group_start,
                                    const int32_t* shared_len, int groups, int heads, int kv_heads, int D, int window,
                                    int sinks, float scale, uint16_t* out, int64_t ld_out, void* workspace,
                                    uint64_t workspace_bytes, void* stream) {
    if (groups < 0) return fail(ALV_ERR_ARG, "bad groups: %d", groups);
    if (groups == 0 && scales)
        return alv_attention_paged8(q, ld_q, static_cast<const uint8_t*>(kpages), static_cast<const uint8_t*>(vpages), k_stride,
                                    v_stride, scales, s_stride, pages, page_size, page_table, ld_table, max_pages, q_start,
                                    kv_len, B, T, max_q, heads, kv_heads, D, window, sinks, scale, out, ld_out, workspace,
                                    workspace_bytes, stream);
    if (groups == 0)
        return alv_attention_paged(q, ld_q, static_cast<const uint16_t*>(kpages), static_cast<const uint16_t*>(vpages), k_stride,
                                   v_stride, pages, page_size, page_table, ld_table, max_pages, q_start, kv_len, B, T, max_q,
                                   heads, kv_heads, D, window, sinks, scale, out, ld_out, workspace, workspace_bytes, stream);
    const SharedCall c{q, ld_q, kpages, vpages, k_stride, v_stride, scales, s_stride, pages, page_size, page_table, ld_table,
                       max_pages, q_start, kv_len, B, T, max_q, group_start, shared_len, groups, heads, kv_heads, D, window,
                       sinks, scale, out, ld_out, workspace, workspace_bytes, stream};
    return scales ? attention_shared8(c) : attention_shared<false>(c);
}
