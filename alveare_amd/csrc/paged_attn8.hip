// Attention over 8-bit pages (paged_attn.h).
#include "paged_attn.h"

using namespace alv;

extern "C" uint64_t alv_attention_paged8_workspace(int heads, int kv_heads, int D, int B, int T, int max_q) {
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || D < 1 || B < 1 || T < 1 || max_q < 0) return 0;
    return attn_plan(heads, kv_heads, D, B, T, max_q, true).part_bytes;
}

extern "C" int alv_attention_paged8(const uint16_t* q, int64_t ld_q, const uint8_t* kpages, const uint8_t* vpages,
                                    int64_t k_stride, int64_t v_stride, const uint8_t* scales, int64_t s_stride, int pages,
                                    int page_size, const int32_t* page_table, int64_t ld_table, int max_pages,
                                    const int32_t* q_start, const int32_t* kv_len, int B, int T, int max_q, int heads,
                                    int kv_heads, int D, int window, int sinks, float scale, uint16_t* out, int64_t ld_out,
                                    void* workspace, uint64_t workspace_bytes, void* stream) {
    if (!scales) return fail(ALV_ERR_ARG, "null pointer");
    PagedAttnArgs a{};
    a.q = q, a.ld_q = ld_q, a.kpages = kpages, a.vpages = vpages, a.k_stride = k_stride, a.v_stride = v_stride;
    a.scales = scales, a.s_stride = s_stride;
    a.heads = heads, a.kv_heads = kv_heads, a.window = window, a.sinks = sinks, a.scale = scale;
    a.out = out, a.ld_out = ld_out;
    if (int rc = attn_check(&a, D, page_table, ld_table, max_pages, q_start, kv_len, B, T, pages, page_size, max_q)) return rc;
    if (T == 0) return ALV_OK;
    const AttnPlan p = attn_plan(heads, kv_heads, D, B, T, max_q, true);
    if (int rc = attn_fits(p, T, heads, B)) return rc;
    if (int rc = attn_workspace(workspace, workspace_bytes, p.part_bytes)) return rc;
    a.part = static_cast<float*>(workspace);
    return attn_launch<true, false>(a, D, p, (hipStream_t)stream);
}
