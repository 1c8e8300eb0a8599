// Attention of sequences that share their first pages (paged_attn.h): bf16 pages.
#include "paged_attn.h"

using namespace alv;

namespace alv {

int shared8_simple(const uint16_t* q, int64_t ld_q, const void* kpages, const void* vpages, int64_t k_stride, int64_t v_stride,
                   const uint8_t* scales, int64_t s_stride, int pages, int page_size, const int32_t* page_table,
                   int64_t ld_table, int max_pages, const int32_t* q_start, const int32_t* kv_len, int B, int T, int max_q,
                   const int32_t* group_start, const int32_t* shared_len, int groups, int heads, int kv_heads, int D,
                   int window, int sinks, float scale, uint16_t* out, int64_t ld_out, void* stream);

namespace {

// What kPre leaves (D values, a maximum and a sum for each row and head), then the
// two runs' own workspace, one after the other's.
struct SharedPlan {
    AttnPlan pre, suf;
    uint64_t pre_bytes, bytes;
};

SharedPlan shared_plan(int heads, int kv_heads, int D, int B, int T, int max_q, int groups) {
    SharedPlan p{};
    p.suf = attn_plan(heads, kv_heads, D, B, T, max_q);
    p.bytes = p.suf.part_bytes;
    if (groups > 0) {
        p.pre = attn_plan(heads, kv_heads, D, groups, T, 0);
        p.pre_bytes = ((uint64_t)T * heads * (D + 2) * sizeof(float) + 15) / 16 * 16;
        p.bytes = p.pre_bytes + std::max(p.pre.part_bytes, p.suf.part_bytes);
    }
    return p;
}

}  // namespace
}  // namespace alv

extern "C" uint64_t alv_attention_shared_workspace(int heads, int kv_heads, int D, int B, int T, int max_q, int groups) {
    if (heads < 1 || heads > kMaxHeads || kv_heads < 1 || heads % kv_heads || D < 1 || D > 512 || B < 1 || T < 1 || max_q < 0 ||
        groups < 0)
        return 0;
    return shared_plan(heads, kv_heads, D, B, T, max_q, groups).bytes;
}

extern "C" int alv_attention_shared(const uint16_t* q, int64_t ld_q, const void* kpages, const void* vpages, int64_t k_stride,
                                    int64_t v_stride, const uint8_t* scales, int64_t s_stride, int pages, int page_size,
                                    const int32_t* page_table, int64_t ld_table, int max_pages, const int32_t* q_start,
                                    const int32_t* kv_len, int B, int T, int max_q, const int32_t* group_start,
                                    const int32_t* shared_len, int groups, int heads, int kv_heads, int D, int window,
                                    int sinks, float scale, uint16_t* out, int64_t ld_out, void* workspace,
                                    uint64_t workspace_bytes, void* stream) {
    PagedAttnArgs a{};
    a.q = q, a.ld_q = ld_q, a.kpages = static_cast<const uint16_t*>(kpages), a.vpages = static_cast<const uint16_t*>(vpages);
    a.k_stride = k_stride, a.v_stride = v_stride, a.heads = heads, a.kv_heads = kv_heads, a.window = window, a.sinks = sinks;
    a.scale = scale, a.out = out, a.ld_out = ld_out;
    if (groups < 0 || (groups > 0 && (!group_start || !shared_len))) return fail(ALV_ERR_ARG, "bad groups: %d", groups);
    if (reinterpret_cast<uintptr_t>(group_start) % 4 || reinterpret_cast<uintptr_t>(shared_len) % 4)
        return fail(ALV_ERR_ALIGN, "group_start and shared_len need 4-byte alignment");
    if (int rc = attn_check(&a, D, page_table, ld_table, max_pages, q_start, kv_len, B, T, pages, page_size, max_q)) return rc;
    if (scales)
        return shared8_simple(q, ld_q, kpages, vpages, k_stride, v_stride, scales, s_stride, pages, page_size, page_table,
                              ld_table, max_pages, q_start, kv_len, B, T, max_q, group_start, shared_len, groups, heads,
                              kv_heads, D, window, sinks, scale, out, ld_out, stream);
    if (T == 0) return ALV_OK;
    const SharedPlan p = shared_plan(heads, kv_heads, D, B, T, max_q, groups);
    if (int rc = attn_fits(p.pre, T, heads, groups)) return rc;
    if (int rc = attn_fits(p.suf, T, heads, B)) return rc;
    if (int rc = attn_workspace(workspace, workspace_bytes, p.bytes)) return rc;
    const hipStream_t s = (hipStream_t)stream;
    if (groups == 0) {
        a.part = static_cast<float*>(workspace);
        return attn_launch<kSuf>(a, D, p.suf, s);
    }
    a.gr = PagedGroups{group_start, shared_len, groups};
    a.pre = static_cast<float*>(workspace);
    a.pre_ml = a.pre + (int64_t)T * heads * D;
    a.part = a.pre + p.pre_bytes / sizeof(float);
    if (int rc = attn_launch<kPre>(a, D, p.pre, s)) return rc;
    return attn_launch<kSuf>(a, D, p.suf, s);
}
