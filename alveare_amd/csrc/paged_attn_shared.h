// Attention of sequences that share their first pages (paged_attn.h).
#pragma once

#include "paged_attn.h"

namespace alv {

// alv_attention_shared's arguments.
struct SharedCall {
    const uint16_t* q;
    int64_t ld_q;
    const void* kpages;
    const void* vpages;
    int64_t k_stride, v_stride;
    const uint8_t* scales;
    int64_t s_stride;
    int pages, page_size;
    const int32_t* page_table;
    int64_t ld_table;
    int max_pages;
    const int32_t* q_start;
    const int32_t* kv_len;
    int B, T, max_q;
    const int32_t* group_start;
    const int32_t* shared_len;
    int groups, heads, kv_heads, D, window, sinks;
    float scale;
    uint16_t* out;
    int64_t ld_out;
    void* workspace;
    uint64_t workspace_bytes;
    void* stream;
};

int attention_shared8(const SharedCall& c);  // of 8-bit pages

namespace {

// The workspace: where the parts of each (row, head) are, what is kept of them (D values,
// a maximum and a sum, for both halves), then the kernels' parts.
struct SharedPlan {
    AttnPlan p;
    uint64_t rec_bytes, kept_bytes, bytes;
};

__attribute__((unused)) SharedPlan shared_plan(int heads, int kv_heads, int D, int B, int T, int max_q, int groups, bool e8) {
    SharedPlan s{};
    s.p = mix_plan(heads, kv_heads, D, B, T, max_q, groups, e8);
    s.rec_bytes = 2 * (uint64_t)T * heads * sizeof(int4);
    s.kept_bytes = ((uint64_t)T * heads * (D + 2) * sizeof(float) + 15) / 16 * 16;
    s.bytes = s.rec_bytes + 2 * s.kept_bytes + s.p.part_bytes;
    return s;
}

template <bool E8>
int attention_shared(const SharedCall& c) {  // of one group at least
    if (!c.group_start || !c.shared_len) return fail(ALV_ERR_ARG, "null pointer");
    if (reinterpret_cast<uintptr_t>(c.group_start) % 4 || reinterpret_cast<uintptr_t>(c.shared_len) % 4)
        return fail(ALV_ERR_ALIGN, "group_start and shared_len need 4-byte alignment");
    PagedAttnArgs a{};
    a.q = c.q, a.ld_q = c.ld_q, a.kpages = c.kpages, a.vpages = c.vpages, a.k_stride = c.k_stride, a.v_stride = c.v_stride;
    a.scales = c.scales, a.s_stride = c.s_stride;
    a.heads = c.heads, a.kv_heads = c.kv_heads, a.window = c.window, a.sinks = c.sinks, a.scale = c.scale;
    a.out = c.out, a.ld_out = c.ld_out;
    if (int rc = attn_check(&a, c.D, c.page_table, c.ld_table, c.max_pages, c.q_start, c.kv_len, c.B, c.T, c.pages, c.page_size,
                            c.max_q))
        return rc;
    // (groups and sequences are counted together, and every workgroup looks at all)
    if (c.groups > kMaxRows || c.B > kMaxRows)
        return fail(ALV_ERR_RANGE, "%d groups of %d sequences (at most 2^22 of each)", c.groups, c.B);
    if (c.T == 0) return ALV_OK;
    const SharedPlan p = shared_plan(c.heads, c.kv_heads, c.D, c.B, c.T, c.max_q, c.groups, E8);
    if (int rc = attn_fits(p.p, c.T, c.heads, c.B)) return rc;
    if (int rc = attn_workspace(c.workspace, c.workspace_bytes, p.bytes)) return rc;
    const hipStream_t s = (hipStream_t)c.stream;
    a.part = static_cast<float*>(c.workspace);
    a.gr = PagedGroups{c.group_start, c.shared_len, c.groups};
    const int64_t rows = (int64_t)c.T * c.heads;
    a.recs = reinterpret_cast<int4*>(c.workspace);
    a.part += p.rec_bytes / sizeof(float);
    for (int half = 0; half < 2; ++half) {
        a.kept[half] = a.part;
        a.kept_ml[half] = a.part + rows * c.D;
        a.part += p.kept_bytes / sizeof(float);
    }
    return attn_launch<E8, true>(a, c.D, p.p, s);
}

}  // namespace
}  // namespace alv
