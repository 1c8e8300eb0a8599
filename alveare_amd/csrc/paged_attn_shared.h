// Attention of sequences that share their first pages (paged_attn.h): one run over
// the groups, one over what is behind what they share.
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

// Two runs: what kPre leaves (D values, a maximum and a sum for each row and head),
// then the runs' own workspace, one after the other's. One (mix.qt > 0): what is kept
// of both parts of a row, where they are, then the line's parts.
struct SharedPlan {
    AttnPlan pre, suf, mix;
    uint64_t rec_bytes, kept_bytes, bytes;
};

__attribute__((unused)) SharedPlan shared_plan(int heads, int kv_heads, int D, int B, int T, int max_q, int groups, bool e8) {
    SharedPlan p{};
    p.suf = attn_plan(heads, kv_heads, D, B, T, max_q, e8);
    p.bytes = p.suf.part_bytes;
    if (groups > 0) {
        p.kept_bytes = ((uint64_t)T * heads * (D + 2) * sizeof(float) + 15) / 16 * 16;
        p.mix = mix_plan(p.suf, heads, kv_heads, D, T, max_q, groups);
        if (p.mix.qt) {
            p.rec_bytes = 2 * (uint64_t)T * heads * sizeof(int4);
            p.bytes = p.rec_bytes + 2 * p.kept_bytes + p.mix.part_bytes;
        } else {
            p.pre = attn_plan(heads, kv_heads, D, groups, T, 0, e8);
            p.bytes = p.kept_bytes + std::max(p.pre.part_bytes, p.suf.part_bytes);
        }
    }
    return p;
}

template <bool E8>
int attention_shared(const SharedCall& c) {
    if (c.groups < 0 || (c.groups > 0 && (!c.group_start || !c.shared_len))) return fail(ALV_ERR_ARG, "bad groups: %d", c.groups);
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
    if (c.T == 0) return ALV_OK;
    const SharedPlan p = shared_plan(c.heads, c.kv_heads, c.D, c.B, c.T, c.max_q, c.groups, E8);
    if (int rc = attn_fits(p.pre, c.T, c.heads, c.groups)) return rc;
    if (int rc = attn_fits(p.suf, c.T, c.heads, c.B)) return rc;
    if (int rc = attn_workspace(c.workspace, c.workspace_bytes, p.bytes)) return rc;
    const hipStream_t s = (hipStream_t)c.stream;
    a.part = static_cast<float*>(c.workspace);
    if (c.groups == 0) return attn_launch<E8, kSuf>(a, c.D, p.suf, s);
    a.gr = PagedGroups{c.group_start, c.shared_len, c.groups};
    const int64_t rows = (int64_t)c.T * c.heads;
    a.recs = reinterpret_cast<int4*>(c.workspace);
    a.pre = a.part + p.rec_bytes / sizeof(float);
    a.pre_ml = a.pre + rows * c.D;
    a.suf = a.pre + p.kept_bytes / sizeof(float);
    a.suf_ml = a.suf + rows * c.D;
    if (p.mix.qt) {
        a.part = a.suf + p.kept_bytes / sizeof(float);
        return attn_launch<E8, kMix>(a, c.D, p.mix, s);
    }
    a.part = a.suf;
    if (int rc = attn_launch<E8, kPre>(a, c.D, p.pre, s)) return rc;
    return attn_launch<E8, kSuf>(a, c.D, p.suf, s);
}

}  // namespace
}  // namespace alv
