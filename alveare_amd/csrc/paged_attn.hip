// Attention of the newest tokens of a batch of sequences over a paged KV cache.
#include <algorithm>

#include "paged.h"
#include "q4_device.h"
#include "row_norm.h"

namespace alv {

namespace {

struct PagedAttnArgs {
    PagedBatch b;
    const uint16_t* q;
    int64_t ld_q;
    const uint16_t* kpages;
    const uint16_t* vpages;
    int64_t k_stride, v_stride;
    int heads, kv_heads, g;
    int window, sinks;
    float scale;
    uint16_t* out;
    int64_t ld_out;
};

// One wave per (row, q head), one position at a time.
template <int D>
__global__ void __launch_bounds__(64) attn_paged_simple_kernel(PagedAttnArgs a) {
    constexpr int RW = D / 64;
    const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y, kvh = h / a.g;
    const SeqRows sr = find_row(a.b, t, lane);
    if (sr.seq < 0) return;
    float q[RW], o[RW] = {}, m = -__builtin_inff(), l = 0.0f;
    for (int e = 0; e < RW; ++e) q[e] = bf16_bits_to_f32(a.q[t * a.ld_q + h * D + RW * lane + e]);
    const int pos = sr.len - sr.n + (t - sr.first);
    const int lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    for (int p = 0; sr.ok && p <= pos; ++p) {
        if (p < lo && p >= a.sinks) p = lo;
        const int page = page_of(a.b, sr.seq, p);
        if (page < 0) continue;
        const int64_t off = (((int64_t)kvh << a.b.shift) + (p & ((1 << a.b.shift) - 1))) * D + RW * lane;
        const uint16_t* k = a.kpages + page * a.k_stride + off;
        const uint16_t* v = a.vpages + page * a.v_stride + off;
        float s = 0.0f;
        for (int e = 0; e < RW; ++e) s += q[e] * bf16_bits_to_f32(k[e]);
        for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x);
        s *= a.scale;
        const float mn = fmaxf(m, s), f = m == mn ? 1.0f : expf(m - mn), w = expf(s - mn);
        for (int e = 0; e < RW; ++e) o[e] = o[e] * f + w * bf16_bits_to_f32(v[e]);
        l = l * f + w;
        m = mn;
    }
    for (int e = 0; e < RW; ++e)
        a.out[t * a.ld_out + h * D + RW * lane + e] = l == 0.0f ? 0 : bf16_rne_bits(o[e] / l);
}

}  // namespace

}  // namespace alv

using namespace alv;

extern "C" uint64_t alv_attention_paged_workspace(int heads, int kv_heads, int D, int B, int T, int max_q) { return 0; }

extern "C" int alv_attention_paged(const uint16_t* q, int64_t ld_q, const uint16_t* kpages, const uint16_t* vpages,
                                   int64_t k_stride, int64_t v_stride, int pages, int page_size,
                                   const int32_t* page_table, int64_t ld_table, int max_pages, const int32_t* q_start,
                                   const int32_t* kv_len, int B, int T, int max_q, int heads, int kv_heads, int D,
                                   int window, int sinks, float scale, uint16_t* out, int64_t ld_out, void* workspace,
                                   uint64_t workspace_bytes, void* stream) {
    PagedAttnArgs a{};
    if (int rc = paged_batch(page_table, ld_table, max_pages, q_start, kv_len, B, T, pages, page_size, &a.b)) return rc;
    if (!kpages || !vpages || (T > 0 && (!q || !out))) return fail(ALV_ERR_ARG, "null pointer");
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || (D != 64 && D != 128 && D != 256 && D != 512) || window < 0 ||
        sinks < 0 || max_q < 0 || ld_q < (int64_t)heads * D || ld_out < (int64_t)heads * D)
        return fail(ALV_ERR_ARG, "bad attention shape heads=%d kv_heads=%d D=%d window=%d sinks=%d ld_q=%lld ld_out=%lld "
                    "(D one of 64, 128, 256, 512)", heads, kv_heads, D, window, sinks, (long long)ld_q, (long long)ld_out);
    if (!(scale >= 0.0f) || scale > 3e38f) return fail(ALV_ERR_ARG, "scale %g: finite and not negative", (double)scale);
    const int64_t page_values = (int64_t)kv_heads * page_size * D;
    if (k_stride < page_values || v_stride < page_values)
        return fail(ALV_ERR_ARG, "page strides %lld and %lld hold fewer than the page's %lld values", (long long)k_stride,
                    (long long)v_stride, (long long)page_values);
    if (reinterpret_cast<uintptr_t>(kpages) % 16 || reinterpret_cast<uintptr_t>(vpages) % 16 || k_stride % 8 ||
        v_stride % 8 || reinterpret_cast<uintptr_t>(q) % 16 || ld_q % 8 || reinterpret_cast<uintptr_t>(out) % 8 ||
        ld_out % 4)
        return fail(ALV_ERR_ALIGN, "q, kpages and vpages and their rows need 16-byte alignment, out and its rows 8-byte");
    if (T == 0) return ALV_OK;
    a.q = q, a.ld_q = ld_q, a.kpages = kpages, a.vpages = vpages, a.k_stride = k_stride, a.v_stride = v_stride;
    a.heads = heads, a.kv_heads = kv_heads, a.g = heads / kv_heads, a.window = window, a.sinks = sinks, a.scale = scale;
    a.out = out, a.ld_out = ld_out;
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, dim3(T, heads), dim3(64), 0, (hipStream_t)stream, a);
        return hip_check(hipGetLastError(), "attn_paged_kernel launch");
    };
    switch (D) {
        case 64: return go(attn_paged_simple_kernel<64>);
        case 128: return go(attn_paged_simple_kernel<128>);
        case 256: return go(attn_paged_simple_kernel<256>);
        default: return go(attn_paged_simple_kernel<512>);
    }
}
