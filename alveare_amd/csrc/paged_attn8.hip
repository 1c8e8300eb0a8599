// Attention over 8-bit pages, and of sequences that share their first pages.
//
// out = sum_p w_p v_p / sum_p w_p with w_p = exp(scale q.k_p - m), as paged_attn.hip
// has it; a value of an 8-bit page is code * 2^(scale - 127). The positions that a
// group shares are read from its first sequence's pages.
//
// One wave per (row, head): a lane per position for the scores, D / 64 columns per
// lane for the output.
#include <limits.h>

#include "paged.h"
#include "q4_device.h"
#include "row_norm.h"

namespace alv {

int shared8_simple(const uint16_t* q, int64_t ld_q, const void* kpages, const void* vpages, int64_t k_stride, int64_t v_stride,
                   const uint8_t* scales, int64_t s_stride, int pages, int page_size, const int32_t* page_table,
                   int64_t ld_table, int max_pages, const int32_t* q_start, const int32_t* kv_len, int B, int T, int max_q,
                   const int32_t* group_start, const int32_t* shared_len, int groups, int heads, int kv_heads, int D,
                   int window, int sinks, float scale, uint16_t* out, int64_t ld_out, void* stream);

namespace {

struct SimpleArgs {
    PagedBatch b;
    PagedGroups gr;
    const uint16_t* q;
    int64_t ld_q;
    const void* kpages;
    const void* vpages;
    int64_t k_stride, v_stride;
    const uint8_t* scales;
    int64_t s_stride;
    int heads, kv_heads, g;
    int window, sinks;
    float scale;
    uint16_t* out;
    int64_t ld_out;
};

__device__ __forceinline__ float power_value(int byte) { return __builtin_bit_cast(float, (uint32_t)byte << 23); }

template <int D, bool E8>
__global__ void __launch_bounds__(256) attn_simple_kernel(SimpleArgs a) {
    constexpr int RW = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = __builtin_amdgcn_readfirstlane((int)(w / a.heads)), h = __builtin_amdgcn_readfirstlane((int)(w % a.heads));
    if (t >= a.b.T) return;
    const SeqRows sr = find_row(a.b, t, lane);
    if (sr.seq < 0) return;
    const int pos = sr.len - sr.n + (t - sr.first), kvh = h / a.g;
    int first;
    const int shared = find_group(a.b, a.gr, sr.seq, lane, &first);
    const uint16_t* q = a.q + (int64_t)t * a.ld_q + h * D;
    const float c = a.scale * 1.44269504088896340736f;
    float m = -3.0e38f, l = 0.0f, acc[RW] = {};
    const int S = 1 << a.b.shift;
    for (int pb = 0; sr.ok && pb <= pos; pb += 64) {
        const int p = pb + lane;
        int page = -1;
        if (p <= pos && (a.window <= 0 || p > pos - a.window || p < a.sinks)) page = page_of(a.b, p < shared ? first : sr.seq, p);
        float s = -__builtin_inff();
        const int64_t row = ((int64_t)kvh << a.b.shift) + (p & (S - 1));
        float vs = 1.0f;
        if (page >= 0) {
            s = 0.0f;
            for (int i = 0; i < D; ++i) {
                float k;
                if constexpr (E8)
                    k = __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(a.kpages)[page * a.k_stride + row * D + i], 0);
                else
                    k = bf16_bits_to_f32(static_cast<const uint16_t*>(a.kpages)[page * a.k_stride + row * D + i]);
                s = __builtin_fmaf(k, bf16_bits_to_f32(q[i]), s);
            }
            if constexpr (E8) {
                s *= power_value(a.scales[page * a.s_stride + 2 * row]);
                vs = power_value(a.scales[page * a.s_stride + 2 * row + 1]);
            }
        }
        float top = s;
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float mn = fmaxf(m, top * c), fac = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        float wt = page >= 0 ? __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -mn)) : 0.0f, sum = wt;
        for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
        l = l * fac + sum;
#pragma unroll
        for (int e = 0; e < RW; ++e) acc[e] *= fac;
        for (uint64_t left = __ballot(page >= 0); left; left &= left - 1) {
            const int j = __builtin_ctzll(left), pj = pb + j;
            const float wj = __shfl(wt, j) * __shfl(vs, j);
            const int64_t at = __shfl(page, j) * a.v_stride + (((int64_t)kvh << a.b.shift) + (pj & (S - 1))) * D + RW * lane;
#pragma unroll
            for (int e = 0; e < RW; ++e) {
                float v;
                if constexpr (E8)
                    v = __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(a.vpages)[at + e], 0);
                else
                    v = bf16_bits_to_f32(static_cast<const uint16_t*>(a.vpages)[at + e]);
                acc[e] = __builtin_fmaf(wj, v, acc[e]);
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < RW; ++e) a.out[(int64_t)t * a.ld_out + h * D + RW * lane + e] = bf16_rne_bits(acc[e] * inv);
}

int attention_simple(SimpleArgs a, bool e8, const int32_t* page_table, int64_t ld_table, int max_pages, const int32_t* q_start,
                     const int32_t* kv_len, int B, int T, int pages, int page_size, int max_q, int D, void* stream) {
    if (int rc = paged_batch(page_table, ld_table, max_pages, q_start, kv_len, B, T, pages, page_size, &a.b)) return rc;
    const int heads = a.heads, kv_heads = a.kv_heads;
    if (!a.kpages || !a.vpages || (T > 0 && (!a.q || !a.out))) return fail(ALV_ERR_ARG, "null pointer");
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || (D != 64 && D != 128 && D != 256 && D != 512) || a.window < 0 ||
        a.sinks < 0 || max_q < 0 || a.ld_q < (int64_t)heads * D || a.ld_out < (int64_t)heads * D)
        return fail(ALV_ERR_ARG, "bad attention shape heads=%d kv_heads=%d D=%d window=%d sinks=%d ld_q=%lld ld_out=%lld "
                    "(D one of 64, 128, 256, 512)", heads, kv_heads, D, a.window, a.sinks, (long long)a.ld_q, (long long)a.ld_out);
    if (heads > kMaxHeads) return fail(ALV_ERR_RANGE, "%d heads (at most %d)", heads, kMaxHeads);
    if (!(a.scale >= 0.0f) || a.scale > 3e38f) return fail(ALV_ERR_ARG, "scale %g: finite and not negative", (double)a.scale);
    const int64_t page_values = (int64_t)kv_heads * page_size * D;
    if (a.k_stride < page_values || a.v_stride < page_values)
        return fail(ALV_ERR_ARG, "page strides %lld and %lld hold fewer than the page's %lld values", (long long)a.k_stride,
                    (long long)a.v_stride, (long long)page_values);
    if (e8 && a.s_stride < 2 * (int64_t)kv_heads * page_size)
        return fail(ALV_ERR_ARG, "scales %lld apart hold fewer than a page's %lld", (long long)a.s_stride, 2ll * kv_heads * page_size);
    const int per = e8 ? 16 : 8;  // values of 16 bytes
    if (reinterpret_cast<uintptr_t>(a.kpages) % 16 || reinterpret_cast<uintptr_t>(a.vpages) % 16 || a.k_stride % per ||
        a.v_stride % per || reinterpret_cast<uintptr_t>(a.q) % 16 || a.ld_q % 8 || reinterpret_cast<uintptr_t>(a.out) % 8 ||
        a.ld_out % 4)
        return fail(ALV_ERR_ALIGN, "q, kpages and vpages and their rows need 16-byte alignment, out and its rows 8-byte");
    if (e8 && (reinterpret_cast<uintptr_t>(a.scales) % 16 || a.s_stride % 16))
        return fail(ALV_ERR_ALIGN, "scales and their pages need 16-byte alignment");
    if (T == 0) return ALV_OK;
    a.g = heads / kv_heads;
    a.window = a.window < a.b.max_pos ? a.window : 0;
    if ((int64_t)T * heads > (int64_t)1 << 30)
        return fail(ALV_ERR_RANGE, "%d rows of %d heads in one call (at most 2^30 rows times heads)", T, heads);
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, dim3((uint32_t)(((int64_t)T * heads + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
        return hip_check(hipGetLastError(), "attn_simple_kernel launch");
    };
    switch (D) {
        case 64: return e8 ? go(attn_simple_kernel<64, true>) : go(attn_simple_kernel<64, false>);
        case 128: return e8 ? go(attn_simple_kernel<128, true>) : go(attn_simple_kernel<128, false>);
        case 256: return e8 ? go(attn_simple_kernel<256, true>) : go(attn_simple_kernel<256, false>);
        default: return e8 ? go(attn_simple_kernel<512, true>) : go(attn_simple_kernel<512, false>);
    }
}

}  // namespace

}  // namespace alv

using namespace alv;

extern "C" uint64_t alv_attention_paged8_workspace(int heads, int kv_heads, int D, int B, int T, int max_q) { return 0; }

extern "C" int alv_attention_paged8(const uint16_t* q, int64_t ld_q, const uint8_t* kpages, const uint8_t* vpages,
                                    int64_t k_stride, int64_t v_stride, const uint8_t* scales, int64_t s_stride, int pages,
                                    int page_size, const int32_t* page_table, int64_t ld_table, int max_pages,
                                    const int32_t* q_start, const int32_t* kv_len, int B, int T, int max_q, int heads,
                                    int kv_heads, int D, int window, int sinks, float scale, uint16_t* out, int64_t ld_out,
                                    void* workspace, uint64_t workspace_bytes, void* stream) {
    if (!scales) return fail(ALV_ERR_ARG, "null pointer");
    SimpleArgs a{};
    a.q = q, a.ld_q = ld_q, a.kpages = kpages, a.vpages = vpages, a.k_stride = k_stride, a.v_stride = v_stride;
    a.scales = scales, a.s_stride = s_stride, a.heads = heads, a.kv_heads = kv_heads, a.window = window, a.sinks = sinks;
    a.scale = scale, a.out = out, a.ld_out = ld_out;
    return attention_simple(a, true, page_table, ld_table, max_pages, q_start, kv_len, B, T, pages, page_size, max_q, D, stream);
}

int alv::shared8_simple(const uint16_t* q, int64_t ld_q, const void* kpages, const void* vpages, int64_t k_stride,
                        int64_t v_stride, const uint8_t* scales, int64_t s_stride, int pages, int page_size,
                        const int32_t* page_table, int64_t ld_table, int max_pages, const int32_t* q_start,
                        const int32_t* kv_len, int B, int T, int max_q, const int32_t* group_start,
                        const int32_t* shared_len, int groups, int heads, int kv_heads, int D, int window, int sinks,
                        float scale, uint16_t* out, int64_t ld_out, void* stream) {
    SimpleArgs a{};
    a.gr = PagedGroups{group_start, shared_len, groups};
    a.q = q, a.ld_q = ld_q, a.kpages = kpages, a.vpages = vpages, a.k_stride = k_stride, a.v_stride = v_stride;
    a.scales = scales, a.s_stride = s_stride, a.heads = heads, a.kv_heads = kv_heads, a.window = window, a.sinks = sinks;
    a.scale = scale, a.out = out, a.ld_out = ld_out;
    return attention_simple(a, true, page_table, ld_table, max_pages, q_start, kv_len, B, T, pages, page_size, max_q, D, stream);
}
