// The paged KV cache's own kernels on gfx950.
//
//   alv_qkv_post_paged  per-head q/k/v norms, RoPE of q and k, insert of k and
//                       v into their pages, for every new token of a batch
//                       (alv_qkv_post's arithmetic, bit for bit)
//   alv_copy_pages      pages copied within each of many caches
#include <limits.h>

#include <algorithm>
#include <new>
#include <vector>

#include "paged.h"
#include "q4_device.h"
#include "row_norm.h"

#pragma clang fp contract(off)

namespace alv {

namespace {

// ---- alv_qkv_post_paged ------------------------------------------------------------

struct PostPagedArgs {
    PagedBatch b;
    const uint16_t* qkv;
    int64_t ld_qkv;
    int k_off, v_off, heads, kv_heads;
    const float* q_w;
    const float* k_w;
    int norm_q, norm_k, norm_v;
    float eps;
    const uint16_t* rope;
    int64_t rope_stride;
    int rope_rows;  // INT_MAX without a table
    int cos_off, sin_off, half;
    uint16_t* q_out;
    int64_t ld_q;
    uint16_t* kpages;
    uint16_t* vpages;
    int64_t k_stride, v_stride;
};

constexpr int kPostMaxWaves = 8;

// One workgroup per packed row (token); a wave takes one head row at a time.
template <int D>
__global__ void __launch_bounds__(64 * kPostMaxWaves) qkv_post_paged_kernel(PostPagedArgs a) {
    constexpr int RW = D / 64;
    __shared__ __align__(16) float rows[kPostMaxWaves][D];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = blockDim.x >> 6;
    const int t = blockIdx.x;
    const SeqRows sr = find_row(a.b, t, lane);
    if (sr.seq < 0) return;
    const int pos = sr.len - sr.n + (t - sr.first);
    const bool ok = sr.ok && pos < a.rope_rows;
    const int page = ok ? page_of(a.b, sr.seq, pos) : -1;
    const int slot = pos & ((1 << a.b.shift) - 1);
    const int total = a.heads + 2 * a.kv_heads;
    float* row = rows[wave];
    for (int r = wave; r < total; r += nw) {
        const int role = r < a.heads ? 0 : (r < a.heads + a.kv_heads ? 1 : 2);
        const int h = role == 0 ? r : (role == 1 ? r - a.heads : r - a.heads - a.kv_heads);
        if (role && page < 0) continue;
        uint16_t* dst = role == 0 ? a.q_out + (int64_t)t * a.ld_q + h * D
                                  : (role == 1 ? a.kpages + page * a.k_stride : a.vpages + page * a.v_stride) +
                                        (((int64_t)h << a.b.shift) + slot) * D;
        if (!ok) {
            for (int e = 0; e < RW; ++e) dst[RW * lane + e] = 0;
            continue;
        }
        const int src = role == 0 ? h * D : (role == 1 || a.v_off < 0 ? a.k_off + h * D : a.v_off + h * D);
        const uint16_t* x = a.qkv + (int64_t)t * a.ld_qkv + src;
        const int norm = role == 0 ? a.norm_q : (role == 1 ? a.norm_k : a.norm_v);
        const float* w = role == 0 ? a.q_w : (role == 1 ? a.k_w : nullptr);
        for (int e = 0; e < RW; ++e) row[RW * lane + e] = bf16_bits_to_f32(x[RW * lane + e]);
        if (norm) {
            const float inv = rms_inv_wave(row, D, a.eps, lane);
            for (int e = 0; e < RW; ++e) {
                const int d = RW * lane + e;
                const float v = mul_rn(row[d], inv);
                row[d] = bf16r(w ? mul_rn(v, w[d]) : v);
            }
        }
        const uint16_t* rr = role < 2 && a.rope ? a.rope + pos * a.rope_stride : nullptr;
        for (int e = 0; e < RW; ++e) {
            const int d = RW * lane + e;
            float y = row[d];
            if (rr && d < 2 * a.half) {
                const int i = d < a.half ? d : d - a.half;
                const float c = bf16_bits_to_f32(rr[a.cos_off + i]), s = bf16_bits_to_f32(rr[a.sin_off + i]);
                y = d < a.half ? sub_rn(mul_rn(row[i], c), mul_rn(row[i + a.half], s))
                               : add_rn(mul_rn(row[d], c), mul_rn(row[i], s));
            }
            dst[d] = bf16_rne_bits(y);
        }
    }
}

// ---- alv_copy_pages ------------------------------------------------------------------

constexpr int kCopyCaches = 128;  // per launch, in the kernel's arguments
constexpr int kCopyPairs = 256;
constexpr int kCopyChunk = 16384;  // bytes per workgroup

struct CopyArgs {
    uint8_t* cache[kCopyCaches];
    int32_t src[kCopyPairs], dst[kCopyPairs];
    int64_t page_bytes, stride;
    int chunks, npairs;
};

__global__ void __launch_bounds__(256) copy_pages_kernel(CopyArgs a) {
    const int chunk = blockIdx.x % a.chunks, pair = blockIdx.x / a.chunks;
    uint8_t* base = a.cache[blockIdx.y];
    const int64_t off = (int64_t)chunk * kCopyChunk;
    const u32x4* s = reinterpret_cast<const u32x4*>(base + a.src[pair] * a.stride + off);
    u32x4* d = reinterpret_cast<u32x4*>(base + a.dst[pair] * a.stride + off);
    const int n = (int)(min(a.page_bytes - off, (int64_t)kCopyChunk) / 16);
    for (int i = threadIdx.x; i < n; i += 256) d[i] = s[i];
}

}  // namespace

}  // namespace alv

using namespace alv;

extern "C" int alv_qkv_post_paged(const uint16_t* qkv, int64_t ld_qkv, int k_off, int v_off, int heads, int kv_heads,
                                  int D, const float* q_w, const float* k_w, int norm_q, int norm_k, int norm_v,
                                  float eps, const uint16_t* rope, int rope_rows, int64_t rope_stride, int cos_off,
                                  int sin_off, int half, const int32_t* page_table, int64_t ld_table, int max_pages,
                                  const int32_t* q_start, const int32_t* kv_len, int B, int T, int pages,
                                  int page_size, uint16_t* kpages, uint16_t* vpages, int64_t k_stride,
                                  int64_t v_stride, uint16_t* q_out, int64_t ld_q, void* stream) {
    PostPagedArgs a{};
    if (int rc = paged_batch(page_table, ld_table, max_pages, q_start, kv_len, B, T, pages, page_size, &a.b)) return rc;
    if (!kpages || !vpages || (T > 0 && (!qkv || !q_out))) return fail(ALV_ERR_ARG, "null pointer");
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || (D != 64 && D != 128 && D != 256 && D != 512) ||
        k_off < heads * D || (v_off >= 0 && v_off < k_off + kv_heads * D) ||
        ld_qkv < (v_off < 0 ? k_off : v_off) + kv_heads * D || ld_q < heads * D)
        return fail(ALV_ERR_ARG, "bad qkv layout heads=%d kv_heads=%d D=%d k_off=%d v_off=%d (D one of 64, 128, 256, 512)",
                    heads, kv_heads, D, k_off, v_off);
    const int64_t page_values = (int64_t)kv_heads * page_size * D;
    if (k_stride < page_values || v_stride < page_values)
        return fail(ALV_ERR_ARG, "page strides %lld and %lld hold fewer than the page's %lld values", (long long)k_stride,
                    (long long)v_stride, (long long)page_values);
    if (rope && (half < 1 || 2 * half > D || rope_rows < 1 || rope_stride < 1 || cos_off < 0 || sin_off < 0 ||
                 cos_off + half > rope_stride || sin_off + half > rope_stride))
        return fail(ALV_ERR_ARG, "bad rope table layout rows=%d stride=%lld cos_off=%d sin_off=%d half=%d for D=%d",
                    rope_rows, (long long)rope_stride, cos_off, sin_off, half, D);
    if (T == 0) return ALV_OK;
    a.qkv = qkv, a.ld_qkv = ld_qkv, a.k_off = k_off, a.v_off = v_off, a.heads = heads, a.kv_heads = kv_heads;
    a.q_w = q_w, a.k_w = k_w, a.norm_q = norm_q, a.norm_k = norm_k, a.norm_v = norm_v, a.eps = eps;
    a.rope = rope, a.rope_stride = rope_stride, a.cos_off = cos_off, a.sin_off = sin_off, a.half = half;
    a.q_out = q_out, a.ld_q = ld_q, a.kpages = kpages, a.vpages = vpages, a.k_stride = k_stride, a.v_stride = v_stride;
    a.rope_rows = rope ? rope_rows : INT_MAX;
    const int threads = 64 * std::min(kPostMaxWaves, heads + 2 * kv_heads);
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, dim3(T), dim3(threads), 0, (hipStream_t)stream, a);
        return hip_check(hipGetLastError(), "qkv_post_paged_kernel launch");
    };
    switch (D) {
        case 64: return go(qkv_post_paged_kernel<64>);
        case 128: return go(qkv_post_paged_kernel<128>);
        case 256: return go(qkv_post_paged_kernel<256>);
        default: return go(qkv_post_paged_kernel<512>);
    }
}

extern "C" int alv_copy_pages(void* const* caches, int ncaches, int64_t page_bytes, int64_t stride_bytes, int pages,
                              const int32_t* src, const int32_t* dst, int npairs, void* stream) {
    if (!caches || (npairs > 0 && (!src || !dst))) return fail(ALV_ERR_ARG, "null pointer");
    if (ncaches < 1 || npairs < 0 || pages < 1 || page_bytes < 16 || page_bytes % 16 || stride_bytes < page_bytes ||
        stride_bytes % 16)
        return fail(ALV_ERR_ARG, "bad page copy: %d caches of %d pages of %lld bytes, %lld apart, %d pairs", ncaches, pages,
                    (long long)page_bytes, (long long)stride_bytes, npairs);
    if (page_bytes > (int64_t)1 << 28) return fail(ALV_ERR_RANGE, "pages of %lld bytes", (long long)page_bytes);
    for (int i = 0; i < ncaches; ++i) {
        if (!caches[i]) return fail(ALV_ERR_ARG, "null pointer");
        if (reinterpret_cast<uintptr_t>(caches[i]) % 16) return fail(ALV_ERR_ALIGN, "caches need 16-byte alignment");
    }
    for (int i = 0; i < npairs; ++i)
        if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages)
            return fail(ALV_ERR_ARG, "pair %d copies page %d to %d of %d pages", i, src[i], dst[i], pages);
    // Every copy may run at the same time as every other: a destination is
    // written once and read by none.
    try {
        std::vector<int32_t> d(dst, dst + npairs), s(src, src + npairs);
        std::sort(d.begin(), d.end());
        std::sort(s.begin(), s.end());
        for (int i = 1; i < npairs; ++i)
            if (d[i] == d[i - 1]) return fail(ALV_ERR_ARG, "page %d is the destination of two copies", d[i]);
        for (int i = 0, j = 0; i < npairs && j < npairs;) {
            if (d[i] == s[j]) return fail(ALV_ERR_ARG, "page %d is both a source and a destination", d[i]);
            if (d[i] < s[j]) ++i; else ++j;
        }
    } catch (const std::bad_alloc&) {
        return fail(ALV_ERR_RANGE, "no host memory to check %d pairs", npairs);
    }
    const int chunks = (int)((page_bytes + kCopyChunk - 1) / kCopyChunk);
    for (int c0 = 0; c0 < ncaches; c0 += kCopyCaches)
        for (int p0 = 0; p0 < npairs; p0 += kCopyPairs) {
            CopyArgs a{};
            const int nc = std::min(ncaches - c0, kCopyCaches);
            a.npairs = std::min(npairs - p0, kCopyPairs);
            for (int i = 0; i < nc; ++i) a.cache[i] = static_cast<uint8_t*>(caches[c0 + i]);
            std::copy(src + p0, src + p0 + a.npairs, a.src);
            std::copy(dst + p0, dst + p0 + a.npairs, a.dst);
            a.page_bytes = page_bytes, a.stride = stride_bytes, a.chunks = chunks;
            hipLaunchKernelGGL(copy_pages_kernel, dim3(chunks * a.npairs, nc), dim3(256), 0, (hipStream_t)stream, a);
            if (int rc = hip_check(hipGetLastError(), "copy_pages_kernel launch")) return rc;
        }
    return ALV_OK;
}
