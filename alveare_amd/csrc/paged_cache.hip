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

// One workgroup per packed row (token). Eight lanes per 128 columns (per head of
// 64), so a wave takes 2 to 8 heads at once: that is the layout in which numpy's
// order of a row's sum of squares (row_norm.h: eight interleaved accumulators
// per 128 values) needs no step on fewer lanes. A lane loads and stores 16-byte
// octets; the float rows in LDS turn octets into accumulators' columns and bring
// a rotated pair's other half.
//
// What bounds it: one token, three dependent trips to memory (the sequence, its
// page and RoPE row, the stores), 5 us; many, the bytes. 16 + 2 x 8 heads of 256,
// 4939 tokens: 48 us, 3.4 TB/s (a wave per head and two-byte accesses: 101 us);
// 42 where the same rows come again and are partly in the last cache.
constexpr int kPostMaxWaves = 8;
constexpr int kLeafPad = 8;  // floats: leaves then start eight banks apart

template <int D>
struct PostGeom {
    static constexpr int Leaf = D < 128 ? D : 128, Leaves = D / Leaf;
    static constexpr int Lanes = 8 * Leaves;      // of a head
    static constexpr int Heads = 64 / Lanes;      // of a wave
    static constexpr int Oct = Leaf / 64;         // octets of a lane
    static constexpr int Row = Leaves * (Leaf + kLeafPad);  // floats of a head in LDS
    // Float of a head's row that holds column c.
    static __device__ __forceinline__ int at(int c) { return c + (c / Leaf) * kLeafPad; }
};

// WIDE: every row 16-byte aligned, a rotated half whole octets.
template <int D, bool WIDE>
__global__ void __launch_bounds__((64 * kPostMaxWaves), (WIDE ? 6 : 2)) qkv_post_paged_kernel(PostPagedArgs a) {
    using G = PostGeom<D>;
    __shared__ __align__(16) float rows[kPostMaxWaves][G::Heads * G::Row];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = blockDim.x >> 6;
    const int t = blockIdx.x;
    const int total = a.heads + 2 * a.kv_heads;
    const int hw = lane / G::Lanes, hl = lane % G::Lanes;  // head of the wave, lane of the head
    float* row = rows[wave] + hw * G::Row;
    const uint16_t* xt = a.qkv + (int64_t)t * a.ld_qkv;

    struct Head {
        int role, h;
        bool in;
        const uint16_t* x;
        const float* w;
    };
    auto head = [&](int r0) {
        Head d;
        const int r = r0 * G::Heads + hw;
        d.in = r < total;
        const int rc = d.in ? r : total - 1;
        d.role = rc < a.heads ? 0 : (rc < a.heads + a.kv_heads ? 1 : 2);
        d.h = d.role == 0 ? rc : (d.role == 1 ? rc - a.heads : rc - a.heads - a.kv_heads);
        d.x = xt + (d.role == 0 ? 0 : (d.role == 1 || a.v_off < 0 ? a.k_off : a.v_off)) + d.h * D;
        d.w = d.role == 0 ? a.q_w : (d.role == 1 ? a.k_w : nullptr);
        return d;
    };
    // Octet e of a lane: columns 8 (hl + Lanes e).
    auto load_x = [&](const Head& d, uint4 (&x)[G::Oct]) {
#pragma unroll
        for (int e = 0; e < G::Oct; ++e) {
            const uint16_t* p = d.x + 8 * (hl + G::Lanes * e);
            if constexpr (WIDE)
                x[e] = *reinterpret_cast<const uint4*>(p);
            else
                __builtin_memcpy(&x[e], p, sizeof(x[e]));
        }
    };
    Head d = head(wave);
    uint4 x[G::Oct];
    load_x(d, x);  // on its way while the sequence is looked up
    const SeqRows sr = find_row(a.b, t, lane);
    if (sr.seq < 0) return;
    const int pos = sr.len - sr.n + (t - sr.first);
    const bool ok = sr.ok && pos < a.rope_rows;
    const int page = ok ? page_of(a.b, sr.seq, pos) : -1;
    const int slot = pos & ((1 << a.b.shift) - 1);
    const uint16_t* rr = ok && a.rope ? a.rope + pos * a.rope_stride : nullptr;

    for (int r0 = wave; r0 * G::Heads < total; r0 += nw) {
        if (r0 != wave) {
            d = head(r0);
            load_x(d, x);
        }
        float f[G::Oct][8];
        const int norm = d.role == 0 ? a.norm_q : (d.role == 1 ? a.norm_k : a.norm_v);
#pragma unroll
        for (int e = 0; e < G::Oct; ++e) {
            unpack8(x[e], f[e]);
            float4* p = reinterpret_cast<float4*>(row + G::at(8 * (hl + G::Lanes * e)));
            p[0] = float4{f[e][0], f[e][1], f[e][2], f[e][3]};
            p[1] = float4{f[e][4], f[e][5], f[e][6], f[e][7]};
        }
        // Leaf hl / 8 by its eight lanes, then the leaves in the recursion's tree.
        float sum = leaf8_sq_n<G::Leaf / 8>(row + (hl >> 3) * (G::Leaf + kLeafPad), hl & 7);
        if (G::Leaves > 1) sum = add_rn(sum, dpp_f<0x140>(sum));
        if (G::Leaves > 2) sum = add_rn(sum, __shfl_xor(sum, 16));
        const float inv = __fdiv_rn(1.0f, sqrtf(add_rn(__fdiv_rn(sum, (float)D), a.eps)));
        const bool rot = d.role < 2 && rr;
#pragma unroll
        for (int e = 0; e < G::Oct; ++e) {
            const int c0 = 8 * (hl + G::Lanes * e);
            if (norm) {
                float w[8];
                load_w8(d.w, c0 / 8, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = mul_rn(f[e][i], inv);
                    f[e][i] = bf16r(d.w ? mul_rn(v, w[i]) : v);
                }
            }
            if (rr) {  // the whole wave: a head's rows hold what its pairs read
                float4* p = reinterpret_cast<float4*>(row + G::at(c0));
                p[0] = float4{f[e][0], f[e][1], f[e][2], f[e][3]};
                p[1] = float4{f[e][4], f[e][5], f[e][6], f[e][7]};
            }
        }
        uint16_t* dst = d.role == 0 ? a.q_out + (int64_t)t * a.ld_q + d.h * D
                                    : (d.role == 1 ? a.kpages + max(page, 0) * a.k_stride : a.vpages + max(page, 0) * a.v_stride) +
                                          (((int64_t)d.h << a.b.shift) + slot) * D;
        const bool put = d.in && (d.role == 0 || page >= 0);
#pragma unroll
        for (int e = 0; e < G::Oct; ++e) {
            const int c0 = 8 * (hl + G::Lanes * e);
            uint16_t out[8];
            if (rot && c0 < 2 * a.half) {
                // run_rope_cpu_gemma (model.py:549-575): y1 = x1 c - x2 s, y2 = x2 c + x1 s.
                if constexpr (WIDE) {
                    const bool low = c0 < a.half;
                    const int i0 = low ? c0 : c0 - a.half;
                    const float4* op = reinterpret_cast<const float4*>(row + G::at(low ? c0 + a.half : i0));
                    const float4 o0 = op[0], o1 = op[1];
                    const float o[8] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w};
                    float cr[8], sn[8];
                    unpack8(*reinterpret_cast<const uint4*>(rr + a.cos_off + i0), cr);
                    unpack8(*reinterpret_cast<const uint4*>(rr + a.sin_off + i0), sn);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float xc = mul_rn(f[e][i], cr[i]), os = mul_rn(o[i], sn[i]);
                        out[i] = bf16_rne_bits(low ? sub_rn(xc, os) : add_rn(xc, os));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int c = c0 + i, k = c < a.half ? c : c - a.half;
                        float y = f[e][i];
                        if (c < 2 * a.half) {
                            const float xc = mul_rn(y, bf16_bits_to_f32(rr[a.cos_off + k]));
                            const float os = mul_rn(row[G::at(c < a.half ? c + a.half : k)], bf16_bits_to_f32(rr[a.sin_off + k]));
                            y = c < a.half ? sub_rn(xc, os) : add_rn(xc, os);
                        }
                        out[i] = bf16_rne_bits(y);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) out[i] = bf16_rne_bits(f[e][i]);
            }
            if (!ok)
#pragma unroll
                for (int i = 0; i < 8; ++i) out[i] = 0;
            if (!put) continue;
            const uint4 o8 = pack8(out);
            if constexpr (WIDE)
                *reinterpret_cast<uint4*>(dst + c0) = o8;
            else
                __builtin_memcpy(dst + c0, &o8, sizeof(o8));
        }
    }
}

// ---- alv_copy_pages ------------------------------------------------------------------

// A workgroup copies 16 KB of one page of one cache, four 16-byte pieces per
// thread; pointers and pairs come in the kernel's arguments, so a call is one
// launch and no transfer. Bound by memory: 450 pages of 64 KB in 32
// caches 370 us, 5.1 TB/s read and written; 6 pages of 64 KB in 24 caches, 4.4 us,
// by the launch (14 us with the checks of 24 tensors on the host).
constexpr int kCopyCaches = 128;  // per launch
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
    const int64_t qw = (int64_t)heads * D, kw = (int64_t)kv_heads * D;
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || (D != 64 && D != 128 && D != 256 && D != 512) || k_off < qw ||
        (v_off >= 0 && v_off < k_off + kw) || ld_qkv < (v_off < 0 ? k_off : v_off) + kw || ld_q < qw)
        return fail(ALV_ERR_ARG, "bad qkv layout heads=%d kv_heads=%d D=%d k_off=%d v_off=%d (D one of 64, 128, 256, 512)",
                    heads, kv_heads, D, k_off, v_off);
    if (heads > kMaxHeads) return fail(ALV_ERR_RANGE, "%d heads (at most %d)", heads, kMaxHeads);
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
    auto rows16 = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
    const bool wide = rows16(qkv, ld_qkv) && rows16(q_out, ld_q) && rows16(kpages, k_stride) && rows16(vpages, v_stride) &&
             k_off % 8 == 0 && (v_off < 0 || v_off % 8 == 0) &&
                      (!rope || (rows16(rope, rope_stride) && cos_off % 8 == 0 && sin_off % 8 == 0 && half % 8 == 0));
    if (reinterpret_cast<uintptr_t>(qkv) % 2 || reinterpret_cast<uintptr_t>(q_out) % 2 || reinterpret_cast<uintptr_t>(rope) % 2 ||
        reinterpret_cast<uintptr_t>(kpages) % 2 || reinterpret_cast<uintptr_t>(vpages) % 2 ||
        reinterpret_cast<uintptr_t>(q_w) % 16 || reinterpret_cast<uintptr_t>(k_w) % 16)
        return fail(ALV_ERR_ALIGN, "q_w and k_w need 16-byte alignment, the bf16 arrays 2-byte");
    const int per_wave = D <= 128 ? 8 : 1024 / D;  // heads
    const int threads = 64 * std::min(kPostMaxWaves, (heads + 2 * kv_heads + per_wave - 1) / per_wave);
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, dim3(T), dim3(threads), 0, (hipStream_t)stream, a);
        return hip_check(hipGetLastError(), "qkv_post_paged_kernel launch");
    };
    switch (D) {
        case 64: return wide ? go(qkv_post_paged_kernel<64, true>) : go(qkv_post_paged_kernel<64, false>);
        case 128: return wide ? go(qkv_post_paged_kernel<128, true>) : go(qkv_post_paged_kernel<128, false>);
        case 256: return wide ? go(qkv_post_paged_kernel<256, true>) : go(qkv_post_paged_kernel<256, false>);
        default: return wide ? go(qkv_post_paged_kernel<512, true>) : go(qkv_post_paged_kernel<512, false>);
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
