// The paged KV cache's own kernels on gfx950.
//
//   alv_qkv_post_paged  per-head q/k/v norms, RoPE of q and k, insert of k and
//                       v into their pages, for every new token of a batch
//                       (alv_qkv_post's arithmetic, bit for bit)
//   alv_qkv_post_paged8 the same into 8-bit pages
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
    void* kpages;  // bf16, or e4m3 codes
    void* vpages;
    int64_t k_stride, v_stride;
    uint8_t* scales;  // of codes
    int64_t s_stride;
};

// One workgroup per packed row (token). Eight lanes per 128 columns (per head of
// 64), so a wave takes 2 to 8 heads at once: that is the layout in which numpy's
// order of a row's sum of squares (row_norm.h: eight interleaved accumulators
// per 128 values) needs no step on fewer lanes. A lane loads and stores 16-byte
// octets; the float rows in LDS turn octets into accumulators' columns and bring
// a rotated pair's other half.
//
// What bounds it: one token, three dependent trips to memory (the sequence, its
// page and RoPE row, the stores), 5 us; many, those trips again, six waves per SIMD
// at a time (more would spill), and the arithmetic between them, by numpy's order and
// two roundings some 30 instructions a value (8-bit pages: the vector ALUs are busy 73 %
// of the time). 16 + 2 x 8 heads of 256, 4939 tokens: 43.5 us, 3.8 TB/s, into bf16 pages
// and 43.4, 3.3 TB/s, into 8-bit ones (rounding and coding value by value 47.6 and 49.3; a
// wave per head and two-byte accesses: 101).
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

// ---- 8-bit pages ---------------------------------------------------------------------
//
// A head's power of two is the smallest that brings its largest finite magnitude
// to 448 = 1.75 * 2^8 (e4m3's largest) or less. A power of two costs e4m3 nothing
// against a finer scale but the place of its smallest values (codes below 2^-6 are
// 2^-14.8 of the largest at most), products with it are exact, and it is one byte.
// Codes are rounded to nearest even, half a step: max(2^-4 of the value, 2^-10 of the
// power); what is not finite becomes NaN.

// The biased exponent, 1 .. 247, from the largest finite magnitude's bf16 bits.
__device__ __forceinline__ int power_of(int bits) {
    return max(1, (bits >> 7) - 8 + ((bits & 0x7F) > 0x60 ? 1 : 0));
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
constexpr int kInfBits = 0x7F80;

// The larger of `top` and the octet's magnitudes by their bits; those of what is not
// finite, from kInfBits on, left out if FINITE.
template <bool FINITE>
__device__ __forceinline__ u16x2 larger_magnitude(u16x2 top, const uint32_t (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u16x2 m = __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu);
        if constexpr (FINITE) m = u16x2{m.x < kInfBits ? m.x : (uint16_t)0, m.y < kInfBits ? m.y : (uint16_t)0};
        top = __builtin_elementwise_max(top, m);
    }
    return top;
}

// Eight bf16 values as codes. (v_cvt_scalef32_pk_fp8_bf16 divides by the power and rounds to
// nearest even; infinities, like NaN, give NaN. Against v_cvt_pk_fp8_f32 of each product: the
// same codes for every bf16 value and power, a third of the instructions.)
__device__ __forceinline__ uint2 encode8(const uint32_t (&w)[4], int power) {
    const float scale = __builtin_bit_cast(float, (uint32_t)power << 23);
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        s16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(s16x2{}, __builtin_bit_cast(bf16x2, w[2 * i]), scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, w[2 * i + 1]), scale, true);
        c[i] = __builtin_bit_cast(uint32_t, r);
    }
    return uint2{c[0], c[1]};
}

// ---- both kinds ------------------------------------------------------------------------

// bf16_rne_bits of eight values, in pairs; NaN, which the conversion passes on, is looked
// for once in all eight.
__device__ __forceinline__ void round8(const float (&f)[8], uint32_t (&w)[4]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{f[2 * i], f[2 * i + 1]}), bf16x2));
        nan |= __builtin_isunordered(f[2 * i], f[2 * i + 1]);
    }
    if (nan)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bf16_rne_bits(f[2 * i]) | ((uint32_t)bf16_rne_bits(f[2 * i + 1]) << 16);
}

// WIDE: every row 16-byte aligned (8-bit pages: 8), a rotated half whole octets.
// E8: 8-bit pages.
template <int D, bool WIDE, bool E8>
__global__ void __launch_bounds__((64 * kPostMaxWaves), (WIDE ? 6 : 2)) qkv_post_paged_kernel(PostPagedArgs a) {
    using G = PostGeom<D>;
    __shared__ __align__(16) float rows[kPostMaxWaves][G::Heads * G::Row];
    __shared__ __align__(16) uint16_t angles[WIDE ? kPostMaxWaves : 1][WIDE ? D : 8];  // a wave's cosines, its sines
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
    // The row's angles, four of each per lane, on their way beside the page's number.
    [[maybe_unused]] uint2 cosines{}, sines{};
    if constexpr (WIDE)
        if (rr && 4 * lane < a.half) {
            cosines = *reinterpret_cast<const uint2*>(rr + a.cos_off + 4 * lane);
            sines = *reinterpret_cast<const uint2*>(rr + a.sin_off + 4 * lane);
        }

    for (int r0 = wave; r0 * G::Heads < total; r0 += nw) {
        if (r0 != wave) {
            d = head(r0);
            load_x(d, x);
        } else if (WIDE && 4 * lane < a.half && rr) {
            *reinterpret_cast<uint2*>(&angles[wave][4 * lane]) = cosines;
            *reinterpret_cast<uint2*>(&angles[wave][D / 2 + 4 * lane]) = sines;
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
        const float inv = __fdiv_rn(1.0f, sqrtf(add_rn(mul_rn(sum, 1.0f / D), a.eps)));  // (D: a power of two)
        const bool rot = d.role < 2 && rr;
#pragma unroll
        for (int e = 0; e < G::Oct; ++e) {
            const int c0 = 8 * (hl + G::Lanes * e);
            if (norm) {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[e][i] = mul_rn(f[e][i], inv);
                if (d.w) {
                    const float4* w = reinterpret_cast<const float4*>(d.w + c0);
                    const float4 w0 = w[0], w1 = w[1];
                    f[e][0] = mul_rn(f[e][0], w0.x), f[e][1] = mul_rn(f[e][1], w0.y);
                    f[e][2] = mul_rn(f[e][2], w0.z), f[e][3] = mul_rn(f[e][3], w0.w);
                    f[e][4] = mul_rn(f[e][4], w1.x), f[e][5] = mul_rn(f[e][5], w1.y);
                    f[e][6] = mul_rn(f[e][6], w1.z), f[e][7] = mul_rn(f[e][7], w1.w);
                }
                uint32_t r[4];
                round8(f[e], r);
                unpack8(uint4{r[0], r[1], r[2], r[3]}, f[e]);
            }
            if (rr) {  // the whole wave: a head's rows hold what its pairs read
                float4* p = reinterpret_cast<float4*>(row + G::at(c0));
                p[0] = float4{f[e][0], f[e][1], f[e][2], f[e][3]};
                p[1] = float4{f[e][4], f[e][5], f[e][6], f[e][7]};
            }
        }
        auto rotated = [&](int e, uint32_t (&out)[4]) __attribute__((always_inline)) {
            const int c0 = 8 * (hl + G::Lanes * e);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = f[e][i];
            if (rot && c0 < 2 * a.half) {
                // run_rope_cpu_gemma (model.py:549-575): y1 = x1 c - x2 s, y2 = x2 c + x1 s.
                if constexpr (WIDE) {
                    const bool low = c0 < a.half;
                    const int i0 = low ? c0 : c0 - a.half;
                    const uint32_t sign = low ? 0x80008000u : 0u;  // (x1 c - x2 s = x1 c + x2 (-s), bit for bit)
                    const float4* op = reinterpret_cast<const float4*>(row + G::at(low ? c0 + a.half : i0));
                    const float4 o0 = op[0], o1 = op[1];
                    const float o[8] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w};
                    float cr[8], sn[8];
                    unpack8(*reinterpret_cast<const uint4*>(&angles[wave][i0]), cr);
                    const uint4 s8 = *reinterpret_cast<const uint4*>(&angles[wave][D / 2 + i0]);
                    unpack8(uint4{s8.x ^ sign, s8.y ^ sign, s8.z ^ sign, s8.w ^ sign}, sn);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = add_rn(mul_rn(y[i], cr[i]), mul_rn(o[i], sn[i]));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int c = c0 + i, k = c < a.half ? c : c - a.half;
                        if (c < 2 * a.half) {
                            const float xc = mul_rn(y[i], bf16_bits_to_f32(rr[a.cos_off + k]));
                            const float os = mul_rn(row[G::at(c < a.half ? c + a.half : k)], bf16_bits_to_f32(rr[a.sin_off + k]));
                            y[i] = c < a.half ? sub_rn(xc, os) : add_rn(xc, os);
                        }
                    }
                }
            }
            round8(y, out);
            if (!ok)
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = 0;
        };
        const bool put = d.in && (d.role == 0 || page >= 0);
        const int64_t at = (((int64_t)d.h << a.b.shift) + slot) * D;  // in its page
        if constexpr (E8) {
            uint32_t out[G::Oct][4];
            u16x2 top2{};
#pragma unroll
            for (int e = 0; e < G::Oct; ++e) {
                rotated(e, out[e]);
                top2 = larger_magnitude<false>(top2, out[e]);
            }
            auto over_head = [&](u16x2 m) __attribute__((always_inline)) {
                int top = max(m.x, m.y);
#pragma unroll
                for (int k = 1; k < G::Lanes; k <<= 1) top = max(top, __shfl_xor(top, k));
                return top;
            };
            int top = over_head(top2);
            if (__any(top >= kInfBits)) {  // (of any head of the wave: its lanes stay together)
                top2 = u16x2{};
#pragma unroll
                for (int e = 0; e < G::Oct; ++e) top2 = larger_magnitude<true>(top2, out[e]);
                top = over_head(top2);
            }
            if (!put) continue;
            const int power = power_of(top);
#pragma unroll
            for (int e = 0; e < G::Oct; ++e) {
                const int c0 = 8 * (hl + G::Lanes * e);
                if (d.role == 0) {
                    uint16_t* dst = a.q_out + (int64_t)t * a.ld_q + d.h * D + c0;
                    if constexpr (WIDE)
                        *reinterpret_cast<uint4*>(dst) = uint4{out[e][0], out[e][1], out[e][2], out[e][3]};
                    else
                        __builtin_memcpy(dst, out[e], sizeof(out[e]));
                } else {
                    uint8_t* dst = d.role == 1 ? static_cast<uint8_t*>(a.kpages) + page * a.k_stride
                                               : static_cast<uint8_t*>(a.vpages) + page * a.v_stride;
                    const uint2 o8 = encode8(out[e], power);
                    if constexpr (WIDE)
                        *reinterpret_cast<uint2*>(dst + at + c0) = o8;
                    else
                        __builtin_memcpy(dst + at + c0, &o8, sizeof(o8));
                }
            }
            if (d.role && hl == 0)
                a.scales[page * a.s_stride + 2 * (((int64_t)d.h << a.b.shift) + slot) + d.role - 1] = (uint8_t)power;
        } else {
            uint16_t* dst = d.role == 0 ? a.q_out + (int64_t)t * a.ld_q + d.h * D
                                        : at + (d.role == 1 ? static_cast<uint16_t*>(a.kpages) + max(page, 0) * a.k_stride
                                                            : static_cast<uint16_t*>(a.vpages) + max(page, 0) * a.v_stride);
#pragma unroll
            for (int e = 0; e < G::Oct; ++e) {
                uint32_t out[4];
                rotated(e, out);
                if (!put) continue;
                const int c0 = 8 * (hl + G::Lanes * e);
                if constexpr (WIDE)
                    *reinterpret_cast<uint4*>(dst + c0) = uint4{out[0], out[1], out[2], out[3]};
                else
                    __builtin_memcpy(dst + c0, out, sizeof(out));
            }
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

namespace alv {
namespace {

// Both kinds of pages: 8-bit ones where scales are given (E8).
template <bool E8>
int post_paged(PostPagedArgs a, int64_t ld_table, int max_pages, const int32_t* page_table, const int32_t* q_start,
               const int32_t* kv_len, int B, int T, int pages, int page_size, int D, int rope_rows, void* stream) {
    if (int rc = paged_batch(page_table, ld_table, max_pages, q_start, kv_len, B, T, pages, page_size, &a.b)) return rc;
    if (!a.kpages || !a.vpages || (E8 && !a.scales) || (T > 0 && (!a.qkv || !a.q_out))) return fail(ALV_ERR_ARG, "null pointer");
    const int heads = a.heads, kv_heads = a.kv_heads, k_off = a.k_off, v_off = a.v_off;
    const int64_t qw = (int64_t)heads * D, kw = (int64_t)kv_heads * D;
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || (D != 64 && D != 128 && D != 256 && D != 512) || k_off < qw ||
        (v_off >= 0 && v_off < k_off + kw) || a.ld_qkv < (v_off < 0 ? k_off : v_off) + kw || a.ld_q < qw)
        return fail(ALV_ERR_ARG, "bad qkv layout heads=%d kv_heads=%d D=%d k_off=%d v_off=%d (D one of 64, 128, 256, 512)",
                    heads, kv_heads, D, k_off, v_off);
    if (heads > kMaxHeads) return fail(ALV_ERR_RANGE, "%d heads (at most %d)", heads, kMaxHeads);
    const int64_t page_values = (int64_t)kv_heads * page_size * D;
    if (a.k_stride < page_values || a.v_stride < page_values)
        return fail(ALV_ERR_ARG, "page strides %lld and %lld hold fewer than the page's %lld values", (long long)a.k_stride,
                    (long long)a.v_stride, (long long)page_values);
    if (E8 && a.s_stride < 2 * (int64_t)kv_heads * page_size)
        return fail(ALV_ERR_ARG, "scales %lld apart hold fewer than a page's %lld", (long long)a.s_stride,
                    2ll * kv_heads * page_size);
    if (a.rope && (a.half < 1 || 2 * (int64_t)a.half > D || rope_rows < 1 || a.rope_stride < 1 || a.cos_off < 0 ||
                   a.sin_off < 0 || a.cos_off + (int64_t)a.half > a.rope_stride || a.sin_off + (int64_t)a.half > a.rope_stride))
        return fail(ALV_ERR_ARG, "bad rope table layout rows=%d stride=%lld cos_off=%d sin_off=%d half=%d for D=%d",
                    rope_rows, (long long)a.rope_stride, a.cos_off, a.sin_off, a.half, D);
    if (T == 0) return ALV_OK;
    a.rope_rows = a.rope ? rope_rows : INT_MAX;
    auto rows16 = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
    auto rows8 = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 8 == 0 && ld % 8 == 0; };
    const bool wide = rows16(a.qkv, a.ld_qkv) && rows16(a.q_out, a.ld_q) &&
                      (E8 ? rows8(a.kpages, a.k_stride) && rows8(a.vpages, a.v_stride)
                          : rows16(a.kpages, a.k_stride) && rows16(a.vpages, a.v_stride)) &&
                      k_off % 8 == 0 && (v_off < 0 || v_off % 8 == 0) &&
                      (!a.rope || (rows16(a.rope, a.rope_stride) && a.cos_off % 8 == 0 && a.sin_off % 8 == 0 && a.half % 8 == 0));
    if (reinterpret_cast<uintptr_t>(a.qkv) % 2 || reinterpret_cast<uintptr_t>(a.q_out) % 2 || reinterpret_cast<uintptr_t>(a.rope) % 2 ||
        (!E8 && (reinterpret_cast<uintptr_t>(a.kpages) % 2 || reinterpret_cast<uintptr_t>(a.vpages) % 2)) ||
        reinterpret_cast<uintptr_t>(a.q_w) % 16 || reinterpret_cast<uintptr_t>(a.k_w) % 16)
        return fail(ALV_ERR_ALIGN, "q_w and k_w need 16-byte alignment, the bf16 arrays 2-byte");
    const int per_wave = D <= 128 ? 8 : 1024 / D;  // heads
    const int threads = 64 * std::min(kPostMaxWaves, (heads + 2 * kv_heads + per_wave - 1) / per_wave);
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, dim3(T), dim3(threads), 0, (hipStream_t)stream, a);
        return hip_check(hipGetLastError(), "qkv_post_paged_kernel launch");
    };
    switch (D) {
        case 64: return wide ? go(qkv_post_paged_kernel<64, true, E8>) : go(qkv_post_paged_kernel<64, false, E8>);
        case 128: return wide ? go(qkv_post_paged_kernel<128, true, E8>) : go(qkv_post_paged_kernel<128, false, E8>);
        case 256: return wide ? go(qkv_post_paged_kernel<256, true, E8>) : go(qkv_post_paged_kernel<256, false, E8>);
        default: return wide ? go(qkv_post_paged_kernel<512, true, E8>) : go(qkv_post_paged_kernel<512, false, E8>);
    }
}

}  // namespace
}  // namespace alv

extern "C" int alv_qkv_post_paged(const uint16_t* qkv, int64_t ld_qkv, int k_off, int v_off, int heads, int kv_heads,
                                  int D, const float* q_w, const float* k_w, int norm_q, int norm_k, int norm_v,
                                  float eps, const uint16_t* rope, int rope_rows, int64_t rope_stride, int cos_off,
                                  int sin_off, int half, const int32_t* page_table, int64_t ld_table, int max_pages,
                                  const int32_t* q_start, const int32_t* kv_len, int B, int T, int pages,
                                  int page_size, uint16_t* kpages, uint16_t* vpages, int64_t k_stride,
                                  int64_t v_stride, uint16_t* q_out, int64_t ld_q, void* stream) {
    PostPagedArgs a{};
    a.qkv = qkv, a.ld_qkv = ld_qkv, a.k_off = k_off, a.v_off = v_off, a.heads = heads, a.kv_heads = kv_heads;
    a.q_w = q_w, a.k_w = k_w, a.norm_q = norm_q, a.norm_k = norm_k, a.norm_v = norm_v, a.eps = eps;
    a.rope = rope, a.rope_stride = rope_stride, a.cos_off = cos_off, a.sin_off = sin_off, a.half = half;
    a.q_out = q_out, a.ld_q = ld_q, a.kpages = kpages, a.vpages = vpages, a.k_stride = k_stride, a.v_stride = v_stride;
    return post_paged<false>(a, ld_table, max_pages, page_table, q_start, kv_len, B, T, pages, page_size, D, rope_rows,
                             stream);
}

extern "C" int alv_qkv_post_paged8(const uint16_t* qkv, int64_t ld_qkv, int k_off, int v_off, int heads, int kv_heads,
                                   int D, const float* q_w, const float* k_w, int norm_q, int norm_k, int norm_v,
                                   float eps, const uint16_t* rope, int rope_rows, int64_t rope_stride, int cos_off,
                                   int sin_off, int half, const int32_t* page_table, int64_t ld_table, int max_pages,
                                   const int32_t* q_start, const int32_t* kv_len, int B, int T, int pages,
                                   int page_size, uint8_t* kpages, uint8_t* vpages, int64_t k_stride, int64_t v_stride,
                                   uint8_t* scales, int64_t s_stride, uint16_t* q_out, int64_t ld_q, void* stream) {
    PostPagedArgs a{};
    a.qkv = qkv, a.ld_qkv = ld_qkv, a.k_off = k_off, a.v_off = v_off, a.heads = heads, a.kv_heads = kv_heads;
    a.q_w = q_w, a.k_w = k_w, a.norm_q = norm_q, a.norm_k = norm_k, a.norm_v = norm_v, a.eps = eps;
    a.rope = rope, a.rope_stride = rope_stride, a.cos_off = cos_off, a.sin_off = sin_off, a.half = half;
    a.q_out = q_out, a.ld_q = ld_q, a.kpages = kpages, a.vpages = vpages, a.k_stride = k_stride, a.v_stride = v_stride;
    a.scales = scales, a.s_stride = s_stride;
    return post_paged<true>(a, ld_table, max_pages, page_table, q_start, kv_len, B, T, pages, page_size, D, rope_rows,
                            stream);
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
