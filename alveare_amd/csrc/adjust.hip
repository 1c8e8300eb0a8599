// What is done to rows of logits between the head and the sampling: penalties for
// tokens that occurred, biases, and the tokens that are allowed.
//
//   x = l > 0 ? l / r : l * r      if the token occurred in the row's history
//   x -= f * c + p                 if it occurred c > 0 times in its generated part
//   x += sum of its biases, in the order of the list
//   x = -infinity                  if its bit is clear
//
// in float64 for the tokens that any of this touches (few), rounded once.
//
// A workgroup takes kRange tokens of one row: it counts the history's tokens among
// them in LDS (integers: their order does not show), notes which list entry is a
// token's first bias, and passes once over the logits, which are on their way
// meanwhile. In place, only what changes is read and written.
//
// Bound by memory where there are rows enough: 64 rows of 262144, 1 % allowed, in place
// 14.7 us, 4.7 TB/s of words and -infinities; 48 rows of 128256 with histories of up to
// 8000 tokens and 300 biases 16.3 us, 3.1 TB/s, by the 16 workgroups of a row that each
// read its whole history (smaller ranges read it more often, larger ones leave CUs idle).
// One row of 262144 with 1500 tokens: 7.3 us, three trips to memory one after the other.
#include <algorithm>

#include "q4_device.h"
#include "q4_host.h"

namespace alv {

namespace {

struct AdjustArgs {
    const float* logits;
    float* out;
    int64_t ld, ld_out;
    int V;
    const int32_t* tokens;
    int64_t ld_tokens;
    int L;
    const int32_t* n_tokens;
    const int32_t* n_prompt;
    const float* rep_dev;
    const float* freq_dev;
    const float* pres_dev;
    float rep, freq, pres;
    const int32_t* bias_tokens;
    const float* bias;
    int64_t ld_bias_tokens, ld_bias;
    int M;
    const uint32_t* allowed;
    int64_t ld_allowed;
};

constexpr int kThreads = 512;
constexpr int kGroups = 4;                        // of 4 tokens, per thread
constexpr int kRange = 4 * kGroups * kThreads;    // tokens of a workgroup

// What is known of a token: how often it was generated, whether it was in the
// prompt, whether it is on the list again, and in the upper bits `entries - i` of its
// first list entry i (0: none). While the upper bits are set the lower ones stay, so
// a maximum of whole words takes the first entry. 32 bits for histories and lists
// that fit, else 64.
template <class Word>
struct Fields;
template <>
struct Fields<uint32_t> {
    static constexpr int kCount = 17, kFirst = 19;
};
template <>
struct Fields<unsigned long long> {
    static constexpr int kCount = 31, kFirst = 33;
};
constexpr int kMostCount = (1 << 17) - 1, kMostEntries = (1 << 13) - 1;

// WIDE: rows 16-byte aligned. COPY: out is elsewhere.
template <class Word, bool WIDE, bool COPY>
__global__ void __launch_bounds__(kThreads) adjust_kernel(AdjustArgs a) {
    using F = Fields<Word>;
    constexpr Word kPrompt = (Word)1 << F::kCount, kTwice = 2 * kPrompt, kCountMask = kPrompt - 1, kLower = 4 * kPrompt - 1;
    extern __shared__ __align__(16) unsigned char smem[];
    Word* const what = reinterpret_cast<Word*>(smem);
    const int tid = threadIdx.x, b = blockIdx.y;
    const int64_t t0 = (int64_t)blockIdx.x * kRange;
    const int n = (int)min((int64_t)kRange, a.V - t0);
    const float* in = a.logits + b * a.ld + t0;
    float* out = a.out + b * a.ld_out + t0;
    const uint32_t* allowed = a.allowed ? a.allowed + b * a.ld_allowed + t0 / 32 : nullptr;
    float4 x[kGroups] = {};
    uint32_t keep[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int i = 4 * (tid + kThreads * g);
        keep[g] = 15;
        if (i < n) {
            if (COPY) {
                if (WIDE && i + 4 <= n) {
                    x[g] = *reinterpret_cast<const float4*>(in + i);
                } else {
                    x[g].x = in[i];
                    x[g].y = in[min(i + 1, n - 1)];
                    x[g].z = in[min(i + 2, n - 1)];
                    x[g].w = in[min(i + 3, n - 1)];
                }
            }
            if (allowed) keep[g] = allowed[i >> 5] >> (i & 31) & 15;
        }
    }
    const float r = a.rep_dev ? a.rep_dev[b] : a.rep, f = a.freq_dev ? a.freq_dev[b] : a.freq;
    const float p = a.pres_dev ? a.pres_dev[b] : a.pres;
    const bool history = a.L > 0 && (r != 1.0f || f != 0.0f || p != 0.0f);
    const bool known = history || a.M > 0;
    const int32_t* list = a.M > 0 ? a.bias_tokens + b * a.ld_bias_tokens : nullptr;
    const float* bias = a.M > 0 ? a.bias + b * a.ld_bias : nullptr;
    if (known) {
        for (int i = tid; i < (int)(kRange * sizeof(Word) / 16); i += kThreads) reinterpret_cast<uint4*>(smem)[i] = uint4{0, 0, 0, 0};
    }
    if (history) {
        const int32_t* row = a.tokens + b * a.ld_tokens;
        const int have = a.n_tokens ? max(0, min(a.n_tokens[b], a.L)) : a.L;
        const int prompt = a.n_prompt ? a.n_prompt[b] : 0;
        // 16-byte pieces from the first aligned token on, four of a thread on their way at once.
        const int lead = min(have, (int)(-(reinterpret_cast<uintptr_t>(row) >> 2) & 3)), pieces = (have - lead) >> 2;
        const int tail = lead + 4 * pieces;
        int single = -1;
        if (tid < lead) single = tid;
        if (tid >= 64 && tail + tid - 64 < have) single = tail + tid - 64;
        const int st = single >= 0 ? row[single] : -1;
        auto note = [&](int token, int i) __attribute__((always_inline)) {
            const int64_t at = token - t0;
            if (at >= 0 && at < n) {
                if (i < prompt)
                    atomicOr(&what[at], kPrompt);
                else
                    atomicAdd(&what[at], (Word)1);
            }
        };
        const int4* piece = reinterpret_cast<const int4*>(row + lead);
        int4 v[4];
        auto load = [&](int q0) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int q = q0 + tid + kThreads * u;
                v[u] = q < pieces ? piece[q] : int4{-1, -1, -1, -1};
            }
        };
        load(0);
        __syncthreads();
        for (int q0 = 0; q0 < pieces; q0 += 4 * kThreads) {
            if (q0) load(q0);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = lead + 4 * (q0 + tid + kThreads * u);
                note(v[u].x, i);
                note(v[u].y, i + 1);
                note(v[u].z, i + 2);
                note(v[u].w, i + 3);
            }
        }
        if (single >= 0) note(st, single);
    }
    if (a.M > 0) {
        __syncthreads();
        for (int i = tid; i < a.M; i += kThreads) {
            const int64_t at = list[i] - t0;
            if (at >= 0 && at < n) atomicMax(&what[at], (Word)(a.M - i) << F::kFirst | (what[at] & kLower));
        }
        __syncthreads();
        for (int i = tid; i < a.M; i += kThreads) {
            const int64_t at = list[i] - t0;
            if (at >= 0 && at < n && what[at] >> F::kFirst != (Word)(a.M - i)) atomicOr(&what[at], kTwice);
        }
    }
    if (known) __syncthreads();
    // The pass over the logits; what is known of a token, few of them, comes after.
    uint32_t left = 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int i = 4 * (tid + kThreads * g);
        if (i >= n) continue;
        const uint32_t k = keep[g];
        if (known) {
            Word w[4];
            __builtin_memcpy(w, __builtin_assume_aligned(what + i, 16), sizeof(w));
#pragma unroll
            for (int e = 0; e < 4; ++e) left |= (uint32_t)(w[e] != 0 && i + e < n) << (4 * g + e);
            left &= ~(15u << (4 * g)) | k << (4 * g);
        }
        if (!COPY && k == 15) continue;
        const float gone = -__builtin_inff();
        if (WIDE && i + 4 <= n && (COPY || k == 0)) {
            float4 v;
            v.x = k & 1 ? x[g].x : gone;
            v.y = k & 2 ? x[g].y : gone;
            v.z = k & 4 ? x[g].z : gone;
            v.w = k & 8 ? x[g].w : gone;
            *reinterpret_cast<float4*>(out + i) = v;
        } else {
            const float l[4] = {x[g].x, x[g].y, x[g].z, x[g].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n && (COPY || !(k >> e & 1))) out[i + e] = k >> e & 1 ? l[e] : gone;
        }
    }
    while (__any(left != 0)) {  // the whole wave, a token of each lane's at a time
        const bool mine = left != 0;
        const int at = mine ? __builtin_ctz(left) : 0, i = mine ? 4 * (tid + kThreads * (at >> 2)) + (at & 3) : 0;
        left &= left - 1;
        float l = 0.0f;
        if (COPY) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const float x0 = x[g].x, x1 = x[g].y, x2 = x[g].z, x3 = x[g].w;
                const float lo = at & 1 ? x1 : x0, hi = at & 1 ? x3 : x2;
                if (at >> 2 == g) l = at & 2 ? hi : lo;
            }
        } else if (mine) {
            l = in[i];
        }
        const Word w = mine ? what[i] : 0;
        double y = l;
        if (w & (kPrompt | kCountMask)) y = y > 0 ? y / (double)r : y * (double)r;
        const Word made = w & kCountMask;
        if (made) y -= (double)f * made + (double)p;
        const int first = a.M - (int)(w >> F::kFirst);
        double sum = w >> F::kFirst ? bias[first] : 0.0;
        // A token that is on the list again: all its biases in order, 4 x 64 entries at a time.
        for (uint64_t more = __ballot((w & kTwice) != 0); more; more &= more - 1) {
            const int lane = __builtin_ctzll(more);
            const int token = (int)t0 + __builtin_amdgcn_readlane(i, lane);
            const int o = __builtin_amdgcn_readlane(first, lane);
            double s = bias[o];
            for (int j0 = o + 1; j0 < a.M; j0 += 256) {
                int entry[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int j = j0 + 64 * u + (tid & 63);
                    entry[u] = j < a.M ? list[j] : -1;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    for (uint64_t hit = __ballot(entry[u] == token); hit; hit &= hit - 1)
                        s += bias[j0 + 64 * u + __builtin_ctzll(hit)];
            }
            if ((tid & 63) == lane) sum = s;
        }
        if (w >> F::kFirst) y += sum;
        if (mine) out[i] = (float)y;
    }
}

}  // namespace

}  // namespace alv

using namespace alv;

extern "C" int alv_adjust_logits(const float* logits, int64_t ld, float* out, int64_t ld_out, int B, int V,
                                 const int32_t* tokens, int64_t ld_tokens, int L, const int32_t* n_tokens,
                                 const int32_t* n_prompt, const float* repetition_dev, float repetition,
                                 const float* frequency_dev, float frequency, const float* presence_dev, float presence,
                                 const int32_t* bias_tokens, int64_t ld_bias_tokens, const float* bias, int64_t ld_bias,
                                 int M, const uint32_t* allowed, int64_t ld_allowed, void* stream) {
    if (B < 0 || V < 1 || L < 0 || M < 0) return fail(ALV_ERR_ARG, "bad shape B=%d V=%d L=%d M=%d", B, V, L, M);
    if (B > 0 && (!logits || !out || (L > 0 && !tokens) || (M > 0 && (!bias_tokens || !bias))))
        return fail(ALV_ERR_ARG, "null pointer");
    // (a list entry that is there again looks through the list: 2^16 of them are tens of milliseconds at most)
    if (B > 65535 || V > 1 << 24 || L > 1 << 30 || M > 1 << 16 || (int64_t)B * V > (int64_t)1 << 35)
        return fail(ALV_ERR_RANGE, "%d rows of %d logits, %d tokens and %d biases each (at most 65535, 2^24, 2^30, 2^16; 2^35 logits)",
                    B, V, L, M);
    if (B > 1 && std::max(ld, ld_out) > (int64_t)1 << 40)
        return fail(ALV_ERR_RANGE, "rows %lld and %lld apart (at most 2^40)", (long long)ld, (long long)ld_out);
    if (!repetition_dev && !(repetition > 0.0f)) return fail(ALV_ERR_ARG, "repetition %g: above 0", (double)repetition);
    if (B > 1 && (ld < V || ld_out < V || ld_tokens < 0 || ld_bias_tokens < 0 || ld_bias < 0 || ld_allowed < 0))
        return fail(ALV_ERR_ARG, "rows of %d logits, %lld and %lld apart", V, (long long)ld, (long long)ld_out);
    if (out == logits && B > 1 && ld != ld_out) return fail(ALV_ERR_ARG, "in place, rows are as far apart as they were");
    // Rows that are elsewhere: none of one's within another's (both may be columns of one array).
    if (B > 0 && out != logits) {
        const int64_t in0 = (int64_t)reinterpret_cast<uintptr_t>(logits), out0 = (int64_t)reinterpret_cast<uintptr_t>(out);
        const int64_t in1 = in0 + 4 * ((B > 1 ? (B - 1) * ld : 0) + V), out1 = out0 + 4 * ((B > 1 ? (B - 1) * ld_out : 0) + V);
        if (in0 < out1 && out0 < in1) {
            const int64_t d = B == 1 ? 0 : ((out0 - in0) / 4 % ld + ld) % ld;
            if (ld != ld_out || d < V || d + V > ld) return fail(ALV_ERR_ARG, "out overlaps logits");
        }
    }
    for (const void* p : {(const void*)logits, (const void*)out, (const void*)tokens, (const void*)n_tokens, (const void*)n_prompt,
                          (const void*)repetition_dev, (const void*)frequency_dev, (const void*)presence_dev,
                          (const void*)bias_tokens, (const void*)bias, (const void*)allowed})
        if (reinterpret_cast<uintptr_t>(p) % 4) return fail(ALV_ERR_ALIGN, "arrays need 4-byte alignment");
    if (B == 0) return ALV_OK;
    AdjustArgs a{};
    a.logits = logits, a.out = out, a.ld = ld, a.ld_out = ld_out, a.V = V;
    a.tokens = tokens, a.ld_tokens = ld_tokens, a.L = L, a.n_tokens = n_tokens, a.n_prompt = n_prompt;
    a.rep_dev = repetition_dev, a.freq_dev = frequency_dev, a.pres_dev = presence_dev;
    a.rep = repetition, a.freq = frequency, a.pres = presence;
    a.bias_tokens = bias_tokens, a.ld_bias_tokens = ld_bias_tokens, a.bias = bias, a.ld_bias = ld_bias, a.M = M;
    a.allowed = allowed, a.ld_allowed = ld_allowed;
    const bool small = L <= kMostCount && M <= kMostEntries;
    const bool wide = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                      (B == 1 || (ld % 4 == 0 && ld_out % 4 == 0));
    const size_t lds = L > 0 || M > 0 ? kRange * (small ? 4 : 8) : 0;
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, dim3((V + kRange - 1) / kRange, B), dim3(kThreads), lds, (hipStream_t)stream, a);
        return hip_check(hipGetLastError(), "adjust_kernel launch");
    };
    using Large = unsigned long long;
    if (out != logits) {
        if (wide) return small ? go(adjust_kernel<uint32_t, true, true>) : go(adjust_kernel<Large, true, true>);
        return small ? go(adjust_kernel<uint32_t, false, true>) : go(adjust_kernel<Large, false, true>);
    }
    if (wide) return small ? go(adjust_kernel<uint32_t, true, false>) : go(adjust_kernel<Large, true, false>);
    return small ? go(adjust_kernel<uint32_t, false, false>) : go(adjust_kernel<Large, false, false>);
}
