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
// token's first bias, and passes once over the logits. In place, only what changes
// is read and written.
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

constexpr int kRange = 4096;     // tokens of a workgroup
constexpr int kThreads = 256;
constexpr uint32_t kPrompt = 1u << 31;  // a count's bit: the token occurred (in the prompt, where nothing else is set)

__global__ void __launch_bounds__(kThreads) adjust_kernel(AdjustArgs a) {
    __shared__ uint32_t count[kRange];
    __shared__ uint32_t owner[kRange];  // index of a token's first list entry, ~0: none
    __shared__ int twice;               // a token is on the list again
    const int tid = threadIdx.x, b = blockIdx.y;
    const int64_t t0 = (int64_t)blockIdx.x * kRange;
    const int n = (int)min((int64_t)kRange, a.V - t0);
    const float r = a.rep_dev ? a.rep_dev[b] : a.rep, f = a.freq_dev ? a.freq_dev[b] : a.freq;
    const float p = a.pres_dev ? a.pres_dev[b] : a.pres;
    const bool history = a.L > 0 && (r != 1.0f || f != 0.0f || p != 0.0f);
    const bool biased = a.M > 0;
    if (history)
        for (int i = tid; i < kRange; i += kThreads) count[i] = 0;
    if (biased)
        for (int i = tid; i < kRange; i += kThreads) owner[i] = ~0u;
    if (tid == 0) twice = 0;
    __syncthreads();
    if (history) {
        const int32_t* row = a.tokens + b * a.ld_tokens;
        const int have = a.n_tokens ? max(0, min(a.n_tokens[b], a.L)) : a.L;
        const int prompt = a.n_prompt ? a.n_prompt[b] : 0;
        for (int i = tid; i < have; i += kThreads) {
            const int64_t x = row[i] - t0;
            if (x >= 0 && x < n) {
                if (i < prompt)
                    atomicOr(&count[x], kPrompt);
                else
                    atomicAdd(&count[x], 1u);
            }
        }
    }
    const int32_t* list = biased ? a.bias_tokens + b * a.ld_bias_tokens : nullptr;
    const float* bias = biased ? a.bias + b * a.ld_bias : nullptr;
    if (biased) {
        for (int i = tid; i < a.M; i += kThreads) {
            const int64_t x = list[i] - t0;
            if (x >= 0 && x < n) atomicMin(&owner[x], (uint32_t)i);
        }
        __syncthreads();
        for (int i = tid; i < a.M; i += kThreads) {
            const int64_t x = list[i] - t0;
            if (x >= 0 && x < n && owner[x] != (uint32_t)i) twice = 1;
        }
    }
    __syncthreads();
    const float* in = a.logits + b * a.ld + t0;
    float* out = a.out + b * a.ld_out + t0;
    const uint32_t* allowed = a.allowed ? a.allowed + b * a.ld_allowed + t0 / 32 : nullptr;
    const bool copy = a.out != a.logits;
    for (int i = tid; i < n; i += kThreads) {
        const uint32_t c = history ? count[i] : 0, o = biased ? owner[i] : ~0u;
        const bool gone = allowed && !(allowed[i >> 5] >> (i & 31) & 1);
        if (!copy && !c && o == ~0u && !gone) continue;
        float x = -__builtin_inff();
        if (!gone) {
            x = in[i];
            if (c || o != ~0u) {
                double y = x;
                if (c) y = y > 0 ? y / (double)r : y * (double)r;
                const uint32_t made = c & ~kPrompt;
                if (made) y -= (double)f * made + (double)p;
                if (o != ~0u) {
                    double s = bias[o];
                    if (twice)
                        for (int j = o + 1; j < a.M; ++j)
                            if (list[j] == t0 + i) s += bias[j];
                    y += s;
                }
                x = (float)y;
            }
        }
        out[i] = x;
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
    if (B > 65535 || V > 1 << 24 || L > 1 << 30 || (int64_t)B * V > (int64_t)1 << 35)
        return fail(ALV_ERR_RANGE, "%d rows of %d logits, %d tokens each (at most 65535, 2^24, 2^30; 2^35 logits)", B, V, L);
    if (!repetition_dev && !(repetition > 0.0f)) return fail(ALV_ERR_ARG, "repetition %g: above 0", (double)repetition);
    if (B > 1 && (ld < V || ld_out < V || ld_tokens < 0 || ld_bias_tokens < 0 || ld_bias < 0 || ld_allowed < 0))
        return fail(ALV_ERR_ARG, "rows of %d logits, %lld and %lld apart", V, (long long)ld, (long long)ld_out);
    if (out == logits && B > 1 && ld != ld_out) return fail(ALV_ERR_ARG, "in place, rows are as far apart as they were");
    // Rows that are elsewhere: none of one's within another's (both may be columns of one array).
    if (B > 0 && out != logits) {
        const int64_t in0 = (int64_t)reinterpret_cast<uintptr_t>(logits), out0 = (int64_t)reinterpret_cast<uintptr_t>(out);
        const int64_t in1 = in0 + 4 * ((B - 1) * ld + V), out1 = out0 + 4 * ((B - 1) * ld_out + V);
        if (in0 < out1 && out0 < in1) {
            const int64_t d = ((out0 - in0) / 4 % ld + ld) % ld;
            if (B == 1 || ld != ld_out || d < V || d + V > ld) return fail(ALV_ERR_ARG, "out overlaps logits");
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
    hipLaunchKernelGGL(adjust_kernel, dim3((V + kRange - 1) / kRange, B), dim3(kThreads), 0, (hipStream_t)stream, a);
    return hip_check(hipGetLastError(), "adjust_kernel launch");
}
