// Sampling from rows of logits with temperature, top-k, top-p and min-p, given
// the random numbers.
//
// Tokens in the order (logit descending, index ascending); w_r = exp((l_r -
// l_0) / T). The three cuts are prefixes of that order: the first k; those with
// sum_{j<r} w_j < p * (sum over the first k); those with w_r >= min_p. With Z the
// sum over the shortest of the three, the token is the first r with
// sum_{j<=r} w_j > u * Z. So all that is needed is three times the same thing:
// where does a running sum over the order cross a target.
//
// Weights are fixed-point 64-bit integers, exp in float64 scaled by 2^(62 -
// log2 of the vocabulary): integer sums do not depend on their order, so atomics
// change no result, and a sum of 2^18 weights is within 2^-36 of itself where
// float32 would shift every border between two tokens by 2^-24.
#include <algorithm>

#include "q4_device.h"
#include "q4_host.h"

namespace alv {

namespace {

struct SampleArgs {
    const float* logits;
    int64_t ld;
    int V;
    const float* u;
    const float* temp_dev;
    const int32_t* topk_dev;
    const float* topp_dev;
    const float* minp_dev;
    float temp, topp, minp;
    int topk;
    int shift;  // fixed-point bits of a weight
    int32_t* token;
    float* prob;
};

struct RowParams {
    bool greedy;
    double inv_t;
    double topp, minp, u;
    int topk;
};

__device__ __forceinline__ RowParams row_params(const SampleArgs& a, int b) {
    RowParams r;
    const float t = a.temp_dev ? a.temp_dev[b] : a.temp;
    const float p = a.topp_dev ? a.topp_dev[b] : a.topp;
    const float m = a.minp_dev ? a.minp_dev[b] : a.minp;
    const float u = a.u[b];
    r.greedy = !(t > 0.0f);
    r.inv_t = fmax(1.0 / (double)t, 1e-300);  // an infinite temperature: every finite logit weighs 1
    r.topk = a.topk_dev ? a.topk_dev[b] : a.topk;
    if (r.topk <= 0 || r.topk > a.V) r.topk = a.V;
    if (r.greedy) r.topk = 1;
    r.topp = p < 1.0f ? fmax((double)p, 0.0) : 1.0;  // NaN: no cut
    r.minp = m > 0.0f ? fmin((double)m, 1.0) : 0.0;
    r.u = u > 0.0f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
    return r;
}

// Order-preserving integer of a logit that is no NaN (both zeros alike).
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// exp((l - m) / T): 1 for l = m also where both are infinite.
__device__ __forceinline__ double weight(float l, float m, double inv_t) {
    return l == m ? 1.0 : exp(((double)l - (double)m) * inv_t);
}
__device__ __forceinline__ uint64_t fixed(double w, double scale) { return (uint64_t)rint(w * scale); }

constexpr int kRowThreads = 1024;
constexpr int kBins = 2048;

struct RowShared {
    uint32_t cnt[kBins];
    unsigned long long sum[kBins];
    unsigned long long wsum[kRowThreads / 64];
    uint32_t wcnt[kRowThreads / 64];
    float wmax[kRowThreads / 64];
    int widx[kRowThreads / 64];
    uint32_t bin;
    uint32_t before_cnt;
    unsigned long long before_sum;
};

struct Pick {
    uint32_t key;       // the crossing value's
    uint32_t cnt;       // tokens before the first that has it
    uint64_t sum;       // their weight
};

// The value at which the running count (by_count) or weight crosses: the one r
// with before_r <= x < before_r + own. Three passes of 11, 11 and 10 bits.
__device__ Pick pick(const float* l, int V, float m, double inv_t, double scale, bool by_count, uint64_t x, RowShared& s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Pick p{0, 0, 0};
    uint32_t mask = 0;
    for (int level = 0; level < 3; ++level) {
        const int sh = level == 0 ? 21 : (level == 1 ? 10 : 0);
        const uint32_t bits = level == 2 ? 0x3FFu : 0x7FFu;
        for (int i = tid; i < kBins; i += kRowThreads) {
            s.cnt[i] = 0;
            s.sum[i] = 0;
        }
        __syncthreads();
        for (int i = tid; i < V; i += kRowThreads) {
            const uint32_t k = key_of(l[i]);
            if ((k & mask) != p.key) continue;
            const uint32_t bin = bits - ((k >> sh) & bits);  // descending
            atomicAdd(&s.cnt[bin], 1u);
            atomicAdd(&s.sum[bin], (unsigned long long)fixed(weight(l[i], m, inv_t), scale));
        }
        __syncthreads();
        // Each thread two bins: the exclusive prefix before them.
        const uint32_t c0 = s.cnt[2 * tid], c1 = s.cnt[2 * tid + 1];
        const uint64_t w0 = s.sum[2 * tid], w1 = s.sum[2 * tid + 1];
        uint32_t c = c0 + c1;
        uint64_t w = w0 + w1;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t cu = __shfl_up(c, o);
            const uint64_t wu = __shfl_up((unsigned long long)w, o);
            if (lane >= o) c += cu, w += wu;
        }
        if (lane == 63) s.wcnt[wave] = c, s.wsum[wave] = w;
        __syncthreads();
        uint32_t cb = p.cnt + c - c0 - c1;
        uint64_t wb = p.sum + w - w0 - w1;
        for (int i = 0; i < wave; ++i) cb += s.wcnt[i], wb += s.wsum[i];
        const uint64_t b0 = by_count ? cb : wb, i0 = by_count ? c0 : w0, i1 = by_count ? c1 : w1;
        if (b0 <= x && x < b0 + i0) s.bin = 2 * tid, s.before_cnt = cb, s.before_sum = wb;
        if (b0 + i0 <= x && x < b0 + i0 + i1) s.bin = 2 * tid + 1, s.before_cnt = cb + c0, s.before_sum = wb + w0;
        __syncthreads();
        p.key |= (bits - s.bin) << sh;
        p.cnt = s.before_cnt;
        p.sum = s.before_sum;
        mask |= bits << sh;
        __syncthreads();
    }
    return p;
}

// One workgroup per row, any values.
__global__ void __launch_bounds__(kRowThreads) sample_row_kernel(SampleArgs a) {
    __shared__ RowShared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
    const float* l = a.logits + b * a.ld;
    const RowParams rp = row_params(a, b);
    // The largest logit and its first index; a NaN counts as largest.
    float m = -__builtin_inff();
    int mi = a.V;
    for (int i = tid; i < a.V; i += kRowThreads) {
        const float v = l[i];
        if (mi == a.V || v > m || (v != v && m == m)) m = v, mi = i;
    }
    for (int o = 32; o; o >>= 1) {
        const float v = __shfl_xor(m, o);
        const int vi = __shfl_xor(mi, o);
        const bool nan = v != v, mnan = m != m;
        if (nan != mnan ? nan : (v > m || ((v == m || nan) && vi < mi))) m = v, mi = vi;
    }
    if (lane == 0) s.wmax[wave] = m, s.widx[wave] = mi;
    __syncthreads();
    m = s.wmax[0], mi = s.widx[0];
    for (int i = 1; i < kRowThreads / 64; ++i) {
        const float v = s.wmax[i];
        const int vi = s.widx[i];
        const bool nan = v != v, mnan = m != m;
        if (vi < a.V && (nan != mnan ? nan : (v > m || ((v == m || nan) && vi < mi)))) m = v, mi = vi;
    }
    if (m != m || m == -__builtin_inff() || rp.topk == 1) {
        if (tid == 0) {
            a.token[b] = m == -__builtin_inff() ? -1 : mi;
            if (a.prob) a.prob[b] = m != m ? m : (m == -__builtin_inff() ? 0.0f : 1.0f);
        }
        return;
    }
    const double scale = __builtin_ldexp(1.0, a.shift);
    // The whole row's weight, and that of the tokens min-p keeps.
    uint64_t S = 0, Sm = 0;
    for (int i = tid; i < a.V; i += kRowThreads) {
        const double w = weight(l[i], m, rp.inv_t);
        const uint64_t f = fixed(w, scale);
        S += f;
        if (w >= rp.minp) Sm += f;
    }
    for (int o = 32; o; o >>= 1) {
        S += __shfl_xor((unsigned long long)S, o);
        Sm += __shfl_xor((unsigned long long)Sm, o);
    }
    __syncthreads();
    if (lane == 0) s.wsum[wave] = S, s.sum[wave] = Sm;
    __syncthreads();
    S = Sm = 0;
    for (int i = 0; i < kRowThreads / 64; ++i) S += s.wsum[i], Sm += s.sum[i];
    __syncthreads();
    uint64_t Z = S;
    auto own_weight = [&](uint32_t key) { return fixed(weight(logit_of(key), m, rp.inv_t), scale); };
    if (rp.topk < a.V) {
        const Pick p = pick(l, a.V, m, rp.inv_t, scale, true, (uint64_t)rp.topk - 1, s);
        Z = p.sum + (uint64_t)(rp.topk - (int)p.cnt) * own_weight(p.key);
    }
    if (rp.topp < 1.0) {
        const uint64_t target = max((uint64_t)1, (uint64_t)ceil(rp.topp * (double)Z));
        if (target < Z) {
            const Pick p = pick(l, a.V, m, rp.inv_t, scale, false, target - 1, s);
            const uint64_t w = own_weight(p.key);
            Z = min(Z, p.sum + ((target - 1 - p.sum) / w + 1) * w);
        }
    }
    Z = min(Z, Sm);
    const uint64_t x = min((uint64_t)(rp.u * (double)Z), Z - 1);
    const Pick p = pick(l, a.V, m, rp.inv_t, scale, false, x, s);
    const uint64_t w = own_weight(p.key);
    int skip = (int)((x - p.sum) / w);  // equal logits ahead of the token, by index
    // The token: the skip-th with that value.
    for (int i0 = 0; i0 < a.V; i0 += kRowThreads) {
        const int i = i0 + tid;
        const bool is = i < a.V && key_of(l[i]) == p.key;
        const uint64_t bal = __ballot(is);
        if (lane == 0) s.wcnt[wave] = __popcll(bal);
        __syncthreads();
        int before = 0, total = 0;
        for (int q = 0; q < kRowThreads / 64; ++q) {
            if (q < wave) before += s.wcnt[q];
            total += s.wcnt[q];
        }
        if (is && before + __popcll(bal & ((1ull << lane) - 1)) == skip) {
            a.token[b] = i;
            if (a.prob) a.prob[b] = (float)(weight(l[i], m, rp.inv_t) / ((double)Z / scale));
        }
        __syncthreads();
        if (skip < total) break;
        skip -= total;
    }
}

}  // namespace

}  // namespace alv

using namespace alv;

extern "C" uint64_t alv_sample_workspace(int B, int V) { return 0; }

extern "C" int alv_sample(const float* logits, int64_t ld, int B, int V, const float* u, const float* temperature_dev,
                          float temperature, const int32_t* top_k_dev, int top_k, const float* top_p_dev, float top_p,
                          const float* min_p_dev, float min_p, int32_t* token, float* prob, void* workspace,
                          uint64_t workspace_bytes, void* stream) {
    if (B < 0 || V < 1 || ld < V) return fail(ALV_ERR_ARG, "bad logits shape B=%d vocab=%d ld=%lld", B, V, (long long)ld);
    if (B == 0) return ALV_OK;
    if (!logits || !u || !token) return fail(ALV_ERR_ARG, "null pointer");
    if (V > 1 << 24 || B > 1 << 16) return fail(ALV_ERR_RANGE, "%d rows of %d logits (at most 65536 of 2^24)", B, V);
    for (const void* p : {(const void*)logits, (const void*)u, (const void*)temperature_dev, (const void*)top_k_dev,
                          (const void*)top_p_dev, (const void*)min_p_dev, (const void*)token, (const void*)prob})
        if (reinterpret_cast<uintptr_t>(p) % 4) return fail(ALV_ERR_ALIGN, "logits, parameters and outputs need 4-byte alignment");
    SampleArgs a{};
    a.logits = logits, a.ld = ld, a.V = V, a.u = u;
    a.temp_dev = temperature_dev, a.topk_dev = top_k_dev, a.topp_dev = top_p_dev, a.minp_dev = min_p_dev;
    a.temp = temperature, a.topk = top_k, a.topp = top_p, a.minp = min_p;
    int bits = 0;
    while ((1 << bits) < V) ++bits;
    a.shift = std::min(52, 62 - bits);
    a.token = token, a.prob = prob;
    hipLaunchKernelGGL(sample_row_kernel, dim3(B), dim3(kRowThreads), 0, (hipStream_t)stream, a);
    return hip_check(hipGetLastError(), "sample_row_kernel launch");
}
