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
// change no result, and the roundings of 2^18 weights add up to about 2^-36 of the
// largest (2^-27 if all went one way), where float32 would shift every border
// between two tokens by 2^-24.
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
    unsigned char* work;
    int pieces;  // of a row; 0: a row is one workgroup's alone
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
// w * scale to the nearest integer, at most 2^52: the last bits of 2^52 plus it.
__device__ __forceinline__ uint64_t fixed(double w, double scale) {
    return __builtin_bit_cast(uint64_t, fma(w, scale, 0x1p52)) - __builtin_bit_cast(uint64_t, 0x1p52);
}

// Targets of the three crossings. top-p keeps what begins below ceil(p S); a
// token is drawn at floor(u Z).
__device__ __forceinline__ uint64_t topp_target(double p, uint64_t S) { return max((uint64_t)1, (uint64_t)ceil(p * (double)S)); }
__device__ __forceinline__ uint64_t draw_target(double u, uint64_t Z) { return min((uint64_t)(u * (double)Z), Z - 1); }

constexpr int kRowThreads = 1024;

// ---- several workgroups per row -----------------------------------------------------
//
// Four launches: the pieces' largest logits; a histogram of the row over x = (l_0 -
// l) / T, from 0 to where a weight rounds to nothing (or the row's range); from
// its prefix sums the bins in which the three crossings can fall, and the
// collection of those bins' tokens; the crossings among those, by comparison
// where they are few, else by a finer histogram first. Every step moves integers,
// so no order of atomics shows. A row whose bins hold more than kCand tokens (thousands
// of one value, or more than a million logits) is left to one workgroup (sample_over).
//
// What bounds it: one row is a chain of launches, each a trip or two to memory (one
// row of 262144: 25 us, of them 4 + 8 + 9 + 4 in the kernels); many rows, the
// histogram (48 rows of 128256, 52 us: 9 + 18 + 16 + 10; reading the logits three
// times is 15 of them).
constexpr int kPieceThreads = 256;
constexpr int kWaves = kPieceThreads / 64;
constexpr int kPiece = 16 * kPieceThreads;  // logits per workgroup (2 or 4 times as many are slower by a half: too few loads on their way)
constexpr int kCoarse = 1024;     // bins
constexpr int kFine = 2048;       // finer bins of the collected ones
constexpr int kCand = 4096;       // tokens collected per row
constexpr int kLast = 128;        // tokens compared one with another (256 take 30 us, 128 in the finer histogram 9)

struct RowWork {  // per row
    float* top;         // [pieces] largest logit
    float* low;         // [pieces] smallest logit above -infinity
    int* at;            // [pieces] first index of the largest
    unsigned long long* minp;   // [pieces] weight that min-p keeps
    unsigned long long* sum;    // [kCoarse] weight of each bin, then its prefix [kCoarse + 1]
    uint32_t* cnt;              // [kCoarse] count of each bin, then its prefix [kCoarse + 1]
    unsigned long long* cw;     // [kCand] collected weights,
    float* cl;          // logits,
    float* cp;          // places in the histogram
    int* ci;            // and indices
    uint32_t* want;     // [kCoarse / 32] a bit per bin to collect
    uint32_t* n;        // collected
    uint32_t* over;     // not 0: those bins hold more than kCand
};

// (offsets of 16 bytes up to where the pieces' values begin)
__host__ __device__ inline uint64_t row_bytes(int pieces) {
    return 8ull * (2 * kCoarse + 2 + kCand) + 4ull * (2 * kCoarse + 4 + 3 * kCand + kCoarse / 32 + 4) + (20ull * pieces + 15 & ~15ull);
}
__device__ __forceinline__ RowWork row_work(const SampleArgs& a, int b) {
    RowWork w;
    unsigned char* p = a.work + (uint64_t)b * row_bytes(a.pieces);
    w.sum = reinterpret_cast<unsigned long long*>(p);
    w.cw = w.sum + 2 * kCoarse + 2;
    w.cnt = reinterpret_cast<uint32_t*>(w.cw + kCand);
    w.cl = reinterpret_cast<float*>(w.cnt + 2 * kCoarse + 4);
    w.cp = w.cl + kCand;
    w.ci = reinterpret_cast<int*>(w.cp + kCand);
    w.want = reinterpret_cast<uint32_t*>(w.ci + kCand);
    w.n = w.want + kCoarse / 32;
    w.over = w.n + 1;
    w.minp = reinterpret_cast<unsigned long long*>(w.n + 4);
    w.top = reinterpret_cast<float*>(w.minp + a.pieces);
    w.low = w.top + a.pieces;
    w.at = reinterpret_cast<int*>(w.low + a.pieces);
    return w;
}

// (value, index) a before b in numpy's argmax order: NaN first, then the larger,
// then the lower index.
__device__ __forceinline__ bool ahead(float va, int ia, float vb, int ib) {
    const bool na = va != va, nb = vb != vb;
    if (na != nb) return na;
    return va > vb || ((va == vb || na) && ia < ib);
}

// This thread's 16 logits of the piece, in 4 groups of 4 (index base + 4
// kPieceThreads g + 4 tid + e); -infinity past the row.
__device__ __forceinline__ void load_piece(const float* l, int V, int base, int tid, float (&v)[16]) {
    if ((reinterpret_cast<uintptr_t>(l) & 15) == 0 && base + kPiece <= V) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 f = *reinterpret_cast<const float4*>(l + base + 4 * kPieceThreads * g + 4 * tid);
            v[4 * g] = f.x, v[4 * g + 1] = f.y, v[4 * g + 2] = f.z, v[4 * g + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = base + 4 * kPieceThreads * g + 4 * tid + e;
                v[4 * g + e] = i < V ? l[i] : -__builtin_inff();
            }
    }
}
__device__ __forceinline__ int piece_index(int base, int tid, int k) {
    return base + 4 * kPieceThreads * (k >> 2) + 4 * tid + (k & 3);
}

__global__ void __launch_bounds__(kPieceThreads) sample_top_kernel(SampleArgs a) {
    __shared__ float st[kWaves], sl[kWaves];
    __shared__ int si[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.y, base = blockIdx.x * kPiece;
    const RowWork rw = row_work(a, b);
    float v[16];
    load_piece(a.logits + b * a.ld, a.V, base, tid, v);
    float m = v[0], lo = __builtin_inff();
    int mi = piece_index(base, tid, 0);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        if (k && ahead(v[k], piece_index(base, tid, k), m, mi)) m = v[k], mi = piece_index(base, tid, k);
        if (v[k] > -__builtin_inff()) lo = fminf(lo, v[k]);
    }
    for (int o = 32; o; o >>= 1) {
        const float u = __shfl_xor(m, o);
        const int ui = __shfl_xor(mi, o);
        if (ahead(u, ui, m, mi)) m = u, mi = ui;
        lo = fminf(lo, __shfl_xor(lo, o));
    }
    if (lane == 0) st[wave] = m, si[wave] = mi, sl[wave] = lo;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kWaves; ++w) {
            if (ahead(st[w], si[w], m, mi)) m = st[w], mi = si[w];
            lo = fminf(lo, sl[w]);
        }
        rw.top[blockIdx.x] = m;
        rw.at[blockIdx.x] = mi;
        rw.low[blockIdx.x] = lo;
        if (blockIdx.x == 0) *rw.n = 0;
    }
    // The row's histogram, clear for the next launch.
    for (int i = blockIdx.x * kPieceThreads + tid; i < kCoarse; i += a.pieces * kPieceThreads) {
        rw.cnt[i] = 0;
        rw.sum[i] = 0;
    }
}

// x from which a weight rounds to nothing.
__device__ __forceinline__ float weightless(const SampleArgs& a) { return (float)(a.shift + 1) * 0.693147182464599609375f; }

// What a row's largest and smallest logits decide.
struct RowRange {
    float m, low;   // the largest, and the smallest above -infinity
    int at;
    bool done;      // the token is `at` (or there is none)
    float bins;     // bins per unit of x
    float end;      // x from which a weight is nothing
};
__device__ __forceinline__ RowRange row_range(const SampleArgs& a, const RowWork& rw, const RowParams& rp, int lane) {
    float m = -__builtin_inff(), lo = __builtin_inff();
    int at = 0x7FFFFFFF;
    for (int i = lane; i < a.pieces; i += 64) {
        if (ahead(rw.top[i], rw.at[i], m, at)) m = rw.top[i], at = rw.at[i];
        lo = fminf(lo, rw.low[i]);
    }
    for (int o = 32; o; o >>= 1) {
        const float u = __shfl_xor(m, o);
        const int ui = __shfl_xor(at, o);
        if (ahead(u, ui, m, at)) m = u, at = ui;
        lo = fminf(lo, __shfl_xor(lo, o));
    }
    RowRange r;
    r.m = m;
    r.low = lo;
    r.at = at;
    r.done = m != m || m == -__builtin_inff() || rp.topk == 1;
    r.end = weightless(a);
    const float range = (float)(((double)m - (double)lo) * rp.inv_t);
    r.bins = (float)kCoarse / fmaxf(fminf(range, r.end), 1e-30f);  // NaN range (infinities): the whole
    return r;
}
// x in bins, from 0; a value of kCoarse or more in the last. The same for equal
// logits and never smaller for a smaller one.
__device__ __forceinline__ double x_of(float l, const RowRange& r, double inv_t) {
    return l == r.m ? 0.0 : ((double)r.m - (double)l) * inv_t;
}
__device__ __forceinline__ float place_of(double x, const RowRange& r) { return fminf((float)x * r.bins, (float)kCoarse - 0.00390625f); }

__global__ void __launch_bounds__(kPieceThreads) sample_hist_kernel(SampleArgs a) {
    __shared__ uint32_t cnt[kCoarse];
    __shared__ unsigned long long sum[kCoarse];
    __shared__ unsigned long long smin[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.y, base = blockIdx.x * kPiece;
    const RowWork rw = row_work(a, b);
    float v[16];
    load_piece(a.logits + b * a.ld, a.V, base, tid, v);
    const RowParams rp = row_params(a, b);
    const RowRange rr = row_range(a, rw, rp, lane);
    if (rr.done) return;
    for (int i = tid; i < kCoarse; i += kPieceThreads) {
        cnt[i] = 0;
        sum[i] = 0;
    }
    __syncthreads();
    const double scale = __builtin_ldexp(1.0, a.shift);
    uint64_t kept = 0;
#pragma unroll 4
    for (int k = 0; k < 16; ++k) {
        const double x = x_of(v[k], rr, rp.inv_t);
        if (!(x < rr.end)) continue;
        const double w = exp(-x);
        const uint64_t f = fixed(w, scale);
        if (w >= rp.minp) kept += f;
        const int bin = (int)place_of(x, rr);
        atomicAdd(&cnt[bin], 1u);
        atomicAdd(&sum[bin], (unsigned long long)f);
    }
    for (int o = 32; o; o >>= 1) kept += __shfl_xor((unsigned long long)kept, o);
    if (lane == 0) smin[wave] = kept;
    __syncthreads();
    for (int i = tid; i < kCoarse; i += kPieceThreads) {
        // (added up here rather than kept per piece: reading 64 pieces'
        // histograms takes one workgroup 30 us)
        if (cnt[i]) {
            atomicAdd(rw.cnt + i, cnt[i]);
            atomicAdd(rw.sum + i, sum[i]);
        }
    }
    if (tid == 0) {
        kept = 0;
        for (int i = 0; i < kWaves; ++i) kept += smin[i];
        rw.minp[blockIdx.x] = kept;
    }
}

// The prefix of a row's histogram, and the bins in which the crossings can fall.
struct PlanShared {
    unsigned long long pre[kCoarse + 1], wsum[kWaves];
    uint32_t prec[kCoarse + 1], wcnt[kWaves], want[kCoarse / 32];
    int hit;
};
// The tokens those bins hold. Each thread has kCoarse / kPieceThreads bins.
__device__ __forceinline__ uint32_t row_plan(const SampleArgs& a, const RowWork& rw, const RowParams& rp, PlanShared& s) {
    constexpr int E = kCoarse / kPieceThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t c[E + 1], own = 0;  // before bin E tid + e
    uint64_t w[E + 1], ownw = 0, Sm = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        c[e] = rw.cnt[E * tid + e];
        w[e] = rw.sum[E * tid + e];
    }
    for (int g = lane; g < a.pieces; g += 64) Sm += rw.minp[g];
    if (tid < kCoarse / 32) s.want[tid] = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) own += c[e], ownw += w[e];
    for (int o = 32; o; o >>= 1) Sm += __shfl_xor((unsigned long long)Sm, o);
    uint32_t ci = own;
    uint64_t wi = ownw;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t cu = __shfl_up(ci, o);
        const uint64_t wu = __shfl_up((unsigned long long)wi, o);
        if (lane >= o) ci += cu, wi += wu;
    }
    if (lane == 63) s.wcnt[wave] = ci, s.wsum[wave] = wi;
    __syncthreads();
    ci -= own, wi -= ownw;
    for (int i = 0; i < wave; ++i) ci += s.wcnt[i], wi += s.wsum[i];
#pragma unroll
    for (int e = 0; e <= E; ++e) {
        const uint32_t cn = e < E ? c[e] : 0;
        const uint64_t wn = e < E ? w[e] : 0;
        c[e] = ci, w[e] = wi;
        if (e < E || tid == kPieceThreads - 1) s.prec[E * tid + e] = ci, s.pre[E * tid + e] = wi;
        ci += cn, wi += wn;
    }
    __syncthreads();
    const uint64_t S = s.pre[kCoarse];
    // The bin in which a count or a sum of x crosses.
    auto bin_at = [&](bool by_count, uint64_t x) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (by_count ? (c[e] <= x && x < c[e + 1]) : (w[e] <= x && x < w[e + 1])) s.hit = E * tid + e;
        __syncthreads();
        return s.hit;
    };
    uint64_t lo = S, hi = S;  // between what the sum of the kept lies
    int t = -1, t0 = -1, t1 = -1;
    if ((uint32_t)rp.topk < s.prec[kCoarse]) {
        t = bin_at(true, (uint64_t)rp.topk - 1);
        lo = s.pre[t];
        hi = s.pre[t + 1];
    }
    if (rp.topp < 1.0) {
        const uint64_t p0 = topp_target(rp.topp, lo), p1 = topp_target(rp.topp, hi);
        t0 = bin_at(false, p0 - 1), t1 = p1 == p0 ? t0 : bin_at(false, p1 - 1);
        lo = min(lo, (uint64_t)s.pre[t0]);
        hi = min(hi, (uint64_t)s.pre[t1 + 1]);
    }
    lo = max(min(lo, Sm), (uint64_t)1);
    hi = max(min(hi, Sm), (uint64_t)1);
    const int d0 = bin_at(false, draw_target(rp.u, lo)), d1 = lo == hi ? d0 : bin_at(false, draw_target(rp.u, hi));
    uint32_t bits = 0, total = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = E * tid + e;
        if (i == t || (i >= t0 && i <= t1) || (i >= d0 && i <= d1)) bits |= 1u << e, total += c[e + 1] - c[e];
    }
    if (bits) atomicOr(&s.want[E * tid >> 5], bits << (E * tid & 31));
    for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
    if (lane == 0) s.wcnt[wave] = total;
    __syncthreads();
    total = 0;
    for (int i = 0; i < kWaves; ++i) total += s.wcnt[i];
    return total;
}

// Each workgroup finds the bins for itself, 12 KB in cache: a launch less.
__global__ void __launch_bounds__(kPieceThreads) sample_collect_kernel(SampleArgs a) {
    __shared__ PlanShared s;
    const int tid = threadIdx.x, lane = tid & 63, b = blockIdx.y, base = blockIdx.x * kPiece;
    const RowWork rw = row_work(a, b);
    float v[16];
    load_piece(a.logits + b * a.ld, a.V, base, tid, v);
    const RowParams rp = row_params(a, b);
    const RowRange rr = row_range(a, rw, rp, lane);
    if (rr.done) return;
    const bool over = row_plan(a, rw, rp, s) > kCand;
    if (blockIdx.x == 0) {  // for the last launch
        for (int i = tid; i <= kCoarse; i += kPieceThreads) {
            rw.cnt[kCoarse + i] = s.prec[i];
            rw.sum[kCoarse + i] = s.pre[i];
        }
        if (tid < kCoarse / 32) rw.want[tid] = s.want[tid];
        if (tid == 0) *rw.over = over;
    }
    if (over) return;
    const double scale = __builtin_ldexp(1.0, a.shift);
    uint32_t mine = 0, mask = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const double x = x_of(v[k], rr, rp.inv_t);
        if (!(x < rr.end)) continue;
        const int bin = (int)place_of(x, rr);
        if (s.want[bin >> 5] >> (bin & 31) & 1) mask |= 1u << k, ++mine;
    }
    if (!__any(mine != 0)) return;
    uint32_t at = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(at, o);
        if (lane >= o) at += u;
    }
    uint32_t first = lane == 63 ? atomicAdd(rw.n, at) : 0;
    at += __shfl(first, 63) - mine;
#pragma unroll 1
    for (int k = 0; __any(mask >> k); ++k) {
        if (!(mask >> k & 1)) continue;
        float lk = v[0];
#pragma unroll
        for (int q = 1; q < 16; ++q) lk = q == k ? v[q] : lk;
        rw.cl[at] = lk;
        rw.cp[at] = place_of(x_of(lk, rr, rp.inv_t), rr);
        rw.cw[at] = fixed(weight(lk, rr.m, rp.inv_t), scale);
        rw.ci[at] = piece_index(base, tid, k);
        ++at;
    }
}

constexpr int kPer = kCand / kRowThreads;  // collected tokens of a thread
constexpr int kLine = 256;
struct LastShared {
    union {
        struct {
            // the collected bins, each cut into kFine / (their number) fine ones
            uint32_t cnt[kFine];
            unsigned long long sum[kFine];
            uint32_t base_cnt[kCoarse];            // by collected bin: what comes before it
            unsigned long long base_sum[kCoarse];
        };
        unsigned long long line[kRowThreads / 64][kLine];  // or the waves' tokens found in a row (OfRow)
    };
    uint32_t pcnt[kFine];
    unsigned long long psum[kFine];
    uint32_t want[kCoarse / 32];
    unsigned long long wsum[kRowThreads / 64];
    uint32_t wcnt[kRowThreads / 64];
    // the tokens of one fine bin
    float el[kLast];
    int ei[kLast];
    unsigned long long ew[kLast];
    int ne, f;
    uint32_t before_cnt;
    unsigned long long before_sum;
    unsigned long long lo, hi;  // the first and last of their places in the order
    // the token found, and the weight up to and with it
    float rl;
    int ri;
    unsigned long long through;
};

// A thread's two bins: counts and weights (c, ws), and what comes before them (cb, wb).
struct BinPair {
    uint32_t cb[kFine / kRowThreads], c[kFine / kRowThreads];
    unsigned long long wb[kFine / kRowThreads], ws[kFine / kRowThreads];
};
// A thread's collected tokens.
// LINE: token q is index i[0] + 1024 q, else i[q].
template <int PER, bool LINE>
struct LastRegs {
    float l[PER];
    int i[LINE ? 1 : PER];
    uint32_t two[PER / 2];  // the fine bins of two tokens each (of none: 0xFFFF)
    unsigned long long w[PER];
    __device__ __forceinline__ int bin(int q) const { return two[q / 2] >> 16 * (q & 1) & 0xFFFFu; }
    __device__ __forceinline__ void set_bin(int q, int f) {
        two[q / 2] = q & 1 ? (two[q / 2] & 0xFFFFu) | (uint32_t)f << 16 : (two[q / 2] & 0xFFFF0000u) | (uint32_t)f;
    }
    __device__ __forceinline__ void no_bins() {
#pragma unroll
        for (int q = 0; q < PER / 2; ++q) two[q] = ~0u;
    }
    __device__ __forceinline__ int index(int q) const {
        if constexpr (!LINE) return i[q];
        int first = i[0];
        asm volatile("" : "+v"(first));  // (as below)
        return first + q * kRowThreads;
    }
};

// A histogram's two bins of this thread, `c0` and `w0` ahead of the first bin.
__device__ __forceinline__ void bin_prefix(const uint32_t* cnt, const unsigned long long* sum, uint32_t c0, uint64_t w0,
                                           BinPair& r, LastShared& s) {
    constexpr int E = kFine / kRowThreads;
    const int tid = threadIdx.x, lane = tid & 63;
    uint32_t own = 0;
    uint64_t ownw = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        r.c[e] = cnt[E * tid + e];
        r.ws[e] = sum[E * tid + e];
        own += r.c[e];
        ownw += r.ws[e];
    }
    uint32_t c = own;
    uint64_t w = ownw;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t cu = __shfl_up(c, o);
        const uint64_t wu = __shfl_up((unsigned long long)w, o);
        if (lane >= o) c += cu, w += wu;
    }
    if (lane == 63) s.wcnt[tid >> 6] = c, s.wsum[tid >> 6] = w;
    __syncthreads();
    c += c0 - own;
    w += w0 - ownw;
    for (int i = 0; i < (tid >> 6); ++i) c += s.wcnt[i], w += s.wsum[i];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        r.cb[e] = c;
        r.wb[e] = w;
        c += r.c[e];
        w += r.ws[e];
    }
}
// The bin in which the running count or weight crosses x, and what comes before it, for all threads behind the
// next barrier.
__device__ __forceinline__ void find_bin(const BinPair& r, bool by_count, uint64_t x, LastShared& s) {
#pragma unroll
    for (int e = 0; e < kFine / kRowThreads; ++e) {
        const uint64_t b = by_count ? r.cb[e] : r.wb[e], own = by_count ? r.c[e] : r.ws[e];
        if (b <= x && x < b + own)
            s.f = threadIdx.x * (kFine / kRowThreads) + e, s.before_cnt = r.cb[e], s.before_sum = r.wb[e];
    }
}

// A token's place in the order (logit descending, index ascending) as one number, the logit's 32 bits above the
// index's (V needs no more than 62 - shift). Computed anew in each turn of a loop: kept, it is two registers a
// token, and 16 tokens leave none (256 rows of 16384 logits 26 -> 44 us, with indices and bins kept too).
__device__ __forceinline__ uint64_t place_in_order(float l, int i, int shift) {
    asm volatile("" : "+v"(l));
    return (uint64_t)~key_of(l) << (62 - shift) | (uint32_t)i;
}

// The collected tokens of fine bin f whose places are in [lo, hi].
template <int PER, bool LINE>
struct OfBin {
    static constexpr bool kAlike = false;
    const LastRegs<PER, LINE>& r;
    int f, shift;
    template <class F>
    __device__ __forceinline__ void operator()(uint64_t lo, uint64_t hi, F each) const {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            if (r.bin(q) != f) continue;
            const uint64_t c = place_in_order(r.l[q], r.index(q), shift);
            if (c >= lo && c <= hi) each(c, r.l[q], r.index(q), r.w[q]);
        }
    }
};

// The row's tokens whose places are in [lo, hi], from the logits: a wave lines up those it finds and takes them 64 at
// a time, so that the exponential runs once for 64 tokens however few of the row they are, and not for a value it has.
struct OfRow {
    static constexpr bool kAlike = true;  // (a run of one value: 64 tokens of one bin, one after the other in an atomic)
    static constexpr int kTurns = 4, kAtOnce = 3;
    static_assert(64 * kAtOnce + 63 <= kLine, "what a turn finds, beside what is left");
    const float* l;
    int V, shift;
    float m;
    double inv_t;
    unsigned long long (*line)[kLine];
    template <class F>
    __device__ __forceinline__ void operator()(uint64_t lo, uint64_t hi, F each) const {
        const int tid = threadIdx.x, lane = tid & 63, bits = 62 - shift;
        const double scale = __builtin_ldexp(1.0, shift);
        const float top = logit_of(~(uint32_t)(lo >> bits)), least = logit_of(~(uint32_t)(hi >> bits));
        unsigned long long* q = line[tid >> 6];
        int i0 = 0, i1 = V, n = 0;
        if (lo >> bits == hi >> bits) {  // one value: of these indices
            i0 = (int)(lo & ((1u << bits) - 1));
            i1 = min(V, (int)(hi & ((1u << bits) - 1)) + 1);
        }
        float had = __builtin_nanf("");
        uint64_t its = 0;
        // (the last k first: nothing moves)
        auto take = [&](int k) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            n -= k;
            if (lane < k) {
                const uint64_t e = q[n + lane];
                const float v = __builtin_bit_cast(float, (uint32_t)e);
                if (v != had) had = v, its = fixed(weight(v, m, inv_t), scale);
                const uint64_t c = place_in_order(v, (int)(e >> 32), shift);
                if (c >= lo && c <= hi) each(c, v, (int)(e >> 32), its);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        };
        constexpr int kAhead = kTurns * kAtOnce;
        for (int base = i0; base < i1; base += kAhead * kRowThreads) {
            float v[kAhead];
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                const int i = base + e * kRowThreads + tid;
                v[e] = i < i1 ? l[i] : -__builtin_inff();  // (no place: m - infinity weighs nothing)
            }
#pragma unroll 1
            for (int t = 0; t < kTurns; ++t) {
#pragma unroll
                for (int e = 0; e < kAtOnce; ++e) {
                    const float ve = v[e];
                    const int i = base + (t * kAtOnce + e) * kRowThreads + tid;
                    const bool is = ve >= least && ve <= top;
                    const uint64_t found = __ballot(is);
                    if (is) q[n + __popcll(found & ((1ull << lane) - 1))] = (uint64_t)i << 32 | __builtin_bit_cast(uint32_t, ve);
                    n += __popcll(found);
                }
#pragma unroll
                for (int e = 0; e + kAtOnce < kAhead; ++e) v[e] = v[e + kAtOnce];
#pragma unroll 1
                while (n >= 64) take(64);
            }
        }
        take(n);
    }
};

// n tokens with places in [lo, hi] cut to at most kLast around the crossing: the places into kFine equal parts, until
// the part that holds it has no more. (Logits that differ in their last bits or not at all: rounded to bf16 there are
// hundreds of each value.) Places differ by one at least, so that ends. A row of 262144 logits with top-p, rounded to
// bf16, 41 us (not rounded 34).
template <class M>
__device__ __forceinline__ void narrow(uint32_t n, uint64_t& lo, uint64_t& hi, bool by_count, uint64_t x, const M& tokens,
                                       LastShared& s) {
    const int tid = threadIdx.x;
    while (n > kLast) {
        const int sh = max(0, 53 - __clzll(hi - lo));  // (hi - lo) >> sh is less than kFine
        const uint32_t c0 = s.before_cnt;
        const uint64_t w0 = s.before_sum;
#pragma unroll
        for (int e = 0; e < kFine / kRowThreads; ++e) {
            s.pcnt[tid + e * kRowThreads] = 0;
            s.psum[tid + e * kRowThreads] = 0;
        }
        __syncthreads();
        tokens(lo, hi, [&](uint64_t c, float, int, uint64_t w) {
            const uint32_t bin = (uint32_t)((c - lo) >> sh);
            bool left = true;
            if constexpr (M::kAlike)
#pragma unroll 1
                for (int turn = 0; turn < 4 && __any(left); ++turn)
                    if (left) {
                        const uint32_t bin0 = __builtin_amdgcn_readfirstlane(bin);
                        const uint32_t w_lo = __builtin_amdgcn_readfirstlane((uint32_t)w);
                        const uint32_t w_hi = __builtin_amdgcn_readfirstlane((uint32_t)(w >> 32));
                        const bool alike = bin == bin0 && w == ((uint64_t)w_hi << 32 | w_lo);
                        const uint64_t same = __ballot(alike);
                        if (alike && (tid & 63) == __builtin_ctzll(same)) {
                            atomicAdd(&s.pcnt[bin], (uint32_t)__popcll(same));
                            atomicAdd(&s.psum[bin], (unsigned long long)(w * __popcll(same)));
                        }
                        left = !alike;
                    }
            if (!left) return;
            atomicAdd(&s.pcnt[bin], 1u);
            atomicAdd(&s.psum[bin], (unsigned long long)w);
        });
        __syncthreads();
        BinPair p;
        bin_prefix(s.pcnt, s.psum, c0, w0, p, s);
        find_bin(p, by_count, x, s);
        __syncthreads();
        n = s.pcnt[s.f];
        lo += (uint64_t)s.f << sh;
        hi = min(hi, lo + ((1ull << sh) - 1));
        __syncthreads();
    }
}

// The token at which the running count or weight crosses x, by comparison of the few in [lo, hi].
template <class M>
__device__ __forceinline__ void pick(uint64_t lo, uint64_t hi, bool by_count, uint64_t x, const M& tokens, LastShared& s) {
    const int tid = threadIdx.x;
    tokens(lo, hi, [&](uint64_t, float l, int i, uint64_t w) {
        const int e = atomicAdd(&s.ne, 1);
        s.el[e] = l;
        s.ei[e] = i;
        s.ew[e] = w;
    });
    __syncthreads();
    const int ne = s.ne;
    if (tid < ne) {
        uint64_t before = by_count ? s.before_cnt : s.before_sum, bsum = s.before_sum;
        const float l = s.el[tid];
        const int id = s.ei[tid];
#pragma unroll 8
        for (int e = 0; e < ne; ++e) {
            const float le = s.el[e];
            const int ie = s.ei[e];
            const uint64_t we = s.ew[e];
            const bool first = (le > l) | ((le == l) & (ie < id));
            before += first ? (by_count ? 1 : we) : 0;
            bsum += first ? we : 0;
        }
        const uint64_t mine = by_count ? 1 : s.ew[tid];
        if (before <= x && x < before + mine) s.rl = l, s.ri = id, s.through = bsum + s.ew[tid];
    }
    __syncthreads();
}

// The same among the collected tokens.
template <int PER, bool LINE>
__device__ __forceinline__ void cross(const LastRegs<PER, LINE>& r, int shift, bool by_count, uint64_t x, LastShared& s) {
    const int tid = threadIdx.x;
    BinPair p;
#pragma unroll
    for (int e = 0; e < kFine / kRowThreads; ++e) {
        const int i = tid * (kFine / kRowThreads) + e;
        p.c[e] = s.cnt[i];
        p.ws[e] = s.sum[i];
        p.cb[e] = e ? p.cb[e - 1] + p.c[e - 1] : s.base_cnt[tid];
        p.wb[e] = e ? p.wb[e - 1] + p.ws[e - 1] : s.base_sum[tid];
    }
    find_bin(p, by_count, x, s);
    if (tid == 0) {
        s.ne = 0;
        s.lo = ~0ull;
        s.hi = 0;
    }
    __syncthreads();
    const int f = s.f;
    const OfBin<PER, LINE> tokens{r, f, shift};
    uint64_t lo = 0, hi = ~0ull;
    if (s.cnt[f] > kLast) {
        unsigned long long first = ~0ull, last = 0;
        tokens(lo, hi, [&](uint64_t c, float, int, uint64_t) {
            first = min(first, (unsigned long long)c);
            last = max(last, (unsigned long long)c);
        });
        for (int o = 32; o; o >>= 1) {
            first = min(first, __shfl_xor(first, o));
            last = max(last, __shfl_xor(last, o));
        }
        if ((tid & 63) == 0) {
            atomicMin(&s.lo, first);
            atomicMax(&s.hi, last);
        }
        __syncthreads();
        lo = s.lo;
        hi = s.hi;
        narrow(s.cnt[f], lo, hi, by_count, x, tokens, s);
    }
    pick(lo, hi, by_count, x, tokens, s);
}

// The three crossings and the token. Z: the weight of all (cut: of which top-k
// leaves some out), Sm of what min-p keeps; at(by_count, x) finds a crossing.
template <class At>
__device__ __forceinline__ void finish(const SampleArgs& a, int b, const RowParams& rp, float m, uint64_t Z, uint64_t Sm,
                                       bool cut, At at, LastShared& s) {
    const int tid = threadIdx.x;
    const double scale = __builtin_ldexp(1.0, a.shift);
#pragma unroll 1
    for (int step = 0; step < 3; ++step) {  // top-k, top-p, the draw
        uint64_t x;
        if (step == 0) {
            if (!cut) continue;
            x = (uint64_t)rp.topk - 1;
        } else if (step == 1) {
            const uint64_t target = topp_target(rp.topp, Z);
            if (rp.topp >= 1.0 || target >= Z) continue;
            x = target - 1;
        } else {
            Z = min(Z, Sm);
            x = draw_target(rp.u, Z);
        }
        at(step == 0, x);
        if (step < 2) Z = min(Z, (uint64_t)s.through);
    }
    if (tid == 0) {
        a.token[b] = s.ri;
        if (a.prob) a.prob[b] = (float)(weight(s.rl, m, rp.inv_t) / ((double)Z / scale));
    }
}

// A row of which more than kCand tokens are in the bins of the crossings (thousands of one value, or more than a
// million logits), by one workgroup: the bins' prefix says in which bin a crossing is and a search over all values
// from which to which logit that reaches; then parts of it as above, each a pass over the row, 20 to 60 us a pass of
// 262144. With top-p, 262144 logits rounded to quarters 206 us, all alike 372; 48 rows of 128256, 172 and 255.
__device__ __forceinline__ void sample_over(const SampleArgs& a, int b, const RowParams& rp, const RowWork& rw,
                                            const RowRange& rr, uint64_t Z, uint64_t Sm, bool cut, LastShared& s) {
    static_assert(kCoarse == kRowThreads, "a bin per thread");
    const int tid = threadIdx.x, bits = 62 - a.shift;
    const uint32_t* cnt = rw.cnt + kCoarse;
    const unsigned long long* sum = rw.sum + kCoarse;
    const OfRow tokens{a.logits + b * a.ld, a.V, a.shift, rr.m, rp.inv_t, s.line};
    // The largest key of bin f or a later one (the row's own from f = 0 on).
    auto edge = [&](int f) {
        uint32_t in = key_of(-__builtin_inff()), out = key_of(rr.m);
        if (f == 0) return out;
        while (out - in > 1) {
            const uint32_t k = in + (out - in) / 2;
            const double x = x_of(logit_of(k), rr, rp.inv_t);
            if (!(x < rr.end) || (int)place_of(x, rr) >= f)
                in = k;
            else
                out = k;
        }
        return in;
    };
    finish(a, b, rp, rr.m, Z, Sm, cut, [&](bool by_count, uint64_t x) {
        const uint64_t b0 = by_count ? cnt[tid] : sum[tid], b1 = by_count ? cnt[tid + 1] : sum[tid + 1];
        if (b0 <= x && x < b1) s.f = tid, s.before_cnt = cnt[tid], s.before_sum = sum[tid];
        if (tid == 0) s.ne = 0;
        __syncthreads();
        const int f = s.f;
        const uint32_t e = edge(f + (tid & 1));
        uint64_t lo = (uint64_t)~(uint32_t)__builtin_amdgcn_readlane((int)e, 0) << bits;
        const uint32_t least = max((uint32_t)__builtin_amdgcn_readlane((int)e, 1) + 1, key_of(rr.low));
        uint64_t hi = (uint64_t)~least << bits | ((1u << bits) - 1);
        narrow(cnt[f + 1] - cnt[f], lo, hi, by_count, x, tokens, s);
        pick(lo, hi, by_count, x, tokens, s);
    }, s);
}

// The token from what was collected.
__device__ __forceinline__ void sample_collected(const SampleArgs& a, int b, const RowParams& rp, LastShared& s) {
    const int tid = threadIdx.x, lane = tid & 63;
    const RowWork rw = row_work(a, b);
    const RowRange rr = row_range(a, rw, rp, lane);
    if (rr.done) {
        if (tid == 0) {
            const bool none = rr.m == -__builtin_inff();
            a.token[b] = none ? -1 : rr.at;
            if (a.prob) a.prob[b] = rr.m != rr.m ? rr.m : (none ? 0.0f : 1.0f);
        }
        return;
    }
    const uint32_t n = *rw.n, over = *rw.over;
    const uint32_t all = rw.cnt[2 * kCoarse];
    uint64_t Z = rw.sum[2 * kCoarse], Sm = 0;
    for (int g = lane; g < a.pieces; g += 64) Sm += rw.minp[g];
    const double scale = __builtin_ldexp(1.0, a.shift);
    for (int o = 32; o; o >>= 1) Sm += __shfl_xor((unsigned long long)Sm, o);
    const bool cut = (uint32_t)rp.topk < all;
    if (over) return sample_over(a, b, rp, rw, rr, Z, Sm, cut, s);
    if (n <= kLast) {
        // Few: each token's place among all, hence what comes before it, at once.
        const uint32_t* cnt = rw.cnt + kCoarse;
        const unsigned long long* sum = rw.sum + kCoarse;
        uint32_t bc = 0;
        uint64_t bs = 0, own = 0;
        float l = 0.0f;
        int id = 0, bin = 0;
        if (tid < (int)n) {
            l = rw.cl[tid];
            id = rw.ci[tid];
            bin = (int)rw.cp[tid];
            own = rw.cw[tid];
            s.el[tid] = l;
            s.ei[tid] = id;
            s.ew[tid] = own;
            s.cnt[tid] = bin;
            bc = cnt[bin];
            bs = sum[bin];
        }
        __syncthreads();
        if (tid < (int)n)
#pragma unroll 8
            for (int e = 0; e < (int)n; ++e) {
                const float le = s.el[e];
                const int ie = s.ei[e];
                const bool first = ((int)s.cnt[e] == bin) & ((le > l) | ((le == l) & (ie < id)));
                const uint64_t we = s.ew[e];
                bc += first ? 1 : 0;
                bs += first ? we : 0;
            }
        if (cut) {
            if (tid < (int)n && bc == (uint32_t)rp.topk - 1) s.through = bs + own;
            __syncthreads();
            Z = s.through;
        }
        if (rp.topp < 1.0) {
            const uint64_t target = topp_target(rp.topp, Z);
            if (target < Z) {
                __syncthreads();
                if (tid < (int)n && bs < target && target <= bs + own) s.through = bs + own;
                __syncthreads();
                Z = min(Z, (uint64_t)s.through);
            }
        }
        Z = min(Z, Sm);
        const uint64_t x = draw_target(rp.u, Z);
        if (tid < (int)n && bs <= x && x < bs + own) {
            a.token[b] = id;
            if (a.prob) a.prob[b] = (float)(weight(l, rr.m, rp.inv_t) / ((double)Z / scale));
        }
        return;
    }
    LastRegs<kPer, false> r;
    float place[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        const int e = tid + q * kRowThreads;
        place[q] = -1.0f;
        r.w[q] = 0;
        if (e < (int)n) {
            place[q] = rw.cp[e];
            r.w[q] = rw.cw[e];
            r.l[q] = rw.cl[e];
            r.i[q] = rw.ci[e];
        }
    }
    const uint32_t bc = rw.cnt[kCoarse + tid];
    const uint64_t bs = rw.sum[kCoarse + tid];
    if (tid < kCoarse / 32) s.want[tid] = rw.want[tid];
#pragma unroll
    for (int e = 0; e < kFine / kRowThreads; ++e) {
        s.cnt[tid + e * kRowThreads] = 0;
        s.sum[tid + e * kRowThreads] = 0;
    }
    __syncthreads();
    // The place of each collected bin among them.
    auto rank = [&](int bin) {
        int k = __popc(s.want[bin >> 5] & ((1u << (bin & 31)) - 1));
        for (int i = 0; i < (bin >> 5); ++i) k += __popc(s.want[i]);
        return k;
    };
    int slots = 0;
    for (int i = 0; i < kCoarse / 32; ++i) slots += __popc(s.want[i]);
    const int F = kFine / slots & ~1;  // (a thread's two fine bins are of one collected one)
    if (s.want[tid >> 5] >> (tid & 31) & 1) {
        const int k = rank(tid);
        s.base_cnt[k] = bc;
        s.base_sum[k] = bs;
    }
    r.no_bins();
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        if (place[q] < 0.0f) continue;
        const int bin = (int)place[q];
        const int f = rank(bin) * F + min((int)((place[q] - (float)bin) * (float)F), F - 1);
        r.set_bin(q, f);
        atomicAdd(&s.cnt[f], 1u);
        atomicAdd(&s.sum[f], r.w[q]);
    }
    __syncthreads();
    BinPair p;
    bin_prefix(s.cnt, s.sum, 0, 0, p, s);
    {
        constexpr int E = kFine / kRowThreads;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            s.pcnt[E * tid + e] = p.cb[e];
            s.psum[E * tid + e] = p.wb[e];
        }
        __syncthreads();
        // From the sum over the collected bins to the one over the row's.
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int k = (E * tid + e) / F;
            if (k >= slots) continue;  // (holds nothing)
            p.cb[e] += s.base_cnt[k] - s.pcnt[k * F];
            p.wb[e] += s.base_sum[k] - s.psum[k * F];
        }
    }
    __syncthreads();
    s.base_cnt[tid] = p.cb[0];
    s.base_sum[tid] = p.wb[0];
    finish(a, b, rp, rr.m, Z, Sm, cut, [&](bool by_count, uint64_t x) { cross(r, a.shift, by_count, x, s); }, s);
}

// A row by one workgroup, PER logits of it in each thread's registers: the fine
// histogram over the whole range at once. One launch, bound by its chain of barriers:
// 4096 logits with cuts 13 us, 16384 21 (the four launches above 24),
// 256 such rows 24 (48).
template <int PER>
__device__ __forceinline__ void sample_small(const SampleArgs& a, int b, const RowParams& rp, LastShared& s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* row = a.logits + b * a.ld;
    LastRegs<PER, true> r;
    r.i[0] = tid;
    float m = -__builtin_inff(), lo = __builtin_inff();
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int i = tid + q * kRowThreads;
        r.l[q] = i < a.V ? row[i] : -__builtin_inff();
        if (i < a.V && ahead(r.l[q], i, m, at)) m = r.l[q], at = i;
        if (r.l[q] > -__builtin_inff()) lo = fminf(lo, r.l[q]);
    }
    for (int o = 32; o; o >>= 1) {
        const float u = __shfl_xor(m, o);
        const int ui = __shfl_xor(at, o);
        if (ahead(u, ui, m, at)) m = u, at = ui;
        lo = fminf(lo, __shfl_xor(lo, o));
    }
    if (lane == 0) s.el[wave] = m, s.ei[wave] = at, s.el[64 + wave] = lo;
#pragma unroll
    for (int e = 0; e < kFine / kRowThreads; ++e) {
        s.cnt[tid + e * kRowThreads] = 0;
        s.sum[tid + e * kRowThreads] = 0;
    }
    __syncthreads();
    for (int i = 0; i < kRowThreads / 64; ++i) {
        if (ahead(s.el[i], s.ei[i], m, at)) m = s.el[i], at = s.ei[i];
        lo = fminf(lo, s.el[64 + i]);
    }
    if (m != m || m == -__builtin_inff() || rp.topk == 1) {
        if (tid == 0) {
            const bool none = m == -__builtin_inff();
            a.token[b] = none ? -1 : at;
            if (a.prob) a.prob[b] = m != m ? m : (none ? 0.0f : 1.0f);
        }
        return;
    }
    const double scale = __builtin_ldexp(1.0, a.shift);
    const float end = weightless(a);
    const float bins = (float)kFine / fmaxf(fminf((float)(((double)m - (double)lo) * rp.inv_t), end), 1e-30f);
    uint64_t Z = 0, Sm = 0;
    uint32_t all = 0;
    r.no_bins();
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const double x = r.l[q] == m ? 0.0 : ((double)m - (double)r.l[q]) * rp.inv_t;
        r.w[q] = 0;
        if (!(x < end)) continue;
        const double w = exp(-x);
        r.w[q] = fixed(w, scale);
        const int f = min((int)((float)x * bins), kFine - 1);
        r.set_bin(q, f);
        Z += r.w[q];
        if (w >= rp.minp) Sm += r.w[q];
        ++all;
        atomicAdd(&s.cnt[f], 1u);
        atomicAdd(&s.sum[f], r.w[q]);
    }
    for (int o = 32; o; o >>= 1) {
        Z += __shfl_xor((unsigned long long)Z, o);
        Sm += __shfl_xor((unsigned long long)Sm, o);
        all += __shfl_xor(all, o);
    }
    __syncthreads();  // and every wave has read el
    if (lane == 0) s.psum[wave] = Z, s.psum[64 + wave] = Sm, s.pcnt[wave] = all;
    BinPair p;
    bin_prefix(s.cnt, s.sum, 0, 0, p, s);
    s.base_cnt[tid] = p.cb[0];
    s.base_sum[tid] = p.wb[0];
    Z = Sm = 0;
    all = 0;
    for (int i = 0; i < kRowThreads / 64; ++i) Z += s.psum[i], Sm += s.psum[64 + i], all += s.pcnt[i];
    finish(a, b, rp, m, Z, Sm, (uint32_t)rp.topk < all, [&](bool by_count, uint64_t x) { cross(r, a.shift, by_count, x, s); }, s);
}
template <int PER>
__global__ void __launch_bounds__(kRowThreads) sample_small_kernel(SampleArgs a) {
    __shared__ LastShared sh;
    const int b = blockIdx.x;
    sample_small<PER>(a, b, row_params(a, b), sh);
}

// One workgroup per row: the token.
__global__ void __launch_bounds__(kRowThreads) sample_last_kernel(SampleArgs a) {
    __shared__ LastShared sh;
    const int b = blockIdx.x;
    sample_collected(a, b, row_params(a, b), sh);
}
}  // namespace

}  // namespace alv

using namespace alv;

namespace alv {
namespace {
// Short rows, as many logits as fit the registers of one workgroup.
constexpr int kSmall = 16 * kRowThreads;
int sample_pieces(int V) { return V <= kSmall ? 0 : (V + kPiece - 1) / kPiece; }
template <class F>
void small_row(int V, F go) {
    if (V <= 4 * kRowThreads)
        go(sample_small_kernel<4>);
    else if (V <= 8 * kRowThreads)
        go(sample_small_kernel<8>);
    else
        go(sample_small_kernel<16>);
}
}  // namespace
}  // namespace alv

extern "C" uint64_t alv_sample_workspace(int B, int V) {
    if (B < 1 || V < 1) return 0;
    const int pieces = sample_pieces(V);
    return pieces ? (uint64_t)B * row_bytes(pieces) : 0;
}

extern "C" int alv_sample(const float* logits, int64_t ld, int B, int V, const float* u, const float* temperature_dev,
                          float temperature, const int32_t* top_k_dev, int top_k, const float* top_p_dev, float top_p,
                          const float* min_p_dev, float min_p, int32_t* token, float* prob, void* workspace,
                          uint64_t workspace_bytes, void* stream) {
    if (B < 0 || V < 1 || ld < V) return fail(ALV_ERR_ARG, "bad logits shape B=%d vocab=%d ld=%lld", B, V, (long long)ld);
    if (B == 0) return ALV_OK;
    if (!logits || !u || !token) return fail(ALV_ERR_ARG, "null pointer");
    if (V > 1 << 24 || B > 65535 || (int64_t)B * sample_pieces(V) > 1 << 23)
        return fail(ALV_ERR_RANGE, "%d rows of %d logits (at most 65535 rows, 2^24 logits in one, 2^35 in all)", B, V);
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
    a.pieces = sample_pieces(V);
    const uint64_t need = alv_sample_workspace(B, V);
    if (need && (!workspace || workspace_bytes < need))
        return fail(ALV_ERR_ARG, "workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
                    (unsigned long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(ALV_ERR_ALIGN, "workspace needs 16-byte alignment");
    a.work = static_cast<unsigned char*>(workspace);
    const hipStream_t st = (hipStream_t)stream;
    if (a.pieces) {
        const dim3 grid(a.pieces, B);
        hipLaunchKernelGGL(sample_top_kernel, grid, dim3(kPieceThreads), 0, st, a);
        hipLaunchKernelGGL(sample_hist_kernel, grid, dim3(kPieceThreads), 0, st, a);
        hipLaunchKernelGGL(sample_collect_kernel, grid, dim3(kPieceThreads), 0, st, a);
    }
    if (a.pieces)
        hipLaunchKernelGGL(sample_last_kernel, dim3(B), dim3(kRowThreads), 0, st, a);
    else
        small_row(V, [&](auto k) { hipLaunchKernelGGL(k, dim3(B), dim3(kRowThreads), 0, st, a); });
    return hip_check(hipGetLastError(), "sample kernels' launch");
}
