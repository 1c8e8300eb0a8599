// Attention of the newest tokens of a batch of sequences over a paged KV cache.
//
// out = sum_p w_p v_p / sum_p w_p with w_p = exp(scale q.k_p - m), the maximum m
// and both sums kept running in float32 over one pass of K and V. Both kernels
// compute the transposes, S' = K Q' and O' = V' P': a lane then has one row's
// scores for several positions, which as bf16 are the next product's operand as
// they stand, and a row's maximum and sum are one lane's (pair's, group's) own.
//
// Two kernels, by how many rows (tokens times q heads of the group) a sequence
// brings: up to 64 at D <= 128, 32 at 256, 16 at 512 (in a small batch 16, at 512 15)
// stream K and V past resident rows, bound by memory; more rows share tiles of K
// and V, bound by the matrix cores. The host plans with max_q (or the average) and
// the kernels sort the sequences by their own counts, so a batch may hold both
// kinds; a small batch with more rows is the tile kernel's alone.
#include <limits.h>

#include <algorithm>
#include <atomic>

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
    int64_t row_limit;  // sequences of more rows (tokens times q heads per kv head) are not this launch's
    int max_tiles;      // tiles of all sequences, per kv head, at most
    int max_items;      // tiles (times kv heads) that may be split: no more than slots; 0: none
    int slots;          // parts that run at once
    int* tab;           // for the merge: how many tiles, then kTabInts for each
    float* part;
};

typedef short s16x4 __attribute__((__vector_size__(4 * sizeof(short))));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// ---- the matrix products' operands ---------------------------------------------------
//
// Scores are computed transposed, S^T = K Q^T (A = 16 positions, B = 16 rows of
// q), so that a lane holds one row's scores and the softmax needs no exchange
// between lanes but for a new maximum; and the output transposed, O^T = V^T P^T,
// whose operand P^T is those scores' registers as they are. V^T comes out of LDS
// through the transposing read (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16
// values, lane i gets column i).

// One 16-byte piece per lane from memory to LDS, no register in between. The
// compiler would wait for it before every LDS read, so it is written out; the
// waits are wait_vm's.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(voff), "s"(r), "s"(soff), "s"(lds)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// At most N of this wave's loads are still in flight.
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A buffer over [base, base + bytes), the same for the whole wave.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t wave_rsrc(const uint16_t* base, uint32_t bytes) {
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32));
    return make_rsrc(reinterpret_cast<const void*>(((uint64_t)hi << 32) | lo), __builtin_amdgcn_readfirstlane((int)bytes));
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p);
}

// The value, as if it were new here: what is computed from it is computed again
// in each turn of a loop rather than kept in registers throughout.
__device__ __forceinline__ uint32_t here(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// The larger (sum) of a value over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_groups(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    auto h = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const uint32_t h0 = h[0], h1 = h[1];
    v = fmaxf(__builtin_bit_cast(float, h0), __builtin_bit_cast(float, h1));
    const uint32_t c = __builtin_bit_cast(uint32_t, v);
    auto q = __builtin_amdgcn_permlane16_swap(c, c, false, false);
    const uint32_t q0 = q[0], q1 = q[1];
    return fmaxf(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1));
}
__device__ __forceinline__ float sum_groups(float v) {
    v += __shfl_xor(v, 32);
    return v + __shfl_xor(v, 16);
}

// Two float32 as bf16, to nearest even (v_cvt_pk_bf16_f32).
__device__ __forceinline__ s16x4 pack4(float a, float b, float c, float d) {
    typedef __bf16 bf16x4 __attribute__((__vector_size__(4 * sizeof(__bf16))));
    bf16x4 v;
    v[0] = (__bf16)a;
    v[1] = (__bf16)b;
    v[2] = (__bf16)c;
    v[3] = (__bf16)d;
    return __builtin_bit_cast(s16x4, v);
}

// LDS pieces of a row are stored at (piece ^ swizzle of the row): the 16 lanes
// that read K at once (16 rows, the same piece) and the 32 that read V (8 rows of
// two pieces, or 4 of four) then fall on different banks.
template <int D>
__device__ __forceinline__ int k_swz(int row) {
    return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swz(int row) {
    return D == 64 ? ((row >> 1) & 1) * 4 + ((row >> 2) & 1) * 2 : (row & 3) * 4 + ((row >> 2) & 1) * 2;
}

// The offset of piece c of a row as what is xored into a swizzled offset (the
// swizzles stay within 16 pieces) and what is added.
template <int D>
__device__ __forceinline__ constexpr uint32_t piece(int c) {
    return (c & (D == 64 ? 7 : 15)) * 16;
}
template <int D>
__device__ __forceinline__ constexpr uint32_t piece_far(int c) {
    return (c & ~(D == 64 ? 7 : 15)) * 16;
}

__device__ __forceinline__ s16x4 read_tr(const unsigned char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p));
}

// Whether a row at position t sees position p.
__device__ __forceinline__ bool sees(const PagedAttnArgs& a, int p, int t) {
    return p <= t && (a.window <= 0 || p > t - a.window || p < a.sinks);
}

// 1 / l of a row, 0 for one that saw nothing.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

__device__ __forceinline__ void store4(uint16_t* dst, f32x4 v, float inv) {
    *reinterpret_cast<s16x4*>(dst) = pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
}

constexpr float kNoMax = -3.0e38f;  // running maximum of a row that has seen nothing
constexpr float kMinScale = 1e-37f;  // -infinity times it is -infinity, a score times it 0
constexpr float kLog2e = 1.44269504088896340736f;
// A row's reference stays while its scores exceed it by no more than this many
// powers of two: weights up to 2^8 lose nothing in float32 or bf16, and most
// blocks then need neither a maximum over the lanes nor a rescaled output.
constexpr float kSlack = 8.0f;

// One row's part (maximum, sum, output: RW values per lane) over units u0 .. u1 - 1
// of its tile, by one wave in plain float32 steps. The matrix products give a
// value of V that is infinite or NaN to every row they compute, seen or not (0
// times it is NaN, and no later step makes that a number again); a wave that ends
// with such an output does its rows again with this.
template <int D>
__device__ void plain_row(const PagedAttnArgs& a, int seq, int kvh, const uint16_t* q, int pos, int us, int ulo, int unit,
                          int u0, int u1, int lane, float (&acc)[D / 64], float& m, float& l) {
    constexpr int RW = D / 64;
    const float c = fmaxf(a.scale * kLog2e, kMinScale);
    m = kNoMax;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < RW; ++e) acc[e] = 0.0f;
    for (int u = u0; u < u1; ++u) {
        const int base = (u < us ? u : u - us + ulo) * unit;
        for (int pb = base; pb < base + unit; pb += 64) {
            const int p = pb + lane;
            int page = -1;
            if (p < base + unit && sees(a, p, pos)) page = page_of(a.b, seq, p);
            float s = -__builtin_inff();
            const int64_t off = (((int64_t)kvh << a.b.shift) + (p & ((1 << a.b.shift) - 1))) * D;
            if (page >= 0) {
                const u32x4* k = reinterpret_cast<const u32x4*>(a.kpages + page * a.k_stride + off);
                s = 0.0f;
                for (int i = 0; i < D / 8; ++i) {
                    const u32x4 kv = k[i], qv = reinterpret_cast<const u32x4*>(q)[i];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t kw = kv[e], qw = qv[e];
                        s = __builtin_fmaf(bf16_bits_to_f32(kw & 0xFFFFu), bf16_bits_to_f32(qw & 0xFFFFu), s);
                        s = __builtin_fmaf(bf16_bits_to_f32(kw >> 16), bf16_bits_to_f32(qw >> 16), s);
                    }
                }
            }
            float top = s;
            for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
            const float mn = fmaxf(m, top * c), fac = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            float w = page >= 0 ? __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -mn)) : 0.0f, sum = w;
            for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
            l = l * fac + sum;
#pragma unroll
            for (int e = 0; e < RW; ++e) acc[e] *= fac;
            for (uint64_t left = __ballot(page >= 0); left; left &= left - 1) {
                const int j = __builtin_ctzll(left), pj = pb + j;
                const float wj = __shfl(w, j);
                const uint16_t* v = a.vpages + __shfl(page, j) * a.v_stride +
                                    (((int64_t)kvh << a.b.shift) + (pj & ((1 << a.b.shift) - 1))) * D + RW * lane;
#pragma unroll
                for (int e = 0; e < RW; ++e) acc[e] = __builtin_fmaf(wj, bf16_bits_to_f32(v[e]), acc[e]);
            }
        }
    }
}

// ---- few rows: a workgroup streams positions -------------------------------------------
//
// A tile is up to 16 QT rows of one (sequence, kv head): rows are (token, q head
// of the group), so the heads that share K and V share the reads. The work, all
// tiles times their units of positions, is one line that the workgroups cut into
// equal parts: lengths may differ by any factor, and no workgroup waits for the
// longest sequence. A workgroup's part holds whole tiles, finished here, and at
// most two cut ones, whose partial results go to its two places in the workspace
// for the merge.
//
// A wave streams blocks of 16 positions of its own (wave w of NW: blocks w, w +
// NW, ...) through a ring of LDS buffers that only it uses: no barrier until the
// tile's end, and 64 to 128 KiB in flight per CU, which is what the memory needs
// to run at its rate. 16 positions never cross a page.
//
// Bound by memory where there is work enough: 64 sequences of 1000 to 4000
// positions, one token each, read K and V at 4.8 TB/s (32 q heads of 64 on 8: 70
// us), 5.2 (16 of 128 on 8: 128 us), 5.6 (16 of 256 on 8: 240 us) and 4.0 (16 of
// 512 on 1: 85 us); a large copy moves 4.9 on this card, reads alone more. One
// sequence of 300 positions is two launches, 14 us with the host's part.

// A sequence's place in the line, per lane of the scan.
struct RowsSeq {
    int first, n, len;
    int tiles;        // row tiles (of each kv head)
    int us, ulo, nu;  // units of first tokens; first unit of the window; units in all
};

constexpr int rows_waves(int D) { return D == 512 ? 2 : (D == 64 ? 8 : 4); }
constexpr int rows_stage(int D) { return 64 * D; }  // bytes of 16 positions' K and V
constexpr int rows_stages(int D) { return 131072 / (rows_waves(D) * rows_stage(D)); }
constexpr int rows_unit(int D) { return 16 * rows_waves(D); }
// The waves' outputs at a tile's end, rows padded to spread over the banks.
constexpr int rows_out_ld(int D) { return D + 4; }
// Whether q's operands stay in LDS rather than registers: where they and the
// output take more than half of a wave's 256 (the rest would spill).
constexpr bool rows_q_lds(int D, int QT) { return QT * D > 256; }
constexpr int rows_lds(int D, int QT) {
    const int ring = rows_waves(D) * rows_stages(D) * rows_stage(D);
    const int outs = rows_waves(D) * 16 * QT * (rows_out_ld(D) * 4);
    return (ring > outs ? ring : outs) + 2 * rows_waves(D) * 16 * QT * 4 + (rows_q_lds(D, QT) ? 32 * QT * D : 0) + 16;
}
constexpr int rows_mls(int D, int QT) {  // where the waves' maxima and sums stand; q behind them
    return rows_lds(D, QT) - 16 - 2 * rows_waves(D) * 16 * QT * 4 - (rows_q_lds(D, QT) ? 32 * QT * D : 0);
}
// Floats of one workspace place: outputs, maxima, sums.
constexpr int rows_part(int D, int QT) { return 16 * QT * (D + 2); }

constexpr int kPartsPerTile = 64;

struct Scan {
    RowsSeq s;          // this lane's sequence
    uint64_t incl;      // work of the sequences of this step up to and with this lane's
    uint64_t base, sum; // work before this step; of this step
    int b0;             // the step's first sequence
    uint32_t tiles;     // of the whole batch, no more than 2^31 (scan_all)
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, l);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l);
    return ((uint64_t)hi << 32) | lo;
}

template <int ROWS, int UNIT>
__device__ __forceinline__ void scan_step(const PagedAttnArgs& a, int b0, int lane, uint64_t base, Scan& sc) {
    const int b = b0 + lane;
    RowsSeq s{};
    uint64_t w = 0;
    if (b < a.b.B) {
        s.first = a.b.q_start[b];
        s.n = a.b.q_start[b + 1] - s.first;
        s.len = a.b.kv_len[b];
        const bool here = s.first >= 0 && s.n > 0 && (int64_t)s.first + s.n <= a.b.T;
        const int64_t rows = here ? (int64_t)s.n * a.g : 0;
        if (here && rows <= a.row_limit) {
            s.tiles = (int)((rows + ROWS - 1) / ROWS);
            if (s.n <= s.len && s.len <= a.b.max_pos) {
                const int lo = a.window > 0 ? max(0, s.len - s.n + 1 - a.window) : 0;
                s.ulo = lo / UNIT;
                s.us = min((min(a.sinks, lo) + UNIT - 1) / UNIT, s.ulo);
                s.nu = s.us + (s.len + UNIT - 1) / UNIT - s.ulo;
            } else {
                s.len = 0;  // malformed: one unit that sees nothing
                s.nu = 1;
            }
            w = (uint64_t)s.tiles * a.kv_heads * s.nu;
        }
    }
    uint64_t x = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t u = __shfl_up((unsigned long long)x, o);
        if (lane >= o) x += u;
    }
    sc.s = s;
    sc.incl = x;
    sc.base = base;
    sc.sum = lane_u64(x, 63);
    sc.b0 = b0;
}

// The first step, and the work of the whole batch.
template <int ROWS, int UNIT>
__device__ __forceinline__ uint64_t scan_all(const PagedAttnArgs& a, int lane, Scan& sc) {
    scan_step<ROWS, UNIT>(a, 0, lane, 0, sc);
    uint64_t total = sc.sum;
    uint32_t tiles = sc.s.nu ? min(sc.s.tiles, kPartsPerTile) : 0;
    for (int b0 = 64; b0 < a.b.B; b0 += 64) {
        Scan t;
        scan_step<ROWS, UNIT>(a, b0, lane, 0, t);
        total = min(total + t.sum, (uint64_t)1 << 62);  // (sequences that overlap: no wrap)
        tiles = min(tiles + (t.s.nu ? min(t.s.tiles, kPartsPerTile) : 0), 1u << 24);
    }
    for (int k = 32; k; k >>= 1) tiles += __shfl_xor(tiles, k);
    sc.tiles = uniform(min(tiles, 1u << 24) * (uint32_t)min(a.kv_heads, 64));
    return total;
}

__device__ __forceinline__ uint64_t div32(uint64_t a, uint64_t b) {  // (32 bits take a third of the steps)
    return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b;
}

struct Found {
    RowsSeq s;
    int seq, kvh, rt;
    int u;            // unit in the tile
    uint64_t tile0;   // the tile's place in the line
};

// The tile and unit at place x of the line (x < total; calls with x rising).
template <int ROWS, int UNIT>
__device__ __forceinline__ Found scan_find(const PagedAttnArgs& a, int lane, Scan& sc, uint64_t x) {
    while (x >= sc.base + sc.sum) scan_step<ROWS, UNIT>(a, sc.b0 + 64, lane, sc.base + sc.sum, sc);
    const uint64_t m = __ballot(sc.base + sc.incl > x);
    const int l = __builtin_ctzll(m);
    Found f;
    f.seq = sc.b0 + l;
    f.s.first = __builtin_amdgcn_readlane(sc.s.first, l);
    f.s.n = __builtin_amdgcn_readlane(sc.s.n, l);
    f.s.len = __builtin_amdgcn_readlane(sc.s.len, l);
    f.s.tiles = __builtin_amdgcn_readlane(sc.s.tiles, l);
    f.s.us = __builtin_amdgcn_readlane(sc.s.us, l);
    f.s.ulo = __builtin_amdgcn_readlane(sc.s.ulo, l);
    f.s.nu = __builtin_amdgcn_readlane(sc.s.nu, l);
    const uint64_t seq_work = (uint64_t)f.s.tiles * a.kv_heads * f.s.nu;
    const uint64_t start = sc.base + lane_u64(sc.incl, l) - seq_work;
    const uint64_t in = x - start;
    const uint64_t tile = div32(in, (uint32_t)f.s.nu);
    f.u = uniform((int)(in - tile * f.s.nu));
    f.tile0 = start + tile * f.s.nu;
    f.kvh = uniform((int)((uint32_t)tile / (uint32_t)f.s.tiles));
    f.rt = uniform((int)((uint32_t)tile - (uint32_t)f.kvh * f.s.tiles));
    return f;
}

// The line of `total` units cut into n parts, the first r of them a unit longer.
struct Cut {
    uint64_t q;
    uint32_t r, n;
    __device__ __forceinline__ uint64_t begin(uint32_t w) const { return q * w + min(w, r); }
    __device__ __forceinline__ uint32_t part_of(uint64_t x) const {  // that holds place x
        const uint64_t longer = (q + 1) * r;
        return (uint32_t)(x < longer ? div32(x, q + 1) : r + div32(x - longer, q));
    }
};
__device__ __forceinline__ Cut make_cut(uint64_t total, uint32_t n) {
    Cut c;
    c.n = n;
    c.q = n ? div32(total, n) : 0;
    c.r = (uint32_t)(total - c.q * n);
    return c;
}

// At most kPartsPerTile parts per tile on average: the merge reads them all (one
// token over 8000 positions on one kv head of 512: 250 parts 117 us, 125 40, 64 33).
__device__ __forceinline__ uint32_t part_count(uint64_t total, const Scan& sc, int grid) {
    return (uint32_t)min(min((uint64_t)grid, (uint64_t)sc.tiles * kPartsPerTile), total);
}

template <int D, int QT>
__global__ void __launch_bounds__((64 * rows_waves(D)), 2) attn_paged_rows_kernel(PagedAttnArgs a) {
    constexpr int NW = rows_waves(D), NS = rows_stages(D), UNIT = rows_unit(D), ROWS = 16 * QT;
    constexpr int NC = D / 8;             // 16-byte pieces of a row
    constexpr int NI = D / 32;            // loads of 64 pieces for 16 positions of K (of V)
    constexpr int HALF = 32 * D;          // bytes of 16 positions' K
    constexpr int RPL = 512 / D;          // rows of one load
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, G = lane >> 4;
    Scan sc;
    const uint64_t total = scan_all<ROWS, UNIT>(a, lane, sc);
    const Cut cut = make_cut(total, part_count(total, sc, gridDim.x));
    if (blockIdx.x >= cut.n) return;
    uint64_t x = cut.begin(blockIdx.x);
    const uint64_t end = cut.begin(blockIdx.x + 1);

    unsigned char* ring = smem + wave * NS * rows_stage(D);
    const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_addr(ring));
    float* mls = reinterpret_cast<float*>(smem + rows_mls(D, QT));  // [wave][max | sum][row]
    int* odds = reinterpret_cast<int*>(smem + rows_lds(D, QT) - 16);
    const float c = fmaxf(a.scale * kLog2e, kMinScale);
    const int S = 1 << a.b.shift;
    // Byte offsets that stay: this lane's piece of a load (memory side), of a K
    // read and of a V read (LDS side).
    const uint32_t dma_k = (lane / NC) * (2 * D) + ((lane % NC) ^ k_swz<D>(lane / NC)) * 16;
    const uint32_t dma_v = (lane / NC) * (2 * D) + ((lane % NC) ^ v_swz<D>(lane / NC)) * 16;
    const uint32_t rd_k = col * (2 * D) + (G ^ k_swz<D>(col)) * 16;
    const int vrow = 4 * G + (col >> 2);
    const uint32_t rd_v = vrow * (2 * D) + (((col >> 1) & 1) ^ v_swz<D>(vrow)) * 16 + (col & 1) * 8;

    while (x < end) {
        const Found f = scan_find<ROWS, UNIT>(a, lane, sc, x);
        const int u0 = f.u, u1 = uniform((int)min((uint64_t)f.s.nu, u0 + (end - x)));
        x += u1 - u0;
        const int nrows = min(ROWS, f.s.n * a.g - f.rt * ROWS);
        const int nblk = f.s.len > 0 ? u1 - u0 : 0;  // this wave's blocks
        auto block_pos = [&](int j) {
            const int u = u0 + j;
            return (u < f.s.us ? u : u - f.s.us + f.s.ulo) * UNIT + 16 * wave;
        };
        // The pages of this wave's blocks, 64 at a time, one per lane.
        const int32_t* table = a.b.table + (int64_t)f.seq * a.b.ld_table;
        int pages = -1, pages0 = 0;
        uint32_t gone_bits = 0;  // by buffer: its page is missing
        auto load_pages = [&](int j0) {
            pages0 = j0;
            const int j = j0 + lane, p = block_pos(j);
            pages = j < nblk && p < f.s.len ? table[p >> a.b.shift] : -1;
            if ((unsigned)pages >= (unsigned)a.b.pages) pages = -1;
        };
        auto page_at = [&](int j) { return __builtin_amdgcn_readlane(pages, j - pages0); };
        auto issue = [&](int j) {
            if (j - pages0 >= 64) load_pages(j);
            const int page = page_at(j), p = block_pos(j);
            // Past the sequence's end, and where the page is missing, zeros arrive.
            const uint32_t bytes = page < 0 ? 0u : (uint32_t)max(0, min(16, f.s.len - p)) * (2 * D);
            const int64_t off = (((int64_t)f.kvh << a.b.shift) + (p & (S - 1))) * D;
            const __amdgpu_buffer_rsrc_t rk = wave_rsrc(a.kpages + max(page, 0) * a.k_stride + off, bytes);
            const __amdgpu_buffer_rsrc_t rv = wave_rsrc(a.vpages + max(page, 0) * a.v_stride + off, bytes);
            gone_bits = (gone_bits & ~(1u << (j % NS))) | ((uint32_t)(page < 0) << (j % NS));
            const uint32_t dst = ring_lds + (uint32_t)(j % NS) * rows_stage(D);
            // Load i brings rows RPL i .. of RPL each; the swizzles are exclusive
            // ors of the row's bits, so the lane's offset within the rows of one
            // load serves all, with the load's own bits applied.
#pragma unroll
            for (int i = 0; i < NI; ++i)
                load_lds16(rk, dma_k ^ (k_swz<D>(RPL * i) * 16), 1024 * i, dst + 1024 * i);
#pragma unroll
            for (int i = 0; i < NI; ++i)
                load_lds16(rv, dma_v ^ (v_swz<D>(RPL * i) * 16), 1024 * i, dst + HALF + 1024 * i);
        };

        // This lane's rows of q, the B operand: row col of each 16, 8 columns of each 32.
        int pos[QT];
        constexpr bool QL = rows_q_lds(D, QT);
        bf16x8 q[QL ? 1 : QT][QL ? 1 : D / 32];
        u32x4* qs = reinterpret_cast<u32x4*>(smem + rows_mls(D, QT) + 2 * NW * ROWS * 4) + lane;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int r = min(16 * t + col, nrows - 1) + f.rt * ROWS;
            const int tok = r / a.g, h = f.kvh * a.g + (r - tok * a.g);
            pos[t] = f.s.len - f.s.n + tok;
            const uint16_t* qr = a.q + (int64_t)(f.s.first + tok) * a.ld_q + h * D + 8 * G;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                if constexpr (QL) {
                    if (i % NW == wave) qs[(t * (D / 32) + i) * 64] = *reinterpret_cast<const u32x4*>(qr + 32 * i);
                } else {
                    q[t][i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(qr + 32 * i));
                }
            }
        }
        if constexpr (QL) {
            __syncthreads();
        } else {
            // Waited for here: the compiler would else wait at their first use, in
            // the loop, each time, for whatever is on its way to LDS by then.
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) asm volatile("" : "+v"(q[t][i]));
        }
        const int pos_lo = f.s.len - f.s.n + (f.rt * ROWS) / a.g;
        const int pos_hi = f.s.len - f.s.n + (f.rt * ROWS + nrows - 1) / a.g;
        f32x4 o[QT][D / 16];
        float m[QT], l[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            m[t] = kNoMax;
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) o[t][d] = f32x4{0, 0, 0, 0};
        }
        if (nblk) load_pages(0);
#pragma unroll 1
        for (int j = 0; j < min(NS, nblk); ++j) issue(j);
#pragma unroll 1
        for (int j = 0; j < nblk; ++j) {
            // Blocks j + 1 .. j + NS - 1 may be in flight.
            if (j + NS <= nblk)
                wait_vm<(NS - 1) * 2 * NI>();
            else
                wait_vm<0>();
            const unsigned char* kt = ring + (j % NS) * rows_stage(D);
            const unsigned char* vt = kt + HALF;
            f32x4 s[QT];
#pragma unroll
            for (int t = 0; t < QT; ++t) s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const bf16x8 k = __builtin_bit_cast(
                    bf16x8, *reinterpret_cast<const u32x4*>(kt + (rd_k ^ piece<D>(4 * i)) + piece_far<D>(4 * i)));
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    if constexpr (QL)
                        s[t] = mfma16x16x32(k, __builtin_bit_cast(bf16x8, qs[(t * (D / 32) + i) * 64]), s[t]);
                    else
                        s[t] = mfma16x16x32(k, q[t][i], s[t]);
                }
            }
            const int p0 = block_pos(j);
            const bool gone = (gone_bits >> (j % NS)) & 1;
            const bool masked = gone || p0 + 15 > pos_lo || (a.window > 0 && p0 <= pos_hi - a.window && p0 + 15 >= a.sinks);
            if (masked) {
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!sees(a, p0 + 4 * G + i, pos[t]) || gone) s[t][i] = -__builtin_inff();
            }
            s16x4 pw[QT];
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const float s0 = s[t][0], s1 = s[t][1], s2 = s[t][2], s3 = s[t][3];
                const float top = fmaxf(fmaxf(s0, s1), fmaxf(s2, s3));
                if (__any(__builtin_fmaf(top, c, -m[t]) > kSlack)) {
                    const float mn = fmaxf(m[t], max_groups(top) * c);
                    const float fac = __builtin_amdgcn_exp2f(m[t] - mn);
                    m[t] = mn;
                    l[t] *= fac;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) o[t][d] *= fac;
                }
                const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s0, c, -m[t]));
                const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s1, c, -m[t]));
                const float w2 = __builtin_amdgcn_exp2f(__builtin_fmaf(s2, c, -m[t]));
                const float w3 = __builtin_amdgcn_exp2f(__builtin_fmaf(s3, c, -m[t]));
                l[t] += (w0 + w1) + (w2 + w3);
                // Weights as bf16, the matrix cores' type: half a step, 2^-8
                // relative each, as much as the output's own rounding (the outputs'
                // mean error against 64 bits: 0.0021 to 0.0024, of which their own
                // rounding is 0.0017).
                pw[t] = pack4(w0, w1, w2, w3);
            }
            auto read_v = [&](int d) __attribute__((always_inline)) {
                return read_tr(vt + (rd_v ^ piece<D>(2 * d)) + piece_far<D>(2 * d));
            };
            constexpr int VB = D / 16 < 8 ? D / 16 : 8;  // V reads on their way at once
#pragma unroll
            for (int d0 = 0; d0 < D / 16; d0 += VB) {
                s16x4 v[VB];
#pragma unroll
                for (int d = 0; d < VB; ++d) v[d] = read_v(d0 + d);
                asm volatile("" ::: "memory");
#pragma unroll
                for (int d = 0; d < VB; ++d)
#pragma unroll
                    for (int t = 0; t < QT; ++t)
                        o[t][d0 + d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v[d], pw[t], o[t][d0 + d], 0, 0, 0);
            }
            // The buffer's reads are done before it is filled again.
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (j + NS < nblk) issue(j + NS);
        }

        // The waves' results: rescaled to the largest maximum and added in order.
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            l[t] = sum_groups(l[t]);
            if (G == 0) {
                mls[wave * 2 * ROWS + 16 * t + col] = m[t];
                mls[(wave * 2 + 1) * ROWS + 16 * t + col] = l[t];
            }
        }
        float odd = 0.0f;
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) odd = __builtin_fmaf(o[t][d][e], 0.0f, odd);
        if (lane == 0) odds[wave] = 0;
        if (__any(odd != 0.0f) && lane == 0) odds[wave] = 1;
        __syncthreads();  // and every wave is done with its ring
        bool again = false;
#pragma unroll
        for (int w = 0; w < NW; ++w) again |= odds[w] != 0;
        const bool whole = u0 == 0 && u1 == f.s.nu;
        float* part = a.part + (size_t)(2 * blockIdx.x + (u0 == 0 ? 1 : 0)) * rows_part(D, QT);
        if (again) {
            for (int r = wave; r < nrows; r += NW) {
                const int rr = r + f.rt * ROWS, tok = rr / a.g, h = f.kvh * a.g + (rr - tok * a.g);
                float acc[D / 64], mr, lr;
                plain_row<D>(a, f.seq, f.kvh, a.q + (int64_t)(f.s.first + tok) * a.ld_q + h * D, f.s.len - f.s.n + tok,
                             f.s.us, f.s.ulo, UNIT, u0, u1, lane, acc, mr, lr);
                const float inv = inverse(lr);
                uint16_t* dst = a.out + (int64_t)(f.s.first + tok) * a.ld_out + h * D + D / 64 * lane;
#pragma unroll
                for (int e = 0; e < D / 64; ++e) {
                    if (whole)
                        dst[e] = bf16_rne_bits(acc[e] * inv);
                    else
                        part[(size_t)r * D + D / 64 * lane + e] = acc[e];
                }
                if (!whole && lane == 0) {
                    part[ROWS * D + r] = mr;
                    part[ROWS * (D + 1) + r] = lr;
                }
            }
            __syncthreads();
            continue;
        }
        float* outs = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            float mx = kNoMax;
#pragma unroll
            for (int w = 0; w < NW; ++w) mx = fmaxf(mx, mls[w * 2 * ROWS + 16 * t + col]);
            const float fac = __builtin_amdgcn_exp2f(m[t] - mx);
            float* row = outs + (size_t)(wave * ROWS + 16 * t + col) * rows_out_ld(D) + 4 * G;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4*>(row + 16 * d) = o[t][d] * fac;
        }
        __syncthreads();
        for (int e = tid; e < nrows * (D / 4); e += 64 * NW) {
            const int r = e / (D / 4), d = 4 * (e - r * (D / 4));
            f32x4 v = *reinterpret_cast<const f32x4*>(outs + (size_t)r * rows_out_ld(D) + d);
            float mx = mls[r], ls = mls[ROWS + r];
#pragma unroll
            for (int w = 1; w < NW; ++w) {
                v += *reinterpret_cast<const f32x4*>(outs + (size_t)(w * ROWS + r) * rows_out_ld(D) + d);
                const float mw = mls[w * 2 * ROWS + r], lw = mls[(w * 2 + 1) * ROWS + r];
                const float mn = fmaxf(mx, mw);
                ls = ls * __builtin_amdgcn_exp2f(mx - mn) + lw * __builtin_amdgcn_exp2f(mw - mn);
                mx = mn;
            }
            if (whole) {
                const int rr = r + f.rt * ROWS, tok = rr / a.g, h = f.kvh * a.g + (rr - tok * a.g);
                store4(a.out + (int64_t)(f.s.first + tok) * a.ld_out + h * D + d, v, inverse(ls));
            } else {
                *reinterpret_cast<f32x4*>(part + (size_t)r * D + d) = v;
                if (d == 0) {
                    part[ROWS * D + r] = mx;
                    part[ROWS * (D + 1) + r] = ls;
                }
            }
        }
        __syncthreads();  // the ring and mls are free again
    }
}

// acc, l of n parts rescaled to the largest maximum and added in order, by one
// wave: the maxima and sums 64 parts at a time, a part per lane (ml(v) points to
// part v's maximum, its sum `gap` floats behind), then eight parts' outputs (o(v)
// points to this lane's) on their way at once.
template <int RW, class ML, class O>
__device__ __forceinline__ void join_parts(int n, int lane, ML ml, int gap, O o, float (&acc)[RW], float& mx, float& l) {
    for (int v0 = 0; v0 < n; v0 += 64) {
        const int c = min(64, n - v0);
        float m = kNoMax, s = 0.0f;
        if (lane < c) {
            const float* p = ml(v0 + lane);
            m = p[0];
            s = p[gap];
        }
        float top = m;
        for (int k = 32; k; k >>= 1) top = fmaxf(top, __shfl_xor(top, k));
        const float mn = fmaxf(mx, top), old = __builtin_amdgcn_exp2f(mx - mn);
        mx = mn;
        const float fac = lane < c ? __builtin_amdgcn_exp2f(m - mn) : 0.0f;
        l *= old;
#pragma unroll
        for (int e = 0; e < RW; ++e) acc[e] *= old;
        for (int q0 = 0; q0 < c; q0 += 8) {
            float t[8][RW];
#pragma unroll
            for (int q = 0; q < 8; ++q) __builtin_memcpy(t[q], o(v0 + min(q0 + q, c - 1)), sizeof(t[q]));
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float f = q0 + q < c ? lane_f(fac, min(q0 + q, c - 1)) : 0.0f;
                l = __builtin_fmaf(lane_f(s, min(q0 + q, c - 1)), f, l);
#pragma unroll
                for (int e = 0; e < RW; ++e) acc[e] = q0 + q < c ? __builtin_fmaf(t[q][e], f, acc[e]) : acc[e];
            }
        }
    }
}

// The cut tiles: wave (boundary, row) joins the parts of the tile in which
// boundary blockIdx.x + 1 is the first, in the order of the line.
template <int D, int QT>
__global__ void __launch_bounds__(256) attn_paged_rows_merge_kernel(PagedAttnArgs a, int grid) {
    constexpr int UNIT = rows_unit(D), ROWS = 16 * QT, RW = D / 64;
    const int lane = threadIdx.x & 63;
    const int r = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
    Scan sc;
    const uint64_t total = scan_all<ROWS, UNIT>(a, lane, sc);
    const Cut cut = make_cut(total, part_count(total, sc, grid));
    const uint32_t w = blockIdx.x + 1;
    if (w >= cut.n) return;
    const Found f = scan_find<ROWS, UNIT>(a, lane, sc, cut.begin(w));
    if (f.u == 0 || cut.begin(w - 1) > f.tile0) return;
    if (r >= min(ROWS, f.s.n * a.g - f.rt * ROWS)) return;
    // Part w - 1 holds the tile's begin in its second place, the later ones
    // theirs in the first.
    auto place = [&](uint32_t v) { return a.part + (size_t)(2 * v + (v == w - 1 ? 1 : 0)) * rows_part(D, QT); };
    const uint32_t last = cut.part_of(f.tile0 + f.s.nu - 1);
    const int n = (int)(last - w + 2);
    float acc[RW] = {}, ls = 0.0f, mx = kNoMax;
    join_parts<RW>(
        n, lane, [&](int v) { return place(w - 1 + v) + ROWS * D + r; }, ROWS,
        [&](int v) { return place(w - 1 + v) + (size_t)r * D + RW * lane; }, acc, mx, ls);
    const int rr = r + f.rt * ROWS, tok = rr / a.g, h = f.kvh * a.g + (rr - tok * a.g);
    const float inv = inverse(ls);
    uint16_t* dst = a.out + (int64_t)(f.s.first + tok) * a.ld_out + h * D + RW * lane;
#pragma unroll
    for (int e = 0; e < RW; ++e) dst[e] = bf16_rne_bits(acc[e] * inv);
}

// ---- many rows: a workgroup shares K and V tiles ------------------------------------------
//
// A tile is TR rows of one (sequence, kv head), 32 per wave (v_mfma_f32_32x32x16),
// against BN positions at a time, K and V in LDS for all waves, the next ones on
// their way while these are used. D = 512: a wave's output would be 256 registers;
// two waves share 32 rows instead, each with half the columns: half of every
// score's products, exchanged through LDS, and half of the output.
// Where there are tiles for less than half of the workgroups that fit, the longer
// ones' positions are split and the parts joined by a second launch.
//
// Bound by the matrix cores and the vector ALUs in turn: a wave's 32 x 32 scores
// take 2 D / 16 matrix instructions and some 70 vector ones (half as many cycles
// as D = 256's products, as many as D = 64's), and LDS delivers K and V to four
// waves in the time of their products. Prompts of 8192 tokens: 32 heads of 64 on
// 8 376 us (732 TFLOP/s), 16 of 128 on 8 329 us (837), 16 of 256 on 8 500 us
// (1100), 16 of 512 on 1 1220 us (900). BN = 32 at D = 128 gains there (310 us)
// and loses on the shorter ones (4096 tokens 120 -> 134 us, 2048 in a 1024 window
// 52 -> 58); reading K ahead of the next loads' addresses costs 2 to 8 % at D <= 128.
constexpr int tile_ds(int D) { return D == 512 ? 2 : 1; }      // waves that share 32 rows
constexpr int tile_waves(int D) { return D == 512 ? 8 : 4; }
constexpr int tile_rows(int D) { return 32 * tile_waves(D) / tile_ds(D); }
constexpr int tile_bn(int D) { return D <= 128 ? 64 : 32; }
constexpr int tile_bytes(int D) { return tile_bn(D) * 2 * D; }  // of K, of V
constexpr int tile_xch(int D) { return D == 512 ? tile_waves(D) * 4096 : 0; }
constexpr int tile_lds(int D) { return 4 * tile_bytes(D) + tile_xch(D); }

typedef float f32x16 __attribute__((__vector_size__(16 * sizeof(float))));

// Tiles of the sequences of more rows than row_limit, up to and with each
// lane's, in one step of 64 sequences.
struct TileScan {
    int first, n, len;
    bool ok;
    int tiles, incl, sum;
};
template <int TR>
__device__ __forceinline__ TileScan tile_scan(const PagedAttnArgs& a, int b0, int lane) {
    TileScan t{};
    const int b = b0 + lane;
    if (b < a.b.B) {
        t.first = a.b.q_start[b];
        t.n = a.b.q_start[b + 1] - t.first;
        t.len = a.b.kv_len[b];
        const bool here = t.first >= 0 && t.n > 0 && (int64_t)t.first + t.n <= a.b.T;
        t.ok = t.n <= t.len && t.len <= a.b.max_pos;
        const int64_t rows = here ? (int64_t)t.n * a.g : 0;
        if (rows > a.row_limit) t.tiles = (int)((rows + TR - 1) / TR);
    }
    int x = t.tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(x, o);
        if (lane >= o) x += u;
    }
    t.incl = x;
    t.sum = __builtin_amdgcn_readlane(x, 63);
    return t;
}

// The positions tile rt of a sequence runs over, in units of BN.
struct TileSpan {
    int rows;            // of the tile
    int pos_lo, pos_hi;  // of its first and last row
    int us, ulo, nu;
};
template <int TR, int BN>
__device__ __forceinline__ TileSpan tile_span(const PagedAttnArgs& a, int n, int len, bool ok, int rt) {
    TileSpan s;
    const int r0 = rt * TR;  // (rows, of one kv head too, stay below 2^30)
    s.rows = min(TR, n * a.g - r0);
    s.pos_lo = len - n + r0 / a.g;
    s.pos_hi = len - n + (r0 + s.rows - 1) / a.g;
    const int lo = a.window > 0 ? max(0, s.pos_lo + 1 - a.window) : 0;
    s.ulo = lo / BN;
    s.us = min((min(a.sinks, lo) + BN - 1) / BN, s.ulo);
    s.nu = ok ? s.us + s.pos_hi / BN + 1 - s.ulo : 0;
    return s;
}

// Items (tiles times kv heads, times their parts) and where each is found: heaviest
// (last) tiles first, kv heads side by side, so that the workgroups an XCD gets
// in turn share theirs where there are eight.
template <int TR>
__device__ __forceinline__ int tile_count(const PagedAttnArgs& a, const TileScan& sc0, int lane) {  // per kv head
    // (no more than there can be: sequences that overlap must not carry the sum away)
    int all = min(sc0.sum, a.max_tiles);
    for (int b0 = 64; b0 < a.b.B; b0 += 64) all = min(all + tile_scan<TR>(a, b0, lane).sum, a.max_tiles);
    return all;
}

// Where tile gt is (sc0: the first 64 sequences, read once for all that needs them).
template <int TR, int BN>
struct TileAt {
    int seq, rt, first, n, len;
    TileSpan sp;
    __device__ __forceinline__ TileAt(const PagedAttnArgs& a, const TileScan& sc0, int gt, int lane) {
        int base = 0, b0 = 0;
        TileScan sc = sc0;
        while (gt >= base + sc.sum) {
            base += sc.sum;
            b0 += 64;
            sc = tile_scan<TR>(a, b0, lane);
        }
        const int l = __builtin_ctzll(__ballot(base + sc.incl > gt));
        seq = b0 + l;
        first = __builtin_amdgcn_readlane(sc.first, l);
        n = __builtin_amdgcn_readlane(sc.n, l);
        len = __builtin_amdgcn_readlane(sc.len, l);
        rt = gt - base - __builtin_amdgcn_readlane(sc.incl - sc.tiles, l);
        sp = tile_span<TR, BN>(a, n, len, __builtin_amdgcn_readlane((int)sc.ok, l) != 0, rt);
    }
};

// ---- fewer tiles than workgroups that fit: their positions in parts
//
// A causal prompt's tiles run over 1 to n units: as many parts of each would leave
// most workgroups idle at the end, so no part has more than `cap` units instead.
// Uneven tiles: three quarters of the average workgroup's units and five more, what
// a part costs beside them, the light tiles filling in behind the heavy. Even ones:
// the total over the workgroups that rounding up leaves, half as many again where
// that makes more parts than run at once, else none is split. (1024 tokens: 16
// heads of 512 74 -> 61 us, 32 of 64 35 -> 31 against two parts each; 512 tokens
// of 16 of 256 37 -> 29 against four; drafts over 4 long contexts 82 -> 77.)
constexpr int kSplitTiles = 512;  // at most, of one kv head
constexpr int kMaxParts = 64;     // of a tile: a lane each in the merge
constexpr int kMinCap = 2;        // (4: 380 tokens of 32 heads of 64 in 3 sequences 27 us for 21)
constexpr int kTabInts = 8;       // entry of part 0, parts, first row of the sequence, tile, rows, kv head

__device__ __forceinline__ int sum64(int v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return uniform(v);
}

// Units of every tile, into LDS, by all waves.
template <int TR, int BN, int NW>
__device__ __forceinline__ void tile_units(const PagedAttnArgs& a, const TileScan& sc0, int tiles, int lane, int wave, int* nu) {
    int base = 0, turn = 0;
    for (int b0 = 0; b0 < a.b.B && base < tiles; b0 += 64) {
        const TileScan sc = b0 ? tile_scan<TR>(a, b0, lane) : sc0;
        for (int x0 = 0; x0 < sc.sum && base + x0 < tiles; x0 += 64, ++turn) {
            if (turn % NW != wave) continue;
            const int x = x0 + lane;
            int l = 0;  // the sequence: the first lane whose tiles end behind x
#pragma unroll
            for (int o = 32; o; o >>= 1)
                if (__shfl(sc.incl, l + o - 1) <= x) l += o;
            l = min(l, 63);
            const int before = __shfl(sc.incl - sc.tiles, l), n = __shfl(sc.n, l), len = __shfl(sc.len, l);
            const bool ok = __shfl((int)sc.ok, l) != 0;
            if (x < sc.sum && base + x < tiles) nu[base + x] = tile_span<TR, BN>(a, n, len, ok, x - before).nu;
        }
        base += sc.sum;
    }
    __syncthreads();
}
__device__ __forceinline__ int tile_parts(int nu, int cap) { return max(1, (nu + cap - 1) / cap); }
// Parts of all tiles of a kv head.
__device__ __forceinline__ int tile_parts_sum(const int* nu, int tiles, int lane, int cap) {
    int c = 0;
    for (int t = lane; t < tiles; t += 64) c += tile_parts(nu[t], cap);
    return sum64(c);
}
__device__ __forceinline__ int tile_cap(const PagedAttnArgs& a, const int* nu, int tiles, int lane, int& parts) {
    int total = 0, most = 0;
    for (int t = lane; t < tiles; t += 64) {
        total += nu[t];
        most = max(most, nu[t]);
    }
    total = sum64(total);
#pragma unroll
    for (int o = 32; o; o >>= 1) most = max(most, __shfl_xor(most, o));
    most = uniform(most);
    const int slots = a.slots / a.kv_heads;  // of a kv head
    const int least = max(kMinCap, (most + kMaxParts - 1) / kMaxParts);
    if ((int64_t)total * 5 <= (int64_t)most * tiles * 3) {  // uneven: the light ones fill in behind the heavy
        const int cap = max(least, (int)((int64_t)total * 3 / (4 * slots)) + 5);
        parts = tile_parts_sum(nu, tiles, lane, cap);
        if (parts <= 2 * slots) return cap;
    }
    int cap = max(least, (total + slots - tiles / 2 - 1) / max(1, slots - tiles / 2));
    for (int turn = 0; turn < 2; ++turn, cap += cap / 2) {
        parts = tile_parts_sum(nu, tiles, lane, cap);
        if (parts <= slots) return cap;
    }
    parts = tiles;
    return INT_MAX / 2;
}

template <int D>
__device__ __forceinline__ void tile_item(const PagedAttnArgs& a, const TileScan& sc0, int gt, int kvh, int split, int nsplit, int entry, int* tab, unsigned char* smem) {
    constexpr int DS = tile_ds(D), NW = tile_waves(D), TR = tile_rows(D), BN = tile_bn(D);
    constexpr int DW = D / DS;            // this wave's columns of the output (and of its scores' products)
    constexpr int TB = tile_bytes(D), NC = D / 8, RPL = 512 / D;
    constexpr int LR = BN / NW;           // positions a wave loads: within one block of 16
    constexpr int NL = LR / RPL;          // its loads of K (of V)
    constexpr int NB = BN / 16;
    constexpr int KR = 4, VR = 4;         // operands of K, of V on their way from LDS
    unsigned char* kbuf = smem;
    unsigned char* vbuf = smem + 2 * TB;
    float* xch = reinterpret_cast<float*>(smem + 4 * TB);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave / DS, dh = wave % DS;
    const int col = lane & 31, h = lane >> 5;

    const TileAt<TR, BN> at_item(a, sc0, gt, lane);
    const int seq = at_item.seq, rt = at_item.rt;
    const int first = at_item.first, n = at_item.n, len = at_item.len;
    const TileSpan sp = at_item.sp;
    const int u0 = uniform((int)((int64_t)sp.nu * split / nsplit));
    const int u1 = uniform((int)((int64_t)sp.nu * (split + 1) / nsplit));
    if (tab && split == 0 && tid == 0) {
        int* e = tab + kTabInts * (1 + gt * a.kv_heads + kvh);
        e[0] = entry, e[1] = nsplit, e[2] = first, e[3] = rt, e[4] = sp.rows, e[5] = kvh;
    }

    const int32_t* table = a.b.table + (int64_t)seq * a.b.ld_table;
    auto unit_pos = [&](int u) { return (u < sp.us ? u : u - sp.us + sp.ulo) * BN; };
    // The pages of 64 units' positions that this wave loads, one per lane; a bit
    // per unit for each of its blocks of 16 that has none.
    int pages = -1, pages0 = u0;
    uint64_t gone[NB] = {};
    auto load_pages = [&](int v0) __attribute__((always_inline)) {
        pages0 = v0;
        const int p = unit_pos(v0 + lane);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const bool in = v0 + lane < u1 && p + 16 * k < len;
            int e = in ? table[(p + 16 * k) >> a.b.shift] : -1;
            if ((unsigned)e >= (unsigned)a.b.pages) e = -1;
            gone[k] = __ballot(in && e < 0);
            pages = k == wave * LR / 16 ? e : pages;
        }
    };
    uint32_t holes = 0;  // NB bits by unit modulo 4
    const uint32_t kb_lds = __builtin_amdgcn_readfirstlane(lds_addr(kbuf)) + wave * LR * (2 * D);
    const uint32_t vb_lds = __builtin_amdgcn_readfirstlane(lds_addr(vbuf)) + wave * LR * (2 * D);
    // The wave's rows start at a multiple of 4, not of 16: their bits of the
    // swizzles are part of the lane's offset.
    const uint32_t dma_k = (lane / NC) * (2 * D) + ((lane % NC) ^ k_swz<D>(wave * LR + lane / NC)) * 16;
    const uint32_t dma_v = (lane / NC) * (2 * D) + ((lane % NC) ^ v_swz<D>(wave * LR + lane / NC)) * 16;
    // Starts unit u's K (then its V) on the way to LDS; K before V, units in order.
    auto issue = [&](int u, bool v) __attribute__((always_inline)) {
        if (u - pages0 >= 64) load_pages(u);
        const int page = __builtin_amdgcn_readlane(pages, u - pages0), p = unit_pos(u) + wave * LR;
        const uint32_t bytes = page < 0 ? 0u : (uint32_t)max(0, min(LR, len - p)) * (2 * D);
        const int64_t off = (((int64_t)kvh << a.b.shift) + (p & ((1 << a.b.shift) - 1))) * D;
        if (!v) {
            uint32_t now = 0;
#pragma unroll
            for (int k = 0; k < NB; ++k) now |= (uint32_t)(gone[k] >> (u - pages0) & 1) << k;
            const int at = NB * (u & 3);
            holes = (holes & ~(((1u << NB) - 1) << at)) | (now << at);
        }
        const uint16_t* src = v ? a.vpages + max(page, 0) * a.v_stride : a.kpages + max(page, 0) * a.k_stride;
        const __amdgpu_buffer_rsrc_t r = wave_rsrc(src + off, bytes);
        const uint32_t dst = (v ? vb_lds : kb_lds) + (u & 1) * TB, at = here(v ? dma_v : dma_k);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t x = v ? (uint32_t)v_swz<D>(RPL * i) : (uint32_t)k_swz<D>(RPL * i);
            load_lds16(r, at ^ (x * 16), 1024 * i, dst + 1024 * i);
        }
    };

    // This lane's row: column col of the wave's 32.
    const int r0 = rt * TR + 32 * rg;
    const int nrows = max(0, min(32, n * a.g - r0));
    const int row = r0 + min(col, max(nrows - 1, 0));
    const int tok = min(row / a.g, n - 1), head = kvh * a.g + row % a.g;
    const int pos = len - n + tok;
    const int wpos_lo = len - n + r0 / a.g;
    const int wpos_hi = len - n + (r0 + max(nrows, 1) - 1) / a.g;
    const float c = fmaxf(a.scale * kLog2e, kMinScale);
    bf16x8 q[DW / 16];
    {
        const uint16_t* qr = a.q + (int64_t)(first + tok) * a.ld_q + head * D + dh * DW + 8 * h;
#pragma unroll
        for (int i = 0; i < DW / 16; ++i) q[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(qr + 16 * i));
        // Waited for here: the compiler would else wait at their first use, in
        // the loop, each time, for whatever is on its way to LDS by then.
#pragma unroll
        for (int i = 0; i < DW / 16; ++i) asm volatile("" : "+v"(q[i]));
    }
    f32x16 o[DW / 32];
#pragma unroll
    for (int d = 0; d < DW / 32; ++d) o[d] = f32x16{};
    float m = kNoMax, l = 0.0f;

    const int vrow = 4 * h + ((lane & 15) >> 2);
    const uint32_t rd_k = col * (2 * D) + (h ^ k_swz<D>(col)) * 16;
    const uint32_t rd_v = vrow * (2 * D) + ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ v_swz<D>(vrow)) * 16 + (lane & 1) * 8;

    // Rows that see nothing of 32 positions at p0 (or are none) are done with them.
    auto skip = [&](int p0) { return nrows == 0 || p0 > wpos_hi; };
    // K q of the 32 positions whose rows begin at ks, over this wave's columns.
    auto scores = [&](const unsigned char* ks) __attribute__((always_inline)) {
        f32x16 s{};
        const uint32_t at = here(rd_k);
        auto read_k = [&](int i) __attribute__((always_inline)) {
            return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(
                ks + (at ^ piece<D>(2 * i)) + piece_far<D>((dh * DW + 16 * i) / 8 & ~15)));
        };
        bf16x8 k[KR];
#pragma unroll
        for (int i = 0; i < KR; ++i) k[i] = read_k(i);
        // The products go ahead of the other workgroup's softmax (three chunks in a
        // 1024 window at D = 256: 78 -> 75 us, 8192 tokens 532 -> 509). At D = 512 the
        // two groups of waves already take turns, and it costs: 4096 tokens 323 -> 331.
        if constexpr (DS == 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < DW / 16; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[i % KR], q[i], s, 0, 0, 0);
            if (i + KR < DW / 16) k[i % KR] = read_k(i + KR);
        }
        if constexpr (DS == 1) __builtin_amdgcn_s_setprio(0);
        return s;
    };
    // Their weights, and the output's share of V.
    auto absorb = [&](const f32x16& sv, int p0, const unsigned char* vs, uint32_t hole) __attribute__((always_inline)) {
        hole &= 3;  // of its two blocks of 16
        float s[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = sv[i];
        const bool masked = hole || p0 + 31 > wpos_lo || (a.window > 0 && p0 <= wpos_hi - a.window && p0 + 31 >= a.sinks);
        if (masked) {
            // Relative to p0 + 4 h, so that positions are constants.
            const int at = pos - p0 - 4 * h, lo = a.window > 0 ? at - a.window : INT_MIN, sk = a.sinks - p0 - 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int p = 8 * (i / 4) + i % 4, hi = hole >> (i / 8) & 1 ? -1 : at;
                s[i] = (p <= hi) & ((p > lo) | (p < sk)) ? s[i] : -__builtin_inff();
            }
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        if (__any(__builtin_fmaf(top, c, -m) > kSlack)) {
            const uint32_t tb = __builtin_bit_cast(uint32_t, top);
            auto sw = __builtin_amdgcn_permlane32_swap(tb, tb, false, false);
            const uint32_t t0 = sw[0], t1 = sw[1];
            const float mn = fmaxf(m, fmaxf(__builtin_bit_cast(float, t0), __builtin_bit_cast(float, t1)) * c);
            const float fac = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= fac;
#pragma unroll
            for (int d = 0; d < DW / 32; ++d) {
                o[d] *= fac;
                asm volatile("" : "+v"(o[d]));  // in place, one after the other
            }
        }
        float w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float si = s[i];
            w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(si, c, -m));
        }
        l += (((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]))) +
             (((w[8] + w[9]) + (w[10] + w[11])) + ((w[12] + w[13]) + (w[14] + w[15])));
        // Weights as bf16, the matrix cores' type (see the streaming kernel).
        bf16x8 pw[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) pw[i >> 3][i & 7] = (__bf16)w[i];
        // Columns 32 d .. of this wave, positions 16 k + 8 e + 4 h .. + 3.
        const uint32_t at = here(rd_v);
        auto read_v = [&](int d, int k) __attribute__((always_inline)) {
            const unsigned char* v = vs + (at ^ piece<D>(4 * d)) + piece_far<D>((dh * DW + 32 * d) / 8 & ~15) + k * 32 * D;
            const s16x4 lo = read_tr(v), hi = read_tr(v + 16 * D);
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        // Operand j: two blocks of columns in turn, then their second 16 positions.
        constexpr int NV = DW / 16;
        auto blk = [](int j) { return (j & ~3) / 2 + (j & 1); };
        bf16x8 v[VR];
#pragma unroll
        for (int j = 0; j < VR; ++j) v[j] = read_v(blk(j), j >> 1 & 1);
        if constexpr (DS == 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            o[blk(j)] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[j % VR], pw[j >> 1 & 1], o[blk(j)], 0, 0, 0);
            if (j + VR < NV) v[j % VR] = read_v(blk(j + VR), (j + VR) >> 1 & 1);
        }
        if constexpr (DS == 1) __builtin_amdgcn_s_setprio(0);
    };

    if (u1 > u0) {
        load_pages(u0);
        issue(u0, false);
        issue(u0, true);
    }
    if constexpr (DS == 1) {
#pragma unroll 1
        for (int u = u0; u < u1; ++u) {
            wait_vm<0>();
            __syncthreads();
            if (u + 1 < u1) {
                issue(u + 1, false);
                issue(u + 1, true);
            }
            const int pt = unit_pos(u);
            const unsigned char* kt = kbuf + (u & 1) * TB;
            const unsigned char* vt = vbuf + (u & 1) * TB;
#pragma unroll 1
            for (int sub = 0; sub < BN / 32 && !skip(pt + 32 * sub); ++sub)
                absorb(scores(kt + sub * 64 * D), pt + 32 * sub, vt + sub * 64 * D, holes >> (NB * (u & 3) + 2 * sub));
        }
    } else {
        // Two groups of waves, one of each per SIMD, half a unit apart: while one
        // multiplies K the other has its softmax and V, so the matrix cores, the
        // vector ALUs and LDS all have work (in step, each waits for the others:
        // 4096 tokens, 16 heads of 512, 342 us; so 328). Phase p, between two barriers:
        // even p = 2 k is unit k's K for group 0 and unit k - 1's V for group 1, odd
        // p the reverse; loads run two phases ahead, unit k's K needed from phase
        // 2 k, its V from 2 k + 1, and each buffer is filled again when its last
        // reader has passed a barrier.
        const int grp = wave / (NW / 2), nu = u1 - u0;
        f32x4* mine = reinterpret_cast<f32x4*>(xch + wave * 1024) + lane;
        const f32x4* other = reinterpret_cast<const f32x4*>(xch + (wave ^ 1) * 1024) + lane;
        auto begin = [&](int phase) __attribute__((always_inline)) {
            if (phase + 1 < 2 * nu)
                wait_vm<NL>();  // the loads issued in the last phase may still be on their way
            else
                wait_vm<0>();
            __syncthreads();
            if (phase + 2 < 2 * nu) issue(u0 + ((phase + 2) >> 1), phase & 1);
        };
        if (nu > 0 && grp == 1) begin(0);
#pragma unroll 1
        for (int u = u0; u < u1; ++u) {
            const int p0 = unit_pos(u);
            f32x16 s{};
            begin(2 * (u - u0) + grp);
            if (!skip(p0)) {
                s = scores(kbuf + (u & 1) * TB);
#pragma unroll
                for (int i = 0; i < 4; ++i) mine[64 * i] = f32x4{s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]};
            }
            begin(2 * (u - u0) + grp + 1);
            if (!skip(p0)) {
                // With the other half's products; the sum is the same in both waves.
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 x = other[64 * i];
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[4 * i + e] += x[e];
                }
                absorb(s, p0, vbuf + (u & 1) * TB, holes >> (NB * (u & 3)));
            }
        }
        if (nu > 0 && grp == 0) begin(2 * nu);
    }

    float* part = a.part + (int64_t)(entry + split * a.kv_heads) * (TR * (D + 2));
    float no = 0.0f;
#pragma unroll
    for (int d = 0; d < DW / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) no = __builtin_fmaf(o[d][i], 0.0f, no);
    bool odd = __any(no != 0.0f);
    if constexpr (DS == 2) {  // in either half's columns
        int* odds = reinterpret_cast<int*>(xch);
        __syncthreads();
        if (lane == 0) odds[wave] = odd;
        __syncthreads();
        odd = odds[wave] | odds[wave ^ 1];
    }
    if (odd) {  // see plain_row; with two waves per row, one does it
        for (int r = 0; dh == 0 && r < nrows; ++r) {
            const int rr = r0 + r, tk = rr / a.g, hd = kvh * a.g + rr % a.g;
            float acc[D / 64], mr, lr;
            plain_row<D>(a, seq, kvh, a.q + (int64_t)(first + tk) * a.ld_q + hd * D, len - n + tk, sp.us, sp.ulo, BN, u0, u1,
                         lane, acc, mr, lr);
            const float inv = inverse(lr);
            uint16_t* dst = a.out + (int64_t)(first + tk) * a.ld_out + hd * D + D / 64 * lane;
            float* pr = part + (32 * rg + r) * D + D / 64 * lane;
#pragma unroll
            for (int e = 0; e < D / 64; ++e) {
                if (nsplit == 1)
                    dst[e] = bf16_rne_bits(acc[e] * inv);
                else
                    pr[e] = acc[e];
            }
            if (nsplit > 1 && lane == 0) {
                part[TR * D + 32 * rg + r] = mr;
                part[TR * (D + 1) + 32 * rg + r] = lr;
            }
        }
        return;
    }
    l += __shfl_xor(l, 32);
    if (col >= nrows) return;
    if (nsplit == 1) {
        const float inv = inverse(l);
        uint16_t* dst = a.out + (int64_t)(first + tok) * a.ld_out + head * D + dh * DW + 4 * h;
#pragma unroll
        for (int d = 0; d < DW / 32; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                store4(dst + 32 * d + 8 * k, f32x4{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]}, inv);
    } else {
        float* dst = part + (32 * rg + col) * D + dh * DW + 4 * h;
#pragma unroll
        for (int d = 0; d < DW / 32; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * k) =
                    f32x4{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]};
        if (dh == 0 && h == 0) {
            part[TR * D + 32 * rg + col] = m;
            part[TR * (D + 1) + 32 * rg + col] = l;
        }
    }
}

template <int D>
__global__ void __launch_bounds__((64 * tile_waves(D)), 2) attn_paged_tile_kernel(PagedAttnArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int TR = tile_rows(D), BN = tile_bn(D);
    static_assert(tile_lds(D) >= 4 * kSplitTiles, "the tiles' units");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const TileScan sc0 = tile_scan<TR>(a, 0, lane);
    const int tiles = tile_count<TR>(a, sc0, lane), items = tiles * a.kv_heads;
    const bool split = items <= a.max_items;
    if (a.tab && blockIdx.x == 0 && tid == 0) a.tab[0] = split ? items : 0;
    if (items == 0) return;  // (the streaming kernel's all; there may be no slots to plan for)
    int gt, kvh, part = 0, parts = 1, entry = 0;
    if (split) {
        int* nu = reinterpret_cast<int*>(smem);
        tile_units<TR, BN, tile_waves(D)>(a, sc0, tiles, lane, wave, nu);
        int all;
        const int cap = tile_cap(a, nu, tiles, lane, all);
        const int e = all * a.kv_heads - 1 - (int)blockIdx.x;
        if (e < 0) return;
        int base = 0, t0 = 0, p, incl;
        while (true) {
            p = t0 + lane < tiles ? tile_parts(nu[t0 + lane], cap) : 0;
            incl = p;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int u = __shfl_up(incl, o);
                if (lane >= o) incl += u;
            }
            const int sum = __builtin_amdgcn_readlane(incl, 63);
            if (e < (base + sum) * a.kv_heads) break;
            base += sum;
            t0 += 64;
        }
        const int l = __builtin_ctzll(__ballot((base + incl) * a.kv_heads > e));
        gt = t0 + l;
        parts = __builtin_amdgcn_readlane(p, l);
        entry = (base + __builtin_amdgcn_readlane(incl, l) - parts) * a.kv_heads;
        part = (e - entry) / a.kv_heads;
        kvh = e - entry - part * a.kv_heads;
        entry += kvh;
        __syncthreads();  // nu gives way to K and V
    } else {
        const int item = items - 1 - (int)blockIdx.x;
        if (item < 0) return;
        gt = item / a.kv_heads;
        kvh = item - gt * a.kv_heads;
    }
    // (tiles of more rows than max_q told of may be more than tab has entries for: they are not split)
    tile_item<D>(a, sc0, uniform(gt), uniform(kvh), uniform(part), uniform(parts), uniform(entry), split ? a.tab : nullptr, smem);
}

// The parts of the tiles joined, `groups` workgroups to a tile, merge_rows(D) of
// its rows at a time: the parts' factors first, a row per wave and a part per
// lane, into LDS, then the outputs, 16 bytes per lane and part.
constexpr int merge_rows(int D) { return 1024 / D; }
template <int D, int PG>
__global__ void __launch_bounds__((256 * PG)) attn_paged_tile_merge_kernel(PagedAttnArgs a, int groups) {
    constexpr int TR = tile_rows(D), R = merge_rows(D), C = D / 4;  // 16-byte pieces of a row
    __shared__ float fac[R][64];
    __shared__ float inv[R];
    __shared__ f32x4 sums[PG > 1 ? PG - 1 : 1][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int item = blockIdx.x / groups;
    if (item >= a.tab[0]) return;
    const int* e = a.tab + kTabInts * (1 + item);
    const int np = e[1], first = e[2], rt = e[3], tile_n = e[4], kvh = e[5];
    if (np == 1) return;
    const float* part = a.part + (int64_t)e[0] * (TR * (D + 2));
    auto at = [&](int v) { return part + (int64_t)v * a.kv_heads * (TR * (D + 2)); };
    const float* mine = at(min(lane, np - 1));
    for (int r0 = blockIdx.x % groups * R; r0 < tile_n; r0 += groups * R) {
        const int rows = min(R, tile_n - r0), r = tid % 256 / C, c = tid % C;
        const int vlo = tid / 256 * np / PG, vhi = (tid / 256 + 1) * np / PG;  // this group's parts
        f32x4 acc{}, x[8];
        auto load = [&](int v0) {
#pragma unroll
            for (int q = 0; q < 8; ++q)
                x[q] = v0 + q < vhi && r < rows ? *reinterpret_cast<const f32x4*>(at(v0 + q) + (r0 + r) * D + 4 * c)
                                               : f32x4{0, 0, 0, 0};
        };
        load(vlo);
#pragma unroll
        for (int w = wave; w < R; w += 4 * PG) {
            const int rr = r0 + min(w, rows - 1);
            const float m = lane < np ? mine[TR * D + rr] : kNoMax, l = lane < np ? mine[TR * (D + 1) + rr] : 0.0f;
            float top = m;
#pragma unroll
            for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
            const float f = __builtin_amdgcn_exp2f(m - top);
            float sum = l * f;
#pragma unroll
            for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
            fac[w][lane] = f;
            if (lane == 0) inv[w] = inverse(sum);
        }
        __syncthreads();
        for (int v0 = vlo; v0 < vhi; v0 += 8) {
            if (v0 != vlo) load(v0);
#pragma unroll
            for (int q = 0; q < 8; ++q) acc += x[q] * fac[r][min(v0 + q, 63)];
        }
        if constexpr (PG > 1) {
            if (tid >= 256) sums[tid / 256 - 1][tid % 256] = acc;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < PG - 1; ++k) acc += sums[k][tid % 256];
        }
        if (r < rows && tid < 256) {
            const int rr = rt * TR + r0 + r, tok = rr / a.g, head = kvh * a.g + rr % a.g;
            store4(a.out + (int64_t)(first + tok) * a.ld_out + head * D + 4 * c, acc, inv[r]);
        }
        __syncthreads();
    }
}

}  // namespace

}  // namespace alv

using namespace alv;

namespace alv {
namespace {

// How a call's work is spread.
struct AttnPlan {
    int qt;              // row tiles of 16 in the streaming kernel (0: not launched)
    int64_t row_limit;   // sequences of at most this many rows are its, the others the tile kernel's
    int grid;            // its workgroups
    int64_t grid_tiles;  // tiles times kv heads of the tile kernel at most (0: not launched),
    int64_t tiles;       // and at most as far as max_q tells
    int slots;           // parts of tiles; 0: none is split
    uint64_t rows_bytes, tab_bytes, part_bytes;
};

AttnPlan attn_plan(int heads, int kv_heads, int D, int B, int T, int max_q) {
    AttnPlan p{};
    const int64_t g = heads / kv_heads;
    max_q = std::min(max_q, T);  // (and its products stay within 64 bits)
    const int qt_max = D <= 128 ? 4 : (D == 256 ? 2 : 1);
    const int64_t most = (max_q > 0 ? max_q : T) * g;          // rows of a sequence at most
    const int64_t rows = (max_q > 0 ? max_q : ((int64_t)T + B - 1) / B) * g;  // as far as is known
    const int64_t slots = (int64_t)device_cus() * (D == 512 ? 1 : 2);
    const int64_t tr = 128;
    auto tiles_of = [&](int64_t row_limit) {  // that sequences of more rows than that have at most
        return (T * g / tr + std::min((int64_t)B, T * g / (row_limit + 1) + 1)) * kv_heads;
    };
    auto tiles_known = [&](int64_t n) { return max_q > 0 ? std::min(n, (int64_t)B * ((max_q * g + tr - 1) / tr) * kv_heads) : n; };
    // A batch of tiles few enough to be cut is the tile kernel's alone, without the
    // other's two launches: its parts read long contexts as fast (0 to 6 tokens each
    // over up to 4000 positions, 10 sequences of 16 heads of 512 63 -> 35 us; a chunk of
    // 300 and eight single tokens over 2000, 16 heads of 256 65 -> 40). And that from
    // more than 16 rows on (32 rows over up to 16000 positions, 6 sequences, D = 256
    // 40 -> 28 us, 128 29 -> 23; 16 rows 31 -> 28 and 20 -> 21, D = 64 36 -> 40), at
    // D = 512 from 16 on (52 -> 40).
    const bool few = tiles_known(tiles_of(0)) <= slots / 2;
    const bool tiles = (B == 1 ? most : rows) > (few ? (D == 512 ? 15 : 16) : 16 * qt_max);
    // No sequence is left for the streaming kernel there, nor where there is one, or
    // all have max_q rows (should they not, the tile kernel takes them all the same).
    const bool stream = !(tiles && (B == 1 || few || (max_q > 0 && (int64_t)B * max_q <= T)));
    if (stream) {
        const int64_t r = tiles ? g : rows;
        p.qt = std::min(qt_max, r <= 16 ? 1 : (r <= 32 ? 2 : 4));
        p.row_limit = tiles ? 16 * p.qt : INT64_MAX;
        p.grid = device_cus();
        p.rows_bytes = (uint64_t)p.grid * 2 * 16 * p.qt * (D + 2) * sizeof(float);
    }
    p.part_bytes = p.rows_bytes;
    if (tiles) {
        static_assert(tile_rows(64) == 128 && tile_rows(128) == 128 && tile_rows(256) == 128 && tile_rows(512) == 128, "");
        p.grid_tiles = tiles_of(p.row_limit);
        p.tiles = tiles_known(p.grid_tiles);
        // (up to half: 1800 tokens of 32 heads of 64, 450 tiles for 512 workgroups, 46 us
        // in parts, 41 whole; 16 of 128, 232 tiles, 42 against 49)
        if (p.tiles <= slots / 2 && p.tiles <= kSplitTiles) {
            p.slots = (int)slots;
            p.tab_bytes = (uint64_t)(p.tiles + 1) * kTabInts * sizeof(int);
            p.part_bytes += p.tab_bytes + std::min((uint64_t)slots * 2, (uint64_t)p.tiles * kMaxParts) * tr * (D + 2) * sizeof(float);
        }
    }
    return p;
}

// Dynamic LDS past 64 KiB, asked for once per kernel and device.
int allow_lds(const void* k, int lds, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (int rc = hip_check(hipGetDevice(&dev), "hipGetDevice")) return rc;
    if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return ALV_OK;
    if (int rc = hip_check(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute"))
        return rc;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return ALV_OK;
}

template <int D, int QT>
int launch_rows(const PagedAttnArgs& a, const AttnPlan& p, hipStream_t s) {
    constexpr int lds = rows_lds(D, QT);
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_lds(reinterpret_cast<const void*>(&attn_paged_rows_kernel<D, QT>), lds, done)) return rc;
    hipLaunchKernelGGL((attn_paged_rows_kernel<D, QT>), dim3(p.grid), dim3(64 * rows_waves(D)), lds, s, a);
    if (int rc = hip_check(hipGetLastError(), "attn_paged_rows_kernel launch")) return rc;
    hipLaunchKernelGGL((attn_paged_rows_merge_kernel<D, QT>), dim3(p.grid - 1, 4 * QT), dim3(256), 0, s, a, p.grid);
    return hip_check(hipGetLastError(), "attn_paged_rows_merge_kernel launch");
}

template <int D>
int launch_tiles(const PagedAttnArgs& a, const AttnPlan& p, hipStream_t s) {
    constexpr int lds = tile_lds(D);
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_lds(reinterpret_cast<const void*>(&attn_paged_tile_kernel<D>), lds, done)) return rc;
    hipLaunchKernelGGL((attn_paged_tile_kernel<D>), dim3((uint32_t)std::max(p.grid_tiles, (int64_t)p.slots * 2)), dim3(64 * tile_waves(D)), lds, s, a);
    if (int rc = hip_check(hipGetLastError(), "attn_paged_tile_kernel launch")) return rc;
    if (p.slots == 0) return ALV_OK;
    // Few tiles are joined by as many workgroups as they have rows for, many by fewer
    // each (a tile in one part costs its workgroups two loads).
    const int groups = (int)std::max((int64_t)1, std::min((int64_t)tile_rows(D) / merge_rows(D), 4096 / p.tiles));
    // Four groups of threads share many parts (drafts over 4 long contexts, 64 parts:
    // 12.5 -> 10.5 us; 16 parts of 32 tiles, D = 256: 15.5 -> 21.4).
    if (p.slots / p.tiles >= 32)
        hipLaunchKernelGGL((attn_paged_tile_merge_kernel<D, 4>), dim3((uint32_t)p.tiles * groups), dim3(1024), 0, s, a, groups);
    else
        hipLaunchKernelGGL((attn_paged_tile_merge_kernel<D, 1>), dim3((uint32_t)p.tiles * groups), dim3(256), 0, s, a, groups);
    return hip_check(hipGetLastError(), "attn_paged_tile_merge_kernel launch");
}

template <int D>
int launch_d(PagedAttnArgs a, const AttnPlan& p, hipStream_t s) {
    float* part = a.part;
    if (p.grid_tiles) {
        if (p.slots) a.tab = reinterpret_cast<int*>(part + p.rows_bytes / sizeof(float));
        a.part = part + (p.rows_bytes + p.tab_bytes) / sizeof(float);
        if (int rc = launch_tiles<D>(a, p, s)) return rc;
    }
    a.part = part;
    if (p.qt == 1) return launch_rows<D, 1>(a, p, s);
    if constexpr (D <= 256)
        if (p.qt == 2) return launch_rows<D, 2>(a, p, s);
    if constexpr (D <= 128)
        if (p.qt == 4) return launch_rows<D, 4>(a, p, s);
    return ALV_OK;
}

}  // namespace
}  // namespace alv

extern "C" uint64_t alv_attention_paged_workspace(int heads, int kv_heads, int D, int B, int T, int max_q) {
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || D < 1 || B < 1 || T < 1 || max_q < 0) return 0;
    return attn_plan(heads, kv_heads, D, B, T, max_q).part_bytes;
}

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
    if (heads > kMaxHeads) return fail(ALV_ERR_RANGE, "%d heads (at most %d)", heads, kMaxHeads);
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
    a.heads = heads, a.kv_heads = kv_heads, a.g = heads / kv_heads, a.sinks = sinks, a.scale = scale;
    a.window = window < a.b.max_pos ? window : 0;  // (all positions are within it)
    a.out = out, a.ld_out = ld_out;
    if ((int64_t)T * heads > (int64_t)1 << 30)  // (the largest launch: 2^32 threads)
        return fail(ALV_ERR_RANGE, "%d rows of %d heads in one call (at most 2^30 rows times heads)", T, heads);
    const AttnPlan p = attn_plan(heads, kv_heads, D, B, T, max_q);
    if (p.grid_tiles * 512 > (int64_t)UINT32_MAX)
        return fail(ALV_ERR_RANGE, "%d rows of %d heads in %d sequences: too many tiles for one call", T, heads, B);
    if (p.part_bytes && (!workspace || workspace_bytes < p.part_bytes))
        return fail(ALV_ERR_ARG, "workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
                    (unsigned long long)p.part_bytes);
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(ALV_ERR_ALIGN, "workspace needs 16-byte alignment");
    a.part = static_cast<float*>(workspace);
    a.row_limit = p.row_limit;
    a.slots = p.slots;
    a.max_items = p.slots ? (int)p.tiles : 0;
    a.max_tiles = (int)(p.grid_tiles / kv_heads);
    const hipStream_t s = (hipStream_t)stream;
    switch (D) {
        case 64: return launch_d<64>(a, p, s);
        case 128: return launch_d<128>(a, p, s);
        case 256: return launch_d<256>(a, p, s);
        default: return launch_d<512>(a, p, s);
    }
}
