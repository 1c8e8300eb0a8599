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
    int64_t row_limit;  // sequences of more rows (tokens times q heads per kv head) are not this launch's
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

// Whether one of the two bf16 values of a word is infinite or NaN: its exponent
// of ones carries into the bit above.
__device__ __forceinline__ uint32_t nonfinite_bits(uint32_t w) {
    return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
}
__device__ __forceinline__ bool any_nonfinite(u32x4 v) {
    return (nonfinite_bits(v[0]) | nonfinite_bits(v[1]) | nonfinite_bits(v[2]) | nonfinite_bits(v[3])) != 0;
}

// LDS pieces of a row are stored at (piece ^ swizzle of the row): the K reads (16
// rows, the same piece) and the transposing V reads (4 rows, two pieces) then
// fall on different banks.
template <int D>
__device__ __forceinline__ int k_swz(int row) {
    return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swz(int row) {
    return D == 64 ? ((row >> 1) & 3) * 2 : (row & 7) * 2;
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

// Where value d (a multiple of 4) of V's row p stands in its tile.
template <int D>
__device__ __forceinline__ uint32_t v_at(int p, int d) {
    return p * (2 * D) + (((d >> 3) ^ v_swz<D>(p)) * 16) + (d & 4) * 2;
}

// o += w v for the four values at `p` that are infinite or NaN, for a lane whose
// row sees them.
__device__ __forceinline__ void add_nonfinite(f32x4& o, const unsigned char* p, bool see, float w) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const uint32_t n0 = nonfinite_bits(v.x), n1 = nonfinite_bits(v.y);
    float x0 = o[0], x1 = o[1], x2 = o[2], x3 = o[3];
    if (see && (n0 & 0x8000u)) x0 = __builtin_fmaf(w, bf16_bits_to_f32(v.x & 0xFFFFu), x0);
    if (see && (n0 >> 31)) x1 = __builtin_fmaf(w, bf16_bits_to_f32(v.x >> 16), x1);
    if (see && (n1 & 0x8000u)) x2 = __builtin_fmaf(w, bf16_bits_to_f32(v.y & 0xFFFFu), x2);
    if (see && (n1 >> 31)) x3 = __builtin_fmaf(w, bf16_bits_to_f32(v.y >> 16), x3);
    o = f32x4{x0, x1, x2, x3};
}
// The eight values at `p`, zeros for those that are infinite or NaN.
__device__ __forceinline__ void zero_nonfinite(unsigned char* p) {
    u32x4 v = *reinterpret_cast<u32x4*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t w = v[e], n = nonfinite_bits(w);
        v[e] = w & ~((n >> 15) * 0xFFFFu);
    }
    *reinterpret_cast<u32x4*>(p) = v;
}

__device__ __forceinline__ s16x4 read_tr(const unsigned char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p));
}

// Whether a row at position t sees position p.
__device__ __forceinline__ bool sees(const PagedAttnArgs& a, int p, int t) {
    return p <= t && (a.window <= 0 || p > t - a.window || p < a.sinks);
}

__device__ __forceinline__ void store4(uint16_t* dst, f32x4 v, float l) {
    uint16_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x = v[e];
        b[e] = l == 0.0f ? (uint16_t)0 : bf16_rne_bits(x / l);
    }
    *reinterpret_cast<uint2*>(dst) = uint2{b[0] | ((uint32_t)b[1] << 16), b[2] | ((uint32_t)b[3] << 16)};
}

constexpr float kNoMax = -3.0e38f;  // running maximum of a row that has seen nothing
constexpr float kMinScale = 1e-37f;  // -infinity times it is -infinity, a score times it 0
constexpr float kLog2e = 1.44269504088896340736f;
// A row's reference stays while its scores exceed it by no more than this many
// powers of two: weights up to 2^8 lose nothing in float32 or bf16, and most
// blocks then need neither a maximum over the lanes nor a rescaled output.
constexpr float kSlack = 8.0f;

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

// A sequence's place in the line, per lane of the scan.
struct RowsSeq {
    int first, n, len;
    int tiles;        // row tiles (of each kv head)
    int us, ulo, nu;  // units of first tokens; first unit of the window; units in all
};

constexpr int rows_waves(int D) { return D == 512 ? 2 : 4; }
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
    return (ring > outs ? ring : outs) + 2 * rows_waves(D) * 16 * QT * 4 + (rows_q_lds(D, QT) ? 32 * QT * D : 0);
}
constexpr int rows_mls(int D, int QT) {  // where the waves' maxima and sums stand; q behind them
    return rows_lds(D, QT) - 2 * rows_waves(D) * 16 * QT * 4 - (rows_q_lds(D, QT) ? 32 * QT * D : 0);
}
// Floats of one workspace place: outputs, maxima, sums.
constexpr int rows_part(int D, int QT) { return 16 * QT * (D + 2); }

struct Scan {
    RowsSeq s;          // this lane's sequence
    uint64_t incl;      // work of the sequences of this step up to and with this lane's
    uint64_t base, sum; // work before this step; of this step
    int b0;             // the step's first sequence
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
    for (int b0 = 64; b0 < a.b.B; b0 += 64) {
        Scan t;
        scan_step<ROWS, UNIT>(a, b0, lane, 0, t);
        total += t.sum;
    }
    return total;
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
    const uint64_t tile = in >> 32 ? in / (uint32_t)f.s.nu : (uint32_t)in / (uint32_t)f.s.nu;
    f.u = uniform((int)(in - tile * f.s.nu));
    f.tile0 = start + tile * f.s.nu;
    f.kvh = uniform((int)((uint32_t)tile / (uint32_t)f.s.tiles));
    f.rt = uniform((int)((uint32_t)tile - (uint32_t)f.kvh * f.s.tiles));
    return f;
}

// Where part w of the line begins.
__device__ __forceinline__ uint64_t part_begin(uint64_t total, uint32_t parts, uint32_t w) {
    const uint64_t q = total / parts, r = total - q * parts;
    return q * w + min((uint64_t)w, r);
}
__device__ __forceinline__ uint32_t part_count(uint64_t total, int grid) {
    return (uint32_t)min((uint64_t)grid, total);
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
    const uint32_t parts = part_count(total, gridDim.x);
    if (blockIdx.x >= parts) return;
    uint64_t x = part_begin(total, parts, blockIdx.x);
    const uint64_t end = part_begin(total, parts, blockIdx.x + 1);

    unsigned char* ring = smem + wave * NS * rows_stage(D);
    const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_addr(ring));
    float* mls = reinterpret_cast<float*>(smem + rows_mls(D, QT));  // [wave][max | sum][row]
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
        if (QL) __syncthreads();
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
            unsigned char* kt = ring + (j % NS) * rows_stage(D);
            unsigned char* vt = kt + HALF;
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
                // Weights as bf16, the matrix cores' type: half a step of 2^-8
                // relative each, as much as the output's own rounding.
                pw[t] = pack4(w0, w1, w2, w3);
            }
            auto read_v = [&](int d) __attribute__((always_inline)) {
                return read_tr(vt + (rd_v ^ piece<D>(2 * d)) + piece_far<D>(2 * d));
            };
            if (masked) {
                // A weight of zero does not keep a value that is no number from
                // the rows that do not see it: such values go to the rows that
                // do one by one, and are zeros for the products.
                bool odd = false;
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    odd |= any_nonfinite(*reinterpret_cast<const u32x4*>(vt + 1024 * i + 16 * lane));
                if (__any(odd)) {
#pragma unroll 1
                    for (int p = 0; p < 16; ++p) {
#pragma unroll
                        for (int t = 0; t < QT; ++t) {
                            const uint64_t w64 = __builtin_bit_cast(uint64_t, pw[t]);
                            const uint32_t w32 = __shfl((int)(uint32_t)(p & 2 ? w64 >> 32 : w64), (p >> 2) * 16 + col);
                            const float w = bf16_bits_to_f32(p & 1 ? w32 >> 16 : w32 & 0xFFFFu);
                            const bool see = !gone && sees(a, p0 + p, pos[t]);
#pragma unroll
                            for (int d = 0; d < D / 16; ++d)
                                add_nonfinite(o[t][d], vt + v_at<D>(p, 16 * d + 4 * G), see, w);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < NI; ++i) zero_nonfinite(vt + 1024 * i + 16 * lane);
                }
            }
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
        __syncthreads();  // and every wave is done with its ring
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
        const bool whole = u0 == 0 && u1 == f.s.nu;
        float* part = a.part + (size_t)(2 * blockIdx.x + (u0 == 0 ? 1 : 0)) * rows_part(D, QT);
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
                store4(a.out + (int64_t)(f.s.first + tok) * a.ld_out + h * D + d, v, ls);
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

// The cut tiles: wave (boundary, row) joins the parts of the tile in which
// boundary blockIdx.x + 1 is the first, in the order of the line.
template <int D, int QT>
__global__ void __launch_bounds__(256) attn_paged_rows_merge_kernel(PagedAttnArgs a, int grid) {
    constexpr int UNIT = rows_unit(D), ROWS = 16 * QT, RW = D / 64;
    const int lane = threadIdx.x & 63;
    const int r = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
    Scan sc;
    const uint64_t total = scan_all<ROWS, UNIT>(a, lane, sc);
    const uint32_t parts = part_count(total, grid), w = blockIdx.x + 1;
    if (w >= parts) return;
    const uint64_t x = part_begin(total, parts, w);
    const Found f = scan_find<ROWS, UNIT>(a, lane, sc, x);
    if (f.u == 0 || part_begin(total, parts, w - 1) > f.tile0) return;
    if (r >= min(ROWS, f.s.n * a.g - f.rt * ROWS)) return;
    const uint64_t tile1 = f.tile0 + f.s.nu;
    // Part w - 1 holds the tile's begin in its second place, the later ones
    // theirs in the first.
    auto place = [&](uint32_t v) { return a.part + (size_t)(2 * v + (v == w - 1 ? 1 : 0)) * rows_part(D, QT); };
    uint32_t last = w;
    while (last + 1 < parts && part_begin(total, parts, last + 1) < tile1) ++last;
    float mx = kNoMax;
    for (uint32_t v = w - 1 + lane; v <= last; v += 64) mx = fmaxf(mx, place(v)[ROWS * D + r]);
    for (int k = 32; k; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k));
    float acc[RW] = {}, ls = 0.0f;
#pragma unroll 4
    for (uint32_t v = w - 1; v <= last; ++v) {
        const float* p = place(v);
        const float fac = __builtin_amdgcn_exp2f(p[ROWS * D + r] - mx);
        ls = __builtin_fmaf(p[ROWS * (D + 1) + r], fac, ls);
        float t[RW];
        __builtin_memcpy(t, p + (size_t)r * D + RW * lane, sizeof(t));
#pragma unroll
        for (int e = 0; e < RW; ++e) acc[e] = __builtin_fmaf(t[e], fac, acc[e]);
    }
    const int rr = r + f.rt * ROWS, tok = rr / a.g, h = f.kvh * a.g + (rr - tok * a.g);
    uint16_t* dst = a.out + (int64_t)(f.s.first + tok) * a.ld_out + h * D + RW * lane;
#pragma unroll
    for (int e = 0; e < RW; ++e) dst[e] = ls == 0.0f ? (uint16_t)0 : bf16_rne_bits(acc[e] / ls);
}

}  // namespace

}  // namespace alv

using namespace alv;

namespace alv {
namespace {

// How a call's work is spread.
struct AttnPlan {
    int qt;      // row tiles of 16 in the streaming kernel
    int64_t row_limit;
    int grid;
    uint64_t part_bytes;
};

AttnPlan attn_plan(int heads, int kv_heads, int D, int B, int T, int max_q) {
    AttnPlan p{};
    const int64_t g = heads / kv_heads;
    const int64_t rows = (max_q > 0 ? std::min(max_q, T) : (T + B - 1) / B) * g;
    const int qt_max = D <= 128 ? 4 : (D == 256 ? 2 : 1);
    p.qt = std::min(qt_max, rows <= 16 ? 1 : (rows <= 32 ? 2 : 4));
    p.row_limit = INT64_MAX;
    p.grid = device_cus();
    p.part_bytes = (uint64_t)p.grid * 2 * 16 * p.qt * (D + 2) * sizeof(float);
    return p;
}

template <int D, int QT>
int launch_rows(const PagedAttnArgs& a, const AttnPlan& p, hipStream_t s) {
    constexpr int lds = rows_lds(D, QT);
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    const void* k = reinterpret_cast<const void*>(&attn_paged_rows_kernel<D, QT>);
    if (int rc = hip_check(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute"))
        return rc;
    hipLaunchKernelGGL((attn_paged_rows_kernel<D, QT>), dim3(p.grid), dim3(64 * rows_waves(D)), lds, s, a);
    if (int rc = hip_check(hipGetLastError(), "attn_paged_rows_kernel launch")) return rc;
    hipLaunchKernelGGL((attn_paged_rows_merge_kernel<D, QT>), dim3(p.grid - 1, 4 * QT), dim3(256), 0, s, a, p.grid);
    return hip_check(hipGetLastError(), "attn_paged_rows_merge_kernel launch");
}

template <int D>
int launch_d(const PagedAttnArgs& a, const AttnPlan& p, hipStream_t s) {
    if (p.qt == 1) return launch_rows<D, 1>(a, p, s);
    if constexpr (D <= 256)
        if (p.qt == 2) return launch_rows<D, 2>(a, p, s);
    if constexpr (D <= 128) return launch_rows<D, 4>(a, p, s);
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
    const AttnPlan p = attn_plan(heads, kv_heads, D, B, T, max_q);
    if (!workspace || workspace_bytes < p.part_bytes)
        return fail(ALV_ERR_ARG, "workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
                    (unsigned long long)p.part_bytes);
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(ALV_ERR_ALIGN, "workspace needs 16-byte alignment");
    a.part = static_cast<float*>(workspace);
    a.row_limit = p.row_limit;
    const hipStream_t s = (hipStream_t)stream;
    switch (D) {
        case 64: return launch_d<64>(a, p, s);
        case 128: return launch_d<128>(a, p, s);
        case 256: return launch_d<256>(a, p, s);
        default: return launch_d<512>(a, p, s);
    }
}
