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
//
// Groups of sequences that share their first positions (MIX): each group is one more
// sequence, of all its members' rows over the shared positions alone, and the batch's
// own run over what is behind. The kernels take the groups and the sequences alike, by
// their rows; what the parts of a row come to is kept, unnormalised, with its maximum
// and sum, and a last launch joins them.
#pragma once

#include <limits.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.h"
#include "q4_device.h"
#include "row_norm.h"

namespace alv {

namespace {

struct PagedAttnArgs {
    PagedBatch b;
    PagedGroups gr;
    const uint16_t* q;
    int64_t ld_q;
    const void* kpages;  // bf16, or codes (E8)
    const void* vpages;
    int64_t k_stride, v_stride;
    const uint8_t* scales;
    int64_t s_stride;
    int heads, kv_heads, g, g_shift;  // g: q heads of a kv head; its logarithm, -1: not a power of two
    int window, sinks;
    float scale;
    uint16_t* out;
    int64_t ld_out;
    int64_t row_limit;  // sequences of more rows (tokens times q heads per kv head) are not this launch's
    int max_tiles;      // tiles of all sequences, per kv head, at most
    int max_items;      // tiles (times kv heads) that may be split: no more than slots; 0: none
    int slots;          // parts that run at once
    int* tab;           // for the merge: how many tiles, then kTabInts for each
    int* cuts;          // for the streaming kernel's: kTabInts for each workgroup
    float* part;
    // MIX: what a row's part comes to where one workgroup had all of it, D values and a
    // maximum and sum for each (row, head): over what is shared, and behind,
    float* kept[2];
    float* kept_ml[2];
    int4* recs;         // where the parts of each are (Rec), those over what is shared first,
    float* tile_part;   // and the tiles' parts
    int grid, tile_places;  // streaming workgroups; parts of tiles that there is room for
};

template <bool E8>
using PageValue = std::conditional_t<E8, uint8_t, uint16_t>;

typedef short s16x4 __attribute__((__vector_size__(4 * sizeof(short))));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
typedef int i32x2 __attribute__((__vector_size__(2 * sizeof(int))));
typedef __attribute__((address_space(3))) i32x2* lds_i32x2;

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
// The same of 4 bytes for each of the first N lanes.
template <int N>
__device__ __forceinline__ void load_lds4(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t lds) {
    if ((threadIdx.x & 63) < N)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
                     :
                     : "v"(voff), "s"(r), "s"(lds)
                     : "memory", "m0");
}
#pragma clang diagnostic pop

// At most N of this wave's loads are still in flight.
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A barrier for what is in LDS: the waves' stores to memory go on (__syncthreads waits for
// them, 1 us and more at a tile's end).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A buffer over [base, base + bytes), the same for the whole wave.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t wave_rsrc(const void* base, uint32_t bytes) {
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

// ---- 8-bit pages ---------------------------------------------------------------------
//
// Codes become bf16 operands in registers (two per instruction; e4m3's four bits fit
// bf16's eight, so nothing is rounded), times a power of two at no cost: K's, of the
// lane's position. A lane's codes of V are several positions': V's powers are factors of
// the weights instead (exact in float32; where tiles are widened ahead of LDS, they too
// go into the conversion).

// Eight codes times a power of two.
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi, float power) {
    typedef __bf16 bf16x2 __attribute__((__vector_size__(2 * sizeof(__bf16))));
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, true);
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2,
                                   3, 4, 5, 6, 7);
}

// The power of two of byte i of a word of biased exponents.
template <int I>
__device__ __forceinline__ float power_of_byte(uint32_t w) {
    const uint32_t b = I == 3 ? w >> 1 : w << (23 - 8 * I);
    return __builtin_bit_cast(float, b & 0x7F800000u);
}

// The streaming kernel keeps codes in LDS, 32 positions of a wave at a time; a row's
// 16-byte pieces (D / 16) stand at (piece ^ swizzle of the row): the 16 rows (of 32)
// that K's reads and the 32 (0 .. 3, 16 .. 19, 4 .. 7, 20 .. 23 by the first half of
// the lanes) that V's touch at once then fall on different banks.
template <int D>
__device__ __forceinline__ constexpr int k8_swz(int row) {
    return D == 64 ? (row >> 2) & 3 : (D == 128 ? (row >> 1) & 7 : row & 15);
}
template <int D>
__device__ __forceinline__ constexpr int v8_swz(int row) {
    return D == 64 ? ((row >> 2) & 1) | ((row >> 3) & 2)
                   : (D == 128 ? ((row >> 1) & 3) | ((row >> 2) & 4) : (row & 7) | ((row >> 1) & 8));
}
template <int D>
__device__ __forceinline__ constexpr uint32_t piece8(int c) {
    return (c & (D >= 256 ? 15 : D / 16 - 1)) * 16;
}
template <int D>
__device__ __forceinline__ constexpr uint32_t piece8_far(int c) {
    return (c & ~(D >= 256 ? 15 : D / 16 - 1)) * 16;
}
__device__ __forceinline__ i32x2 read_tr8(const unsigned char* p) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2)(p));
}

// Of N slots' powers in LDS V's from slot `have` on, behind the end, cleared: any byte may be
// there, and a weight of 0 times an infinite power is NaN. (K's make scores that the mask
// drops.)
template <int N>
__device__ __forceinline__ void clear_powers(unsigned char* pairs, int have) {
    const int i = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, here(0)));  // (the lane, no register kept)
    if (i < N && i >= have) pairs[2 * i + 1] = 0;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// What a row sees of its launch's positions: from .. cap, of these the window of its
// own position `pos` and the first tokens.
struct Sight {
    int pos, cap, from;
};
__device__ __forceinline__ bool sees(const PagedAttnArgs& a, int p, const Sight& s) {
    return p <= s.cap && p >= s.from && (a.window <= 0 || p > s.pos - a.window || p < a.sinks);
}

// 1 / l of a row, 0 for one that saw nothing.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

__device__ __forceinline__ void store4(uint16_t* dst, f32x4 v, float inv) {
    *reinterpret_cast<s16x4*>(dst) = pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
}

// Where a row's part goes that one workgroup had all of: four values v at column d of
// head h of packed row t, unnormalised, with the row's maximum and sum. `half`: over what
// is shared 0, behind 1; `alone`: the row has no other part.
template <int D, bool MIX>
__device__ __forceinline__ void finish4(const PagedAttnArgs& a, int64_t t, int h, int d, f32x4 v, float m, float l, int half,
                                        bool alone) {
    if (MIX && !alone) {
        const int64_t row = t * a.heads + h;
        *reinterpret_cast<f32x4*>(a.kept[half] + row * D + d) = v;
        if (d == 0) {
            a.kept_ml[half][2 * row] = m;
            a.kept_ml[half][2 * row + 1] = l;
        }
        return;
    }
    store4(a.out + t * a.ld_out + h * D + d, v, inverse(l));
}

// The same of RW values per lane, a row per wave.
template <int D, bool MIX>
__device__ __forceinline__ void finish_row(const PagedAttnArgs& a, int64_t t, int h, int lane, const float (&acc)[D / 64], float m,
                                           float l, int half, bool alone) {
    constexpr int RW = D / 64;
    if (MIX && !alone) {
        const int64_t row = t * a.heads + h;
#pragma unroll
        for (int e = 0; e < RW; ++e) a.kept[half][row * D + RW * lane + e] = acc[e];
        if (lane == 0) {
            a.kept_ml[half][2 * row] = m;
            a.kept_ml[half][2 * row + 1] = l;
        }
        return;
    }
    const float inv = inverse(l);
    uint16_t* dst = a.out + t * a.ld_out + h * D + RW * lane;
#pragma unroll
    for (int e = 0; e < RW; ++e) dst[e] = bf16_rne_bits(acc[e] * inv);
}

// Where a row's part is: {first place, places, row of the tile, positions shared}. Places
// are the streaming workgroups' (w's second, then the first ones of w + 1, ...) or, with
// kTileRec in the row, the tiles' parts (a.kv_heads apart). No places: what it comes to
// was kept, or (kDone) is the row's output.
constexpr int kWhole = 0, kDone = -1, kTileRec = 1 << 16;

// One sequence of a launch (lane's own): rows, positions and where they begin.
struct SeqIn {
    int first, n, len;  // len: positions up to which it runs
    int seq;            // whose row of the table they are in
    int from;           // what precedes is shared; of a group: sequence behind its last
    int lo;             // position of the first row (of a group: the lowest of any row, with a window)
    bool here, ok;      // has rows in the batch; well formed
};

// The groups take whole steps of 64, the sequences follow.
template <bool MIX>
__device__ __forceinline__ int group_steps(const PagedAttnArgs& a) {
    return MIX ? (a.gr.n + 63) & ~63 : 0;
}
template <bool MIX>
__device__ __forceinline__ int seq_count(const PagedAttnArgs& a) {
    return group_steps<MIX>(a) + a.b.B;
}

// The packed rows of group `start` .. end - 1 that are the batch's (none: nothing is shared).
struct GroupRows {
    int first, n;
};
__device__ __forceinline__ GroupRows group_rows(const PagedAttnArgs& a, int start, int end) {
    const int first = max(0, a.b.q_start[start]), last = min(a.b.T, a.b.q_start[end]);
    return {first, last > first ? last - first : 0};
}

// Group j0 + lane over what it shares (j0 uniform).
__device__ __forceinline__ SeqIn group_in(const PagedAttnArgs& a, int j0, int lane) {
    SeqIn s{};
    const int j = j0 + lane;
    int end = 0;
    if (j < a.gr.n) {
        s.seq = a.gr.start[j];
        end = a.gr.start[j + 1];
        s.len = group_len(a.b, s.seq, end, a.gr.len[j]);
        if (s.len > 0) {
            const GroupRows r = group_rows(a, s.seq, end);
            s.first = r.first, s.n = r.n;
            s.here = s.ok = r.n > 0;
            s.len = s.here ? s.len : 0;
            s.from = s.here ? end : 0;
        }
    }
    if (a.window > 0) {
        for (uint64_t left = __ballot(s.here); left; left &= left - 1) {
            const int l = __builtin_ctzll(left);
            const int hi = __builtin_amdgcn_readlane(end, l);
            int low = INT_MAX;
            for (int c = __builtin_amdgcn_readlane(s.seq, l) + lane; c < hi; c += 64) {
                const int n = a.b.q_start[c + 1] - a.b.q_start[c];
                if (n > 0) low = min(low, a.b.kv_len[c] - n);
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) low = min(low, __shfl_xor(low, o));
            if (lane == l) s.lo = max(0, low);
        }
    }
    return s;
}

// Sequence b0 + lane of the batch (b0 uniform), behind what it shares. groups: the first
// 64 as group_in gave them, where the caller has them (two trips to memory less).
template <bool MIX>
__device__ __forceinline__ SeqIn batch_in(const PagedAttnArgs& a, int b0, int lane, const SeqIn* groups = nullptr) {
    SeqIn s{};
    const int b = b0 + lane;
    if (b < a.b.B) {
        s.seq = b;
        s.first = a.b.q_start[b];
        s.n = a.b.q_start[b + 1] - s.first;
        s.len = a.b.kv_len[b];
        s.here = s.first >= 0 && s.n > 0 && (int64_t)s.first + s.n <= a.b.T;
        s.ok = s.n <= s.len && s.len <= a.b.max_pos;
        s.lo = s.len - s.n;
    }
    if constexpr (MIX) {
        for (int j0 = 0; j0 < a.gr.n; j0 += 64) {
            const int j = j0 + lane;
            int lo = INT_MAX, hi = 0, len = 0;
            GroupRows rows{};
            if (j0 == 0 && groups) {
                if (j < a.gr.n) {  // (none shared: no end)
                    lo = groups->seq, hi = groups->from, len = groups->len;
                    rows = {groups->first, groups->n};
                }
            } else if (j < a.gr.n) {
                lo = a.gr.start[j];
                hi = a.gr.start[j + 1];
                len = group_len(a.b, lo, hi, a.gr.len[j]);
                if (len > 0) rows = group_rows(a, lo, hi);
            }
            int l = 0;  // the last group that begins at b or before
#pragma unroll
            for (int o = 32; o; o >>= 1)
                if (__shfl(lo, l + o) <= b) l += o;
            const int end = __shfl(hi, l), shared = __shfl(len, l), begin = __shfl(lo, l);
            const int first = __shfl(rows.first, l), n = __shfl(rows.n, l);
            // (beside members that are malformed the group's rows may not be all of this one's)
            if (begin <= b && b < end && s.here && first <= s.first && s.first - first <= n - s.n) s.from = shared;
        }
        if (!s.ok) s.from = 0;
    }
    return s;
}

template <bool MIX>
__device__ __forceinline__ SeqIn seq_in(const PagedAttnArgs& a, int b0, int lane, const SeqIn* groups = nullptr) {
    if constexpr (MIX)
        if (b0 < group_steps<MIX>(a)) return group_in(a, b0, lane);
    return batch_in<MIX>(a, b0 - group_steps<MIX>(a), lane, groups);
}

// Of a group: the positions of NR packed rows (lane's own each) of the sequences seq ..
// end - 1, by the whole wave.
template <int NR>
__device__ __forceinline__ void row_positions(const PagedAttnArgs& a, int seq, int end, const int (&t)[NR], int (&pos)[NR]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < NR; ++r) pos[r] = -1;
    for (int c0 = seq; c0 < end; c0 += 64) {
        const int c = c0 + lane;
        int lo = INT_MAX, off = 0;
        if (c < end) {
            lo = a.b.q_start[c];
            off = a.b.kv_len[c] - a.b.q_start[c + 1];  // its last row is at kv_len - 1
        }
        const int low = __builtin_amdgcn_readlane(lo, 0);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            int l = 0;  // the last sequence that begins at this row or before
#pragma unroll
            for (int o = 32; o; o >>= 1)
                if (__shfl(lo, l + o) <= t[r]) l += o;
            const int v = t[r] + __shfl(off, l);
            if (low <= t[r]) pos[r] = v;
        }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) pos[r] = min(max(pos[r], -1), a.b.max_pos);
}

__device__ __forceinline__ int min64(int v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = min(v, __shfl_xor(v, o));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int max64(int v) { return -min64(-v); }

// The units of positions that a run begins with, before it goes on from `lo`, the first
// that a window holds: `us` units of first tokens from 0 on, then from unit `ulo` on. own:
// behind the `from` positions that a group shares; where the gap is no more units than they
// are, straight from there.
struct Begin {
    int us, ulo;
};
template <int UNIT>
__device__ __forceinline__ Begin begin_units(const PagedAttnArgs& a, int lo, bool own, int from) {
    if (own && a.sinks <= from) return {0, max(lo, from) / UNIT};
    const int ulo = lo / UNIT, us = min((min(a.sinks, lo) + UNIT - 1) / UNIT, ulo);
    if (own && us + from / UNIT >= ulo) return {0, from / UNIT};
    return {us, ulo};
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
template <int D, bool E8>
__device__ void plain_row(const PagedAttnArgs& a, int seq, int kvh, const uint16_t* q, const Sight pos, int us, int ulo, int unit,
                          int u0, int u1, int lane, float (&acc)[D / 64], float& m, float& l) {
    constexpr int RW = D / 64;
    using T = PageValue<E8>;
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
            float s = -__builtin_inff(), up = 1.0f;
            const int64_t slot = ((int64_t)kvh << a.b.shift) + (p & ((1 << a.b.shift) - 1));
            if (page >= 0) {
                const T* row = static_cast<const T*>(a.kpages) + page * a.k_stride + slot * D;
                s = 0.0f;
                for (int i = 0; i < D / 8; ++i) {
                    const u32x4 qv = reinterpret_cast<const u32x4*>(q)[i];
                    u32x4 kv;
                    if constexpr (E8) {
                        const uint2 codes = reinterpret_cast<const uint2*>(row)[i];
                        kv = __builtin_bit_cast(u32x4, widen8(codes.x, codes.y, 1.0f));
                    } else {
                        kv = reinterpret_cast<const u32x4*>(row)[i];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t kw = kv[e], qw = qv[e];
                        s = __builtin_fmaf(bf16_bits_to_f32(kw & 0xFFFFu), bf16_bits_to_f32(qw & 0xFFFFu), s);
                        s = __builtin_fmaf(bf16_bits_to_f32(kw >> 16), bf16_bits_to_f32(qw >> 16), s);
                    }
                }
                if constexpr (E8) {
                    const uint32_t e = *reinterpret_cast<const uint16_t*>(a.scales + page * a.s_stride + 2 * slot);
                    s *= power_of_byte<0>(e);
                    up = power_of_byte<1>(e);
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
            if constexpr (E8) w *= up;
            for (uint64_t left = __ballot(page >= 0); left; left &= left - 1) {
                const int j = __builtin_ctzll(left), pj = pb + j;
                const float wj = __shfl(w, j);
                const T* v = static_cast<const T*>(a.vpages) + __shfl(page, j) * a.v_stride +
                             (((int64_t)kvh << a.b.shift) + (pj & ((1 << a.b.shift) - 1))) * D + RW * lane;
#pragma unroll
                for (int e = 0; e < RW; ++e)
                    acc[e] = __builtin_fmaf(wj, E8 ? __builtin_amdgcn_cvt_f32_fp8(v[e], 0) : bf16_bits_to_f32(v[e]), acc[e]);
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
//
// 8-bit pages: half the bytes, so twice the positions in each block and, where its LDS
// holds both, two workgroups per CU, one computing while the other waits (not at 512, nor
// with q in LDS too: there as many waves in one, where half of them were left when two
// were counted on: 16 tokens of 64 sequences of 116 to 3016 positions, 16 heads of 256 on 8
// 205 -> 131 us, 32 of 128 on 8 220 -> 128). 64 sequences of 100 to 8000 positions, 32 q
// heads of 64 on 8: 63 us, 4.5 TB/s, of them 2 for the merge; the same over bf16 pages 114.

// With groups or 8-bit pages a tile has kTileCost places in the line ahead of its units,
// what its begin and end cost beside them: parts of many short tiles were the last to end
// (64 sequences of 20 to 1500 own positions: 99 thousand cycles where the median took 66).
// A part that ends among them leaves the tile to the next.
constexpr int kTileCost = 3;
constexpr int tile_cost(bool E8, bool MIX) { return E8 || MIX ? kTileCost : 0; }

// A sequence's place in the line, per lane of the scan.
struct RowsSeq {
    int first, n, len;
    int seq, from;    // see SeqIn
    int tiles;        // row tiles (of each kv head)
    int us, ulo, nu;  // units of first tokens; first unit of the window; units in all
};

// TWO: two workgroups per CU (rows_two), else one.
constexpr int rows_waves(int D, bool TWO) { return (D == 512 ? 2 : (D == 64 ? 8 : 4)) / (TWO ? 2 : 1); }
// A wave's block: 16 positions' K and V, or 32 of 8-bit ones and their powers.
constexpr int rows_block(bool E8) { return E8 ? 32 : 16; }
constexpr int rows_stage(int D, bool E8) { return 64 * D + (E8 ? 64 : 0); }
constexpr int rows_stages(int D) { return 131072 / (rows_waves(D, false) * 64 * D); }
constexpr int rows_unit(int D, bool E8, bool TWO) { return rows_block(E8) * rows_waves(D, TWO); }
// The waves' outputs at a tile's end, rows padded to spread over the banks.
constexpr int rows_out_ld(int D) { return D + 4; }
// Whether q's operands stay in LDS rather than registers: where they and the
// output take more than half of a wave's 256 (the rest would spill).
constexpr bool rows_q_lds(int D, int QT) { return QT * D > 256; }
// The waves' flags of outputs that are not finite, an int each, at the end.
constexpr int rows_flags(int D, bool TWO) { return (4 * rows_waves(D, TWO) + 15) / 16 * 16; }
constexpr int rows_lds(int D, int QT, bool E8, bool TWO) {
    const int NW = rows_waves(D, TWO), ring = NW * rows_stages(D) * rows_stage(D, E8);
    const int outs = NW * 16 * QT * (rows_out_ld(D) * 4);
    return (ring > outs ? ring : outs) + 2 * NW * 16 * QT * 4 + (rows_q_lds(D, QT) ? 32 * QT * D : 0) +
           rows_flags(D, TWO);
}
constexpr int rows_mls(int D, int QT, bool E8, bool TWO) {  // where the waves' maxima and sums stand; q behind them
    return rows_lds(D, QT, E8, TWO) - rows_flags(D, TWO) - 2 * rows_waves(D, TWO) * 16 * QT * 4 -
           (rows_q_lds(D, QT) ? 32 * QT * D : 0);
}
// Whether two workgroups share a CU: 8-bit pages, and where both fit its LDS.
constexpr int kCuLds = 160 * 1024;
constexpr bool rows_two(int D, int QT, bool E8) { return E8 && D <= 256 && 2 * rows_lds(D, QT, E8, true) <= kCuLds; }
// Floats of one workspace place: outputs, maxima, sums.
constexpr int rows_part(int D, int QT) { return 16 * QT * (D + 2); }

constexpr int kPartsPerTile = 64;
constexpr int kTabInts = 8;  // an entry of the merges' tables

struct Scan {
    RowsSeq s;          // this lane's sequence
    uint64_t incl;      // work of the sequences of this step up to and with this lane's
    uint64_t base, sum; // work before this step; of this step
    int b0;             // the step's first sequence
    uint32_t tiles;     // of the whole batch, no more than 2^31 (scan_all)
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// The token that row r (tokens times q heads of the group) belongs to: a division is 25
// instructions, one after the other, several times a tile.
__device__ __forceinline__ int per_head(const PagedAttnArgs& a, int r) { return a.g_shift >= 0 ? r >> a.g_shift : r / a.g; }
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, l);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l);
    return ((uint64_t)hi << 32) | lo;
}

template <int ROWS, int UNIT, int COST, bool MIX>
__device__ __forceinline__ void scan_step(const PagedAttnArgs& a, int b0, int lane, uint64_t base, Scan& sc,
                                          const SeqIn* groups = nullptr) {
    const bool suf = MIX && b0 >= group_steps<MIX>(a);
    const SeqIn in = seq_in<MIX>(a, b0, lane, groups);
    RowsSeq s{};
    s.first = in.first, s.n = in.n, s.len = in.len, s.seq = in.seq, s.from = in.from;
    uint64_t w = 0;
    const int64_t rows = in.here ? (int64_t)s.n * a.g : 0;
    if (in.here && rows <= a.row_limit) {
        s.tiles = (int)((rows + ROWS - 1) / ROWS);
        if (in.ok) {
            const int lo = a.window > 0 ? max(0, in.lo + 1 - a.window) : 0;
            const Begin at = begin_units<UNIT>(a, lo, suf, s.from);
            s.us = at.us, s.ulo = at.ulo;
            // (one at least: there may be nothing within the window, nothing behind what is shared)
            s.nu = s.us + max((s.len + UNIT - 1) / UNIT - s.ulo, !MIX ? INT_MIN : s.us ? 0 : 1);
        } else {
            s.len = 0;  // malformed: one unit that sees nothing
            s.nu = 1;
        }
        w = (uint64_t)s.tiles * a.kv_heads * (COST + s.nu);
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

// The first step (and `next`, the second: the first of sequences behind up to 64
// groups), and the work of the whole batch.
template <int ROWS, int UNIT, int COST, bool MIX>
__device__ __forceinline__ uint64_t scan_all(const PagedAttnArgs& a, int lane, Scan& sc, Scan& next) {
    scan_step<ROWS, UNIT, COST, MIX>(a, 0, lane, 0, sc);
    uint64_t total = sc.sum;
    uint32_t tiles = sc.s.nu ? min(sc.s.tiles, kPartsPerTile) : 0;
    for (int b0 = 64; b0 < seq_count<MIX>(a); b0 += 64) {
        Scan t;
        SeqIn groups{};
        groups.seq = sc.s.seq, groups.from = sc.s.from, groups.len = sc.s.len;
        groups.first = sc.s.first, groups.n = sc.s.n;
        scan_step<ROWS, UNIT, COST, MIX>(a, b0, lane, total, t, MIX ? &groups : nullptr);
        if (MIX && b0 == 64) next = t;
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
    bool pre;         // of a group, over what it shares
    int at;           // place in the tile: COST, then its units
    uint64_t tile0;   // the tile's place in the line
};

// The tile and unit at place x of the line (x < total; calls with x rising).
template <int ROWS, int UNIT, int COST, bool MIX>
__device__ __forceinline__ Found scan_find(const PagedAttnArgs& a, int lane, Scan& sc, uint64_t x) {
    while (x >= sc.base + sc.sum) scan_step<ROWS, UNIT, COST, MIX>(a, sc.b0 + 64, lane, sc.base + sc.sum, sc);
    const uint64_t m = __ballot(sc.base + sc.incl > x);
    const int l = __builtin_ctzll(m);
    Found f;
    f.seq = MIX ? __builtin_amdgcn_readlane(sc.s.seq, l) : sc.b0 + l;
    f.pre = MIX && sc.b0 < group_steps<MIX>(a);
    f.s.from = !MIX ? 0 : __builtin_amdgcn_readlane(sc.s.from, l);
    f.s.first = __builtin_amdgcn_readlane(sc.s.first, l);
    f.s.n = __builtin_amdgcn_readlane(sc.s.n, l);
    f.s.len = __builtin_amdgcn_readlane(sc.s.len, l);
    f.s.tiles = __builtin_amdgcn_readlane(sc.s.tiles, l);
    f.s.us = __builtin_amdgcn_readlane(sc.s.us, l);
    f.s.ulo = __builtin_amdgcn_readlane(sc.s.ulo, l);
    f.s.nu = __builtin_amdgcn_readlane(sc.s.nu, l);
    const uint32_t places = COST + f.s.nu;
    const uint64_t seq_work = (uint64_t)f.s.tiles * a.kv_heads * places;
    const uint64_t start = sc.base + lane_u64(sc.incl, l) - seq_work;
    const uint64_t in = x - start;
    const uint64_t tile = div32(in, places);
    f.at = uniform((int)(in - tile * places));
    f.tile0 = start + tile * places;
    f.kvh = f.s.tiles == 1 ? uniform((int)tile) : uniform((int)((uint32_t)tile / (uint32_t)f.s.tiles));
    f.rt = uniform((int)((uint32_t)tile - (uint32_t)f.kvh * f.s.tiles));
    return f;
}

// The tile behind f in the line, if it is the same sequence's.
template <int COST>
__device__ __forceinline__ bool scan_next(const PagedAttnArgs& a, Found& f) {
    const bool last = f.rt + 1 == f.s.tiles;
    if (last && f.kvh + 1 == a.kv_heads) return false;
    f.kvh += last;
    f.rt = last ? 0 : f.rt + 1;
    f.at = 0;
    f.tile0 += COST + f.s.nu;
    return true;
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

template <int D, int QT, bool E8, bool MIX>
__global__ void __launch_bounds__((64 * rows_waves(D, rows_two(D, QT, E8))), 2) attn_paged_rows_kernel(PagedAttnArgs a) {
    constexpr bool TWO = rows_two(D, QT, E8);
    constexpr int NW = rows_waves(D, TWO), NS = rows_stages(D), UNIT = rows_unit(D, E8, TWO), ROWS = 16 * QT;
    constexpr int BP = rows_block(E8), NH = BP / 16;  // positions of a block, 16 at a time (within a page)
    constexpr int STAGE = rows_stage(D, E8);
    constexpr int NC = E8 ? D / 16 : D / 8;  // 16-byte pieces of a row
    constexpr int NI = NC / 4;            // loads of 64 pieces for 16 positions of K (of V)
    constexpr int HALF = 32 * D;          // bytes of a block's K
    constexpr int RPL = 64 / NC;          // rows of one load
    constexpr int LOADS = NH * 2 * NI + E8;   // of a block, at least
    constexpr int COST = tile_cost(E8, MIX);
    using T = PageValue<E8>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, G = lane >> 4;
    Scan sc, next;
    const uint64_t total = scan_all<ROWS, UNIT, COST, MIX>(a, lane, sc, next);
    const Cut cut = make_cut(total, part_count(total, sc, gridDim.x));
    // The tile that begins in this part and ends in a later one, for the merge: the last
    // part it is in, first row of its sequence, tile, rows, kv head.
    [[maybe_unused]] int* const cut_tile = a.cuts + kTabInts * blockIdx.x;
    if (!MIX && threadIdx.x == 0) cut_tile[0] = 0;
    if (blockIdx.x >= cut.n) return;
    uint64_t x = cut.begin(blockIdx.x);
    if (MIX && seq_count<MIX>(a) > 64 && x >= next.base) sc = next;  // (a step anew is 3 us)
    const uint64_t end = cut.begin(blockIdx.x + 1);

    unsigned char* ring = smem + wave * NS * STAGE;
    const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_addr(ring));
    float* mls = reinterpret_cast<float*>(smem + rows_mls(D, QT, E8, TWO));  // [wave][max | sum][row]
    int* odds = reinterpret_cast<int*>(smem + rows_lds(D, QT, E8, TWO) - rows_flags(D, TWO));
    const float c = fmaxf(a.scale * kLog2e, kMinScale);
    const int S = 1 << a.b.shift;
    // Byte offsets that stay: this lane's piece of a load (memory side), of a K
    // read and of a V read (LDS side).
    constexpr auto kz = [](int row) { return E8 ? k8_swz<D>(row) : k_swz<D>(row); };
    constexpr auto vz = [](int row) { return E8 ? v8_swz<D>(row) : v_swz<D>(row); };
    const uint32_t dma_k = (lane / NC) * (16 * NC) + ((lane % NC) ^ kz(lane / NC)) * 16;
    const uint32_t dma_v = (lane / NC) * (16 * NC) + ((lane % NC) ^ vz(lane / NC)) * 16;
    const uint32_t rd_k = col * (16 * NC) + (G ^ kz(col)) * 16;
    // V's transposing reads: 4 rows of a lane group's, or 8, the ones whose scores it has.
    const int vrow = E8 ? 4 * G + (col >> 1 & 3) + 16 * (col >> 3) : 4 * G + (col >> 2);
    const uint32_t rd_v = vrow * (16 * NC) + ((E8 ? 0 : (col >> 1) & 1) ^ vz(vrow)) * 16 + (col & 1) * 8;

    Found f;
    for (bool begun = false; x < end; begun = true) {
        if (!begun || !scan_next<COST>(a, f)) f = scan_find<ROWS, UNIT, COST, MIX>(a, lane, sc, x);
        const int u0 = max(0, f.at - COST), u1 = uniform((int)min((int64_t)f.s.nu, (int64_t)(end - f.tile0) - COST));
        if (COST > 0 && u1 <= 0) break;
        x = f.tile0 + COST + u1;
        const int nrows = min(ROWS, f.s.n * a.g - f.rt * ROWS);
        const int nblk = f.s.len > 0 ? u1 - u0 : 0;  // this wave's blocks
        const bool pre = MIX && f.pre, suf = MIX && !f.pre, alone = suf && f.s.from == 0;
        auto block_pos = [&](int j) {
            const int u = u0 + j;
            return (u < f.s.us ? u : u - f.s.us + f.s.ulo) * UNIT + BP * wave;
        };
        // The pages of this wave's blocks, 64 at a time, one per lane.
        const int32_t* table = a.b.table + (int64_t)f.seq * a.b.ld_table;
        int pages0 = 0;
        uint32_t gone_bits = 0;  // by buffer: its page (of the first 16, of the others) is missing
        int pages = -1;                        // bf16
        [[maybe_unused]] uint64_t ka = 0, va = 0, sa = 0;  // 8-bit: where a block's K, V and powers begin
        [[maybe_unused]] int have = 0;         // and how many positions there are; bit 8: its page is missing
        // (pages of 16: a block's halves each)
        const int halves = E8 && a.b.shift < 5 ? 1 : 0;
        auto load_pages = [&](int j0) {
            pages0 = j0;
            const int j = j0 + (lane >> halves), p = block_pos(j) + 16 * (lane & halves);
            // (what a group shares is not this sequence's to read: its entries may be any)
            pages = j < nblk && p < f.s.len && (!suf || p >= f.s.from) ? table[p >> a.b.shift] : -1;
            if ((unsigned)pages >= (unsigned)a.b.pages) pages = -1;
            if constexpr (E8) {
                const int64_t slot = ((int64_t)f.kvh << a.b.shift) + (p & (S - 1));
                const int64_t page = max(pages, 0);
                ka = reinterpret_cast<uint64_t>(a.kpages) + page * a.k_stride + slot * D;
                va = reinterpret_cast<uint64_t>(a.vpages) + page * a.v_stride + slot * D;
                sa = reinterpret_cast<uint64_t>(a.scales) + page * a.s_stride + slot * 2;
                have = pages < 0 ? 256 : max(0, min(halves ? 16 : 32, f.s.len - p));
            }
        };
        // Load i brings rows RPL i .. of RPL each; the swizzles are exclusive ors of the
        // row's bits, so the lane's offset within the rows of one load serves all, with
        // the load's own bits applied.
        // Past the sequence's end, and where the page is missing, zeros arrive.
        auto issue = [&](int j) {
            const uint32_t dst = ring_lds + (uint32_t)(j % NS) * STAGE;
            if constexpr (E8) {
                if (j - pages0 >= 64 >> halves) load_pages(j);
                auto part = [&](auto count, int at, uint32_t half) __attribute__((always_inline)) {
                    constexpr int N = decltype(count)::value;  // rows: 16, or all 32
                    const uint64_t k = lane_u64(ka, at), v = lane_u64(va, at), s = lane_u64(sa, at);
                    const int n = __builtin_amdgcn_readlane(have, at);
                    const uint32_t rows = n & 63;
                    gone_bits |= (uint32_t)(n >> 8) * (N == 32 ? 3u : 1u << half) << (NH * (j % NS));
                    const __amdgpu_buffer_rsrc_t rk = make_rsrc(reinterpret_cast<const void*>(k), rows * D);
                    const __amdgpu_buffer_rsrc_t rv = make_rsrc(reinterpret_cast<const void*>(v), rows * D);
                    const uint32_t to = dst + half * (16 * D);
#pragma unroll
                    for (int i = 0; i < N / RPL; ++i)
                        load_lds16(rk, dma_k ^ (kz(RPL * i) * 16), 1024 * i, to + 1024 * i);
#pragma unroll
                    for (int i = 0; i < N / RPL; ++i)
                        load_lds16(rv, dma_v ^ ((vz(RPL * i) ^ (half ? vz(16) : 0)) * 16), 1024 * i, to + HALF + 1024 * i);
                    // (a page's powers, 16 pairs at least, are there whatever its positions)
                    load_lds4<N / 2>(make_rsrc(reinterpret_cast<const void*>(s), rows ? 2 * N : 0), lane * 4, dst + 64 * D + 32 * half);
                };
                gone_bits &= ~(3u << (NH * (j % NS)));
                if (halves) {
                    part(std::integral_constant<int, 16>(), 2 * (j - pages0), 0);
                    part(std::integral_constant<int, 16>(), 2 * (j - pages0) + 1, 1);
                } else {
                    part(std::integral_constant<int, 32>(), j - pages0, 0);
                }
            } else {
                if (j - pages0 >= 64) load_pages(j);
                const int page = __builtin_amdgcn_readlane(pages, j - pages0), p = block_pos(j);
                const uint32_t bytes = page < 0 ? 0u : (uint32_t)max(0, min(16, f.s.len - p)) * (2 * D);
                const int64_t off = (((int64_t)f.kvh << a.b.shift) + (p & (S - 1))) * D;
                const __amdgpu_buffer_rsrc_t rk = wave_rsrc(static_cast<const T*>(a.kpages) + max(page, 0) * a.k_stride + off, bytes);
                const __amdgpu_buffer_rsrc_t rv = wave_rsrc(static_cast<const T*>(a.vpages) + max(page, 0) * a.v_stride + off, bytes);
                gone_bits = (gone_bits & ~(1u << (j % NS))) | ((uint32_t)(page < 0) << (j % NS));
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    load_lds16(rk, dma_k ^ (kz(RPL * i) * 16), 1024 * i, dst + 1024 * i);
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    load_lds16(rv, dma_v ^ (vz(RPL * i) * 16), 1024 * i, dst + HALF + 1024 * i);
            }
        };

        // This lane's rows of q, the B operand: row col of each 16, 8 columns of each 32.
        Sight pos[QT];
        int row_t[QT];
        constexpr bool QL = rows_q_lds(D, QT);
        bf16x8 q[QL ? 1 : QT][QL ? 1 : D / 32];
        u32x4* qs = reinterpret_cast<u32x4*>(smem + rows_mls(D, QT, E8, TWO) + 2 * NW * ROWS * 4) + lane;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int r = min(16 * t + col, nrows - 1) + f.rt * ROWS;
            const int tok = per_head(a, r), h = f.kvh * a.g + (r - tok * a.g);
            row_t[t] = f.s.first + tok;
            pos[t].pos = pos[t].cap = f.s.len - f.s.n + tok;
            pos[t].from = suf ? f.s.from : 0;
            // (of codes, 16 bytes of a lane's are two operands: 16 columns of each 64)
            const uint16_t* qr = a.q + (int64_t)(f.s.first + tok) * a.ld_q + h * D + (E8 ? 16 : 8) * G;
            constexpr auto q_at = [](int i) { return E8 ? 64 * (i / 2) + 8 * (i % 2) : 32 * i; };
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                if constexpr (QL) {
                    if (i % NW == wave) qs[(t * (D / 32) + i) * 64] = *reinterpret_cast<const u32x4*>(qr + q_at(i));
                } else {
                    q[t][i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(qr + q_at(i)));
                }
            }
        }
        if (nblk) load_pages(0);  // (its trip to memory beside q's)
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
        int pos_lo = f.s.len - f.s.n + per_head(a, f.rt * ROWS);
        int pos_hi = f.s.len - f.s.n + per_head(a, f.rt * ROWS + nrows - 1);
        if (pre) {
            int p[QT];
            row_positions<QT>(a, f.seq, f.s.from, row_t, p);
            int lo = INT_MAX, hi = -1;
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                pos[t].pos = p[t];
                pos[t].cap = min(p[t], f.s.len - 1);
                lo = min(lo, pos[t].cap);
                hi = max(hi, p[t]);
            }
            pos_lo = min64(lo), pos_hi = max64(hi);
        }
        f32x4 o[QT][D / 16];
        float m[QT], l[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            m[t] = kNoMax;
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) o[t][d] = f32x4{0, 0, 0, 0};
        }
#pragma unroll 1
        for (int j = 0; j < min(NS, nblk); ++j) issue(j);
        auto blocks = [&](auto count) __attribute__((always_inline)) {
            constexpr int NT = decltype(count)::value;  // row tiles of 16 that there are
#pragma unroll 1
            for (int j = 0; j < nblk; ++j) {
                // Blocks j + 1 .. j + NS - 1 may be in flight.
                if (j + NS <= nblk)
                    wait_vm<(NS - 1) * LOADS>();
                else
                    wait_vm<0>();
                const unsigned char* kt = ring + (j % NS) * STAGE;
                const unsigned char* vt = kt + HALF;
                if (E8 && j + 1 == nblk) clear_powers<BP>(ring + (j % NS) * STAGE + 64 * D, f.s.len - block_pos(j));
                f32x4 s[NH][NT];
                constexpr int KB = QT * D >= 512 ? (QT == 4 ? 1 : 2) : 0;  // K reads of codes at once, where registers are short
                [[maybe_unused]] i32x2 powers[NH];  // of this lane's positions: k's, v's in turn
#pragma unroll
                for (int hf = 0; hf < NH; ++hf) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) s[hf][t] = f32x4{0, 0, 0, 0};
                    auto product = [&](bf16x8 k, int i) __attribute__((always_inline)) {
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            if constexpr (QL)
                                s[hf][t] = mfma16x16x32(k, __builtin_bit_cast(bf16x8, qs[(t * (D / 32) + i) * 64]), s[hf][t]);
                            else
                                s[hf][t] = mfma16x16x32(k, q[t][i], s[hf][t]);
                        }
                    };
                    if constexpr (E8) {
                        powers[hf] = *reinterpret_cast<const i32x2*>(kt + 64 * D + 32 * hf + 8 * G);
                        const float kp = power_of_byte<0>(*reinterpret_cast<const uint16_t*>(kt + 64 * D + 32 * hf + 2 * col));
#pragma unroll
                        for (int i = 0; i < D / 64; ++i) {
                            if (KB > 0 && i % (KB > 0 ? KB : 1) == 0) asm volatile("" ::: "memory");
                            const u32x4 k = *reinterpret_cast<const u32x4*>(kt + hf * (16 * D) + (rd_k ^ piece8<D>(4 * i)) +
                                                                            piece8_far<D>(4 * i));
                            product(widen8(k[0], k[1], kp), 2 * i);
                            product(widen8(k[2], k[3], kp), 2 * i + 1);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < D / 32; ++i)
                            product(__builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(
                                                                   kt + (rd_k ^ piece<D>(4 * i)) + piece_far<D>(4 * i))), i);
                    }
                }
                float vp[NH][4];  // V's powers
                if constexpr (E8) {
#pragma unroll
                    for (int hf = 0; hf < NH; ++hf) {
                        const uint32_t p0 = powers[hf][0], p1 = powers[hf][1];
                        vp[hf][0] = power_of_byte<1>(p0), vp[hf][1] = power_of_byte<3>(p0);
                        vp[hf][2] = power_of_byte<1>(p1), vp[hf][3] = power_of_byte<3>(p1);
                    }
                }
                const int p0 = block_pos(j);
                const uint32_t gone = gone_bits >> (NH * (j % NS)) & ((1u << NH) - 1);
                const bool masked = gone || p0 + BP - 1 > pos_lo || (suf && p0 < f.s.from) ||
                                    (a.window > 0 && p0 <= pos_hi - a.window && p0 + BP - 1 >= a.sinks);
                if (masked) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        // Relative to p0 + 4 G, so that positions are constants; selects, no branches.
                        const int base = p0 + 4 * G, top = pos[t].cap - base, begin = pos[t].from - base;
                        const int lo = a.window > 0 ? pos[t].pos - a.window - base : INT_MIN, sk = a.sinks - base;
#pragma unroll
                        for (int hf = 0; hf < NH; ++hf) {
                            const int hi = gone >> hf & 1 ? INT_MIN : top;
                            f32x4 v = s[hf][t];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int p = 16 * hf + i;
                                bool seen = (p <= hi) & ((p > lo) | (p < sk));
                                if (MIX) seen &= p >= begin;
                                const float x = v[i];
                                v[i] = seen ? x : -__builtin_inff();
                            }
                            s[hf][t] = v;
                        }
                    }
                }
                typedef __bf16 Weights __attribute__((__vector_size__(4 * NH * sizeof(__bf16))));
                Weights pw[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float top = -__builtin_inff();
#pragma unroll
                    for (int hf = 0; hf < NH; ++hf) {
                        const float s0 = s[hf][t][0], s1 = s[hf][t][1], s2 = s[hf][t][2], s3 = s[hf][t][3];
                        const float most = fmaxf(fmaxf(s0, s1), fmaxf(s2, s3));
                        top = hf ? fmaxf(top, most) : most;
                    }
                    if (__any(__builtin_fmaf(top, c, -m[t]) > kSlack)) {
                        const float mn = fmaxf(m[t], max_groups(top) * c);
                        const float fac = __builtin_amdgcn_exp2f(m[t] - mn);
                        m[t] = mn;
                        l[t] *= fac;
#pragma unroll
                        for (int d = 0; d < D / 16; ++d) o[t][d] *= fac;
                    }
                    // Weights as bf16, the matrix cores' type: half a step, 2^-8
                    // relative each, as much as the output's own rounding (the outputs'
                    // mean error against 64 bits: 0.0021 to 0.0024, of which their own
                    // rounding is 0.0017).
#pragma unroll
                    for (int hf = 0; hf < NH; ++hf) {
                        float w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float si = s[hf][t][i];
                            w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(si, c, -m[t]));
                        }
                        l[t] += (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) pw[t][4 * hf + i] = (__bf16)(E8 ? w[i] * vp[hf][i] : w[i]);
                    }
                }
                auto read_v = [&](int d) __attribute__((always_inline)) {
                    if constexpr (E8)
                        return read_tr8(vt + (rd_v ^ piece8<D>(d)) + piece8_far<D>(d));
                    else
                        return read_tr(vt + (rd_v ^ piece<D>(2 * d)) + piece_far<D>(2 * d));
                };
                constexpr int VB = D / 16 < 8 ? D / 16 : (E8 && QT * D >= 512 ? (QT == 4 ? 2 : 4) : 8);  // V reads on their way at once
#pragma unroll
                for (int d0 = 0; d0 < D / 16; d0 += VB) {
                    std::conditional_t<E8, i32x2, s16x4> v[VB];
#pragma unroll
                    for (int d = 0; d < VB; ++d) v[d] = read_v(d0 + d);
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int d = 0; d < VB; ++d) {
                        if constexpr (E8) {
                            const bf16x8 vb = widen8(v[d][0], v[d][1], 1.0f);
#pragma unroll
                            for (int t = 0; t < NT; ++t) o[t][d0 + d] = mfma16x16x32(vb, pw[t], o[t][d0 + d]);
                        } else {
#pragma unroll
                            for (int t = 0; t < NT; ++t)
                                o[t][d0 + d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v[d], __builtin_bit_cast(s16x4, pw[t]),
                                                                                         o[t][d0 + d], 0, 0, 0);
                        }
                    }
                }
                // The buffer's reads are done before it is filled again.
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (j + NS < nblk) issue(j + NS);
            }
        };
        if (MIX && QT > 1 && nrows <= 16)
            blocks(std::integral_constant<int, 1>());
        else
            blocks(std::integral_constant<int, QT>());

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
        auto note = [&]() __attribute__((always_inline)) {  // where this tile's parts are
            if constexpr (MIX) {
                const int places = whole ? 0 : (int)cut.part_of(f.tile0 + COST + f.s.nu - 1) - (int)blockIdx.x + 1;
                for (int r = u0 == 0 ? tid : nrows; r < nrows; r += 64 * NW) {
                    const int rr = r + f.rt * ROWS, tok = per_head(a, rr), h = f.kvh * a.g + (rr - tok * a.g);
                    const int64_t row = (int64_t)(f.s.first + tok) * a.heads + h;
                    a.recs[(pre ? 0 : (int64_t)a.b.T * a.heads) + row] =
                        int4{(int)blockIdx.x, !whole ? places : (alone ? kDone : kWhole), r, f.s.from};
                }
            } else if (u0 == 0 && !whole && tid == 0) {
                cut_tile[0] = (int)cut.part_of(f.tile0 + COST + f.s.nu - 1);
                cut_tile[1] = f.s.first, cut_tile[2] = f.rt, cut_tile[3] = nrows, cut_tile[4] = f.kvh;
            }
        };
        float* part = a.part + (size_t)(2 * blockIdx.x + (u0 == 0 ? 1 : 0)) * rows_part(D, QT);
        if (again) {
            for (int r = wave; r < nrows; r += NW) {
                const int rr = r + f.rt * ROWS, tok = per_head(a, rr), h = f.kvh * a.g + (rr - tok * a.g);
                float acc[D / 64], mr, lr;
                Sight at{f.s.len - f.s.n + tok, f.s.len - f.s.n + tok, suf ? f.s.from : 0};
                if (pre) {
                    const int one[1] = {f.s.first + tok};
                    int p[1];
                    row_positions<1>(a, f.seq, f.s.from, one, p);
                    at.pos = p[0], at.cap = min(p[0], f.s.len - 1);
                }
                plain_row<D, E8>(a, f.seq, f.kvh, a.q + (int64_t)(f.s.first + tok) * a.ld_q + h * D, at, f.s.us, f.s.ulo, UNIT, u0, u1,
                             lane, acc, mr, lr);
                if (whole) {
                    finish_row<D, MIX>(a, f.s.first + tok, h, lane, acc, mr, lr, !pre, alone);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < D / 64; ++e) part[(size_t)r * D + D / 64 * lane + e] = acc[e];
                if (lane == 0) {
                    part[ROWS * D + r] = mr;
                    part[ROWS * (D + 1) + r] = lr;
                }
            }
            note();
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
        lds_barrier();
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
                const int rr = r + f.rt * ROWS, tok = per_head(a, rr), h = f.kvh * a.g + (rr - tok * a.g);
                finish4<D, MIX>(a, f.s.first + tok, h, d, v, mx, ls, !pre, alone);
            } else {
                *reinterpret_cast<f32x4*>(part + (size_t)r * D + d) = v;
                if (d == 0) {
                    part[ROWS * D + r] = mx;
                    part[ROWS * (D + 1) + r] = ls;
                }
            }
        }
        note();
        lds_barrier();  // the ring and mls are free again
    }
}

// acc, l of n parts rescaled to the largest maximum and added in order, by one
// wave: the maxima and sums 64 parts at a time, a part per lane (top(v) points to
// part v's maximum, sum(v) to its sum), then eight parts' outputs (o(v) points to
// this lane's) on their way at once.
template <int RW, class M, class L, class O>
__device__ __forceinline__ void join_parts(int n, int lane, M top_of, L sum_of, O o, float (&acc)[RW], float& mx, float& l) {
    for (int v0 = 0; v0 < n; v0 += 64) {
        const int c = min(64, n - v0);
        float m = kNoMax, s = 0.0f;
        if (lane < c) {
            m = *top_of(v0 + lane);
            s = *sum_of(v0 + lane);
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

// The cut tiles: a wave per row joins the parts of the tile that begins in part
// blockIdx.x and ends in a later one, in the order of the line. (What the streaming
// workgroups wrote of it is one trip to memory; the scan for it anew took 2 us.)
template <int D, int QT>
__global__ void __launch_bounds__(256) attn_paged_rows_merge_kernel(PagedAttnArgs a) {
    constexpr int ROWS = 16 * QT, RW = D / 64;
    const int lane = threadIdx.x & 63;
    const int r = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
    const int w = blockIdx.x;
    const int* e = a.cuts + kTabInts * w;
    const int last = e[0], first = e[1], rt = e[2], nrows = e[3], kvh = e[4];
    if (last == 0 || r >= nrows) return;
    // Part w holds the tile's begin in its second place, the later ones theirs in the first.
    auto place = [&](int v) { return a.part + (size_t)(2 * (w + v) + (v == 0 ? 1 : 0)) * rows_part(D, QT); };
    float acc[RW] = {}, ls = 0.0f, mx = kNoMax;
    join_parts<RW>(
        last - w + 1, lane, [&](int v) { return place(v) + ROWS * D + r; }, [&](int v) { return place(v) + ROWS * (D + 1) + r; },
        [&](int v) { return place(v) + (size_t)r * D + RW * lane; }, acc, mx, ls);
    const int rr = r + rt * ROWS, tok = per_head(a, rr), h = kvh * a.g + (rr - tok * a.g);
    finish_row<D, false>(a, first + tok, h, lane, acc, mx, ls, 0, true);
}

// MIX: the parts of every (row, head) joined, in the order shared, own: by a wave, or
// (PG = 4: few rows, of many parts) by four, a quarter of each half's places each.
// Records of sequences that are malformed may hold anything: they are not followed out
// of bounds. Few rows: three trips to memory, 7 us; 576 rows of 512 in 45 parts 16 us, 3.7
// TB/s.
template <int D, int QT, int PG>
__global__ void __launch_bounds__(256) attn_paged_join_kernel(PagedAttnArgs a) {
    constexpr int ROWS = 16 * QT, RW = D / 64, TR = 128;
    __shared__ float sums[PG > 1 ? PG : 1][D + 2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = PG > 1 ? wave : 0;
    const int64_t rows = (int64_t)a.b.T * a.heads;
    for (int64_t row = (int64_t)blockIdx.x * (4 / PG) + (PG > 1 ? 0 : wave); row < rows; row += (int64_t)gridDim.x * (4 / PG)) {
        const int t = uniform((int)(row / a.heads)), h = uniform((int)(row % a.heads));
        const int4 recs[2] = {a.recs[row], a.recs[rows + row]};
        const SeqRows sr = find_row(a.b, t, lane);
        if (sr.seq < 0 || sr.first < 0 || (int64_t)sr.first + sr.n > a.b.T || uniform(recs[1].y) == kDone) continue;
        float acc[RW] = {}, ls = 0.0f, mx = kNoMax;
        // The places of both halves as one list (a whole part is one place).
        struct {
            int w, n, r, rows;
            bool tile, whole;
        } x[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            auto& p = x[half];
            p.w = uniform(recs[half].x), p.n = uniform(recs[half].y), p.r = uniform(recs[half].z) & (kTileRec - 1);
            p.tile = uniform(recs[half].z) & kTileRec, p.whole = p.n == kWhole;
            p.rows = p.tile ? TR : ROWS;
            const int most = p.tile ? a.tile_places : a.grid;
            const int64_t last = p.w + (int64_t)(p.n - 1) * (p.tile ? a.kv_heads : 1);
            if (p.whole)
                p.n = 1;
            else if (p.n < 1 || p.w < 0 || p.r >= p.rows || last >= most)
                p.n = 0;
        }
        if (uniform(recs[1].w) <= 0) x[0].n = 0;
        const int n = x[0].n + x[1].n;
        auto from = [&](int half, int v) {
            const auto& p = x[half];
            return p.tile ? a.tile_part + (int64_t)(p.w + v * a.kv_heads) * (TR * (D + 2))
                          : a.part + (size_t)(2 * (p.w + v) + (v == 0 ? 1 : 0)) * rows_part(D, QT);
        };
        auto top_of = [&](int half, int v) {
            const auto& p = x[half];
            return p.whole ? a.kept_ml[half] + 2 * row : from(half, v) + p.rows * D + p.r;
        };
        auto out_of = [&](int half, int v) {
            const auto& p = x[half];
            return (p.whole ? a.kept[half] + row * D : from(half, v) + (size_t)p.r * D) + RW * lane;
        };
        const int lo = (int)((int64_t)n * part / PG), hi = (int)((int64_t)n * (part + 1) / PG), n0 = x[0].n;
        join_parts<RW>(
            hi - lo, lane, [&](int v) { return lo + v < n0 ? top_of(0, lo + v) : top_of(1, lo + v - n0); },
            [&](int v) {
                return lo + v < n0 ? top_of(0, lo + v) + (x[0].whole ? 1 : x[0].rows)
                                   : top_of(1, lo + v - n0) + (x[1].whole ? 1 : x[1].rows);
            },
            [&](int v) { return lo + v < n0 ? out_of(0, lo + v) : out_of(1, lo + v - n0); }, acc, mx, ls);
        if constexpr (PG > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < RW; ++e) sums[wave][RW * lane + e] = acc[e];
            if (lane == 0) {
                sums[wave][D] = mx;
                sums[wave][D + 1] = ls;
            }
            __syncthreads();
            if (wave) continue;
#pragma unroll
            for (int e = 0; e < RW; ++e) acc[e] = 0.0f;
            ls = 0.0f, mx = kNoMax;
            join_parts<RW>(
                PG, lane, [&](int v) { return &sums[v][D]; }, [&](int v) { return &sums[v][D + 1]; },
                [&](int v) { return &sums[v][RW * lane]; }, acc, mx, ls);
        }
        finish_row<D, false>(a, t, h, lane, acc, mx, ls, 0, true);
    }
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
//
// 8-bit pages: the widening is 2 vector instructions a matrix one more, 4096 tokens of 16
// heads of 512 on one behind 2048 706 us (780 TFLOP/s): matrix cores busy 30 % of the
// time, vector ALUs 46 %, the waves waiting 36 %. Groups: drafts of 16 sequences (0 to 5
// tokens) over 20032 shared positions, 5 tiles in 45 parts each, 65 us, and 16 for the
// join of 60 MB of parts.
constexpr int tile_ds(int D) { return D == 512 ? 2 : 1; }      // waves that share 32 rows
constexpr int tile_waves(int D) { return D == 512 ? 8 : 4; }
constexpr int tile_rows(int D) { return 32 * tile_waves(D) / tile_ds(D); }
constexpr int tile_bn(int D) { return D <= 128 ? 64 : 32; }
constexpr int tile_bytes(int D) { return tile_bn(D) * 2 * D; }  // of K, of V
constexpr int tile_xch(int D) { return D == 512 ? tile_waves(D) * 4096 : 0; }
// 8-bit pages: whether LDS holds codes, widened at each read, and how many units of
// them; else they are widened on their way there. Codes halve what LDS delivers, which
// bounds D >= 256 (with the products), for two vector instructions per matrix one;
// D <= 128 is bound by the vector ALUs already.
constexpr bool tile_codes(int D, bool E8) { return E8 && D >= 256; }
constexpr int tile_stages(int D) { return D == 512 ? 3 : 4; }
constexpr int kPowers = 4;  // units whose powers are kept (V's are read when the next K's buffer is filled again)
constexpr int tile_lds(int D, bool E8) {
    return (tile_codes(D, E8) ? tile_stages(D) * 2 * tile_bn(D) * D + kPowers * 2 * tile_bn(D) : 4 * tile_bytes(D)) + tile_xch(D);
}
// The swizzle of V's codes there: the 8 rows (0 .. 3, 8 .. 11) of two pieces that half
// the lanes read at once on different banks.
__device__ __forceinline__ constexpr int vt8_swz(int row) { return ((row & 3) | ((row >> 1) & 4)) << 1; }

typedef float f32x16 __attribute__((__vector_size__(16 * sizeof(float))));

// Tiles of the sequences of more rows than row_limit, up to and with each
// lane's, in one step of 64 sequences.
struct TileScan {
    SeqIn s;
    int tiles, incl, sum;
};
template <int TR, bool MIX>
__device__ __forceinline__ TileScan tile_scan(const PagedAttnArgs& a, int b0, int lane, const SeqIn* groups = nullptr) {
    TileScan t{};
    t.s = seq_in<MIX>(a, b0, lane, groups);
    const int64_t rows = t.s.here ? (int64_t)t.s.n * a.g : 0;
    if (rows > a.row_limit) t.tiles = (int)((rows + TR - 1) / TR);
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
    int pos_lo, pos_hi;  // of its first and last row (of a group: the lowest and the highest there can be)
    int us, ulo, nu;
};
template <int TR, int BN, bool MIX>
__device__ __forceinline__ TileSpan tile_span(const PagedAttnArgs& a, int n, int len, bool ok, int from, int low, bool pre, int rt) {
    TileSpan s;
    const int r0 = rt * TR;  // (rows, of one kv head too, stay below 2^30)
    s.rows = min(TR, n * a.g - r0);
    s.pos_lo = pre ? low : len - n + r0 / a.g;
    s.pos_hi = pre ? len - 1 : len - n + (r0 + s.rows - 1) / a.g;
    const int lo = a.window > 0 ? max(0, s.pos_lo + 1 - a.window) : 0;
    const Begin at = begin_units<BN>(a, lo, MIX && !pre, from);
    s.us = at.us, s.ulo = at.ulo;
    s.nu = ok ? s.us + max(s.pos_hi / BN + 1 - s.ulo, !MIX ? INT_MIN : 0) : 0;
    return s;
}

// Items (tiles times kv heads, times their parts) and where each is found: heaviest
// (last) tiles first, kv heads side by side, so that the workgroups an XCD gets
// in turn share theirs where there are eight.
// Step b0 / 64: the first two are read once for all that needs them (a step behind
// groups is 3 us).
struct TileSteps {
    TileScan s0, s1;
};
template <int TR, bool MIX>
__device__ __forceinline__ TileScan tile_step(const PagedAttnArgs& a, const TileSteps& s, int b0, int lane) {
    if (b0 == 0) return s.s0;
    if (MIX && b0 == 64) return s.s1;
    return tile_scan<TR, MIX>(a, b0, lane, MIX ? &s.s0.s : nullptr);
}

template <int TR, bool MIX>
__device__ __forceinline__ int tile_count(const PagedAttnArgs& a, const TileSteps& steps, int lane) {  // per kv head
    // (no more than there can be: sequences that overlap must not carry the sum away)
    int all = min(steps.s0.sum, a.max_tiles);
    for (int b0 = 64; b0 < seq_count<MIX>(a); b0 += 64) all = min(all + tile_step<TR, MIX>(a, steps, b0, lane).sum, a.max_tiles);
    return all;
}

// Where tile gt is.
template <int TR, int BN, bool MIX>
struct TileAt {
    int seq, rt, first, n, len, from;
    bool pre;
    TileSpan sp;
    __device__ __forceinline__ TileAt(const PagedAttnArgs& a, const TileSteps& steps, int gt, int lane) {
        int base = 0, b0 = 0;
        TileScan sc = steps.s0;
        while (gt >= base + sc.sum) {
            base += sc.sum;
            b0 += 64;
            sc = tile_step<TR, MIX>(a, steps, b0, lane);
        }
        const int l = __builtin_ctzll(__ballot(base + sc.incl > gt));
        seq = MIX ? __builtin_amdgcn_readlane(sc.s.seq, l) : b0 + l;
        pre = MIX && b0 < group_steps<MIX>(a);
        first = __builtin_amdgcn_readlane(sc.s.first, l);
        n = __builtin_amdgcn_readlane(sc.s.n, l);
        len = __builtin_amdgcn_readlane(sc.s.len, l);
        from = !MIX ? 0 : __builtin_amdgcn_readlane(sc.s.from, l);
        rt = gt - base - __builtin_amdgcn_readlane(sc.incl - sc.tiles, l);
        sp = tile_span<TR, BN, MIX>(a, n, len, __builtin_amdgcn_readlane((int)sc.s.ok, l) != 0, from,
                                    MIX ? __builtin_amdgcn_readlane(sc.s.lo, l) : 0, pre, rt);
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
// (entries: that of part 0, parts, first row of the sequence, tile, rows, kv head)

__device__ __forceinline__ int sum64(int v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return uniform(v);
}

// Units of every tile, into LDS, by all waves.
template <int TR, int BN, int NW, bool MIX>
__device__ __forceinline__ void tile_units(const PagedAttnArgs& a, const TileSteps& steps, int tiles, int lane, int wave, int* nu) {
    int base = 0, turn = 0;
    for (int b0 = 0; b0 < seq_count<MIX>(a) && base < tiles; b0 += 64) {
        const TileScan sc = tile_step<TR, MIX>(a, steps, b0, lane);
        for (int x0 = 0; x0 < sc.sum && base + x0 < tiles; x0 += 64, ++turn) {
            if (turn % NW != wave) continue;
            const int x = x0 + lane;
            int l = 0;  // the sequence: the first lane whose tiles end behind x
#pragma unroll
            for (int o = 32; o; o >>= 1)
                if (__shfl(sc.incl, l + o - 1) <= x) l += o;
            l = min(l, 63);
            const int before = __shfl(sc.incl - sc.tiles, l), n = __shfl(sc.s.n, l), len = __shfl(sc.s.len, l);
            const bool ok = __shfl((int)sc.s.ok, l) != 0;
            const int from = MIX ? __shfl(sc.s.from, l) : 0, low = MIX ? __shfl(sc.s.lo, l) : 0;
            if (x < sc.sum && base + x < tiles)
                nu[base + x] = tile_span<TR, BN, MIX>(a, n, len, ok, from, low, MIX && b0 < group_steps<MIX>(a), x - before).nu;
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
template <bool MIX>
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
        if (parts <= (MIX ? slots : 2 * slots)) return cap;
        // A group's tile's parts are as long as can be: no second turn, but the smallest cap of
        // 64, a lane each, whose parts all run at once (drafts of 16 sequences over 20032 shared
        // positions and up to 3000 of their own, heads of 512: 150 -> 106 us; this search for
        // every call costs 64 tokens over 4 prompts of 4000 3 us of 60).
        if constexpr (MIX) {
            const int lo = max(least, (total + slots - 1) / slots), mine = lo + lane * (1 + lo / 48);
            const float inv = 1.0f / (float)mine;
            int n = 0;
#pragma unroll 4
            for (int t = 0; t < tiles; ++t)  // (one off at millions of units only)
                n += (int)(((float)max(1, nu[t]) + (float)mine - 0.5f) * inv);
            const uint64_t fit = __ballot(n <= slots);
            if (fit) {
                const int best = __builtin_amdgcn_readlane(mine, __builtin_ctzll(fit));
                parts = tile_parts_sum(nu, tiles, lane, best);
                if (parts <= slots) return best;
            }
        }
    }
    int cap = max(least, (total + slots - tiles / 2 - 1) / max(1, slots - tiles / 2));
    for (int turn = 0; turn < 2; ++turn, cap += cap / 2) {
        parts = tile_parts_sum(nu, tiles, lane, cap);
        if (parts <= slots) return cap;
    }
    parts = tiles;
    return INT_MAX / 2;
}

template <int D, bool E8, bool MIX>
__device__ __forceinline__ void tile_item(const PagedAttnArgs& a, const TileSteps& steps, int gt, int kvh, int split, int nsplit,
                                          int entry, int* tab, unsigned char* smem) {
    constexpr int DS = tile_ds(D), NW = tile_waves(D), TR = tile_rows(D), BN = tile_bn(D);
    constexpr int DW = D / DS;            // this wave's columns of the output (and of its scores' products)
    constexpr int TB = tile_bytes(D), NC = D / 8, RPL = 512 / D;
    constexpr int LR = BN / NW;           // positions a wave loads: within one block of 16
    constexpr int NL = LR / RPL;          // its loads of K (of V)
    constexpr int NB = BN / 16;
    constexpr int KR = 4, VR = 4;         // operands of K, of V on their way from LDS
    constexpr bool LC = tile_codes(D, E8);
    constexpr int TC = BN * D, NST = tile_stages(D);  // bytes of a unit's K as codes; units in LDS
    unsigned char* kbuf = smem;
    unsigned char* vbuf = smem + (LC ? NST * TC : 2 * TB);
    [[maybe_unused]] unsigned char* pow = smem + 2 * NST * TC;  // pairs of powers, of kPowers units
    float* xch = reinterpret_cast<float*>(smem + tile_lds(D, E8) - tile_xch(D));
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave / DS, dh = wave % DS;
    const int col = lane & 31, h = lane >> 5;

    const TileAt<TR, BN, MIX> at_item(a, steps, gt, lane);
    const int seq = at_item.seq, rt = at_item.rt;
    const int first = at_item.first, n = at_item.n, len = at_item.len, from = at_item.from;
    const bool pre = MIX && at_item.pre, suf = MIX && !at_item.pre, alone = suf && from == 0;
    const TileSpan sp = at_item.sp;
    const int u0 = uniform((int)((int64_t)sp.nu * split / nsplit));
    const int u1 = uniform((int)((int64_t)sp.nu * (split + 1) / nsplit));
    if constexpr (MIX) {
        for (int r = split == 0 ? tid : sp.rows; r < sp.rows; r += 64 * NW) {
            const int rr = rt * TR + r;
            const int64_t row = (int64_t)(first + rr / a.g) * a.heads + kvh * a.g + rr % a.g;
            a.recs[(pre ? 0 : (int64_t)a.b.T * a.heads) + row] =
                int4{entry, nsplit > 1 ? nsplit : (alone ? kDone : kWhole), r | kTileRec, from};
        }
    } else if (tab && split == 0 && tid == 0) {
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
            const bool in = v0 + lane < u1 && p + 16 * k < len && (!suf || p + 16 * k >= from);  // (else any entry may be there)
            int e = in ? table[(p + 16 * k) >> a.b.shift] : -1;
            if ((unsigned)e >= (unsigned)a.b.pages) e = -1;
            gone[k] = __ballot(in && e < 0);
            pages = k == wave * LR / 16 ? e : pages;
        }
    };
    uint32_t holes = 0;  // NB bits by unit modulo 4
    const uint32_t kb_lds = __builtin_amdgcn_readfirstlane(lds_addr(kbuf)) + wave * LR * (LC ? D : 2 * D);
    const uint32_t vb_lds = __builtin_amdgcn_readfirstlane(lds_addr(vbuf)) + wave * LR * (LC ? D : 2 * D);
    // The wave's rows start at a multiple of 4, not of 16: their bits of the
    // swizzles are part of the lane's offset.
    const uint32_t dma_k = (lane / NC) * (2 * D) + ((lane % NC) ^ k_swz<D>(wave * LR + lane / NC)) * 16;
    const uint32_t dma_v = (lane / NC) * (2 * D) + ((lane % NC) ^ v_swz<D>(wave * LR + lane / NC)) * 16;
    // Starts unit u's K (then its V) on the way to LDS; K before V, units in order.
    [[maybe_unused]] auto issue = [&](int u, bool v) __attribute__((always_inline)) {
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
        const uint16_t* src = v ? static_cast<const uint16_t*>(a.vpages) + max(page, 0) * a.v_stride
                                : static_cast<const uint16_t*>(a.kpages) + max(page, 0) * a.k_stride;
        const __amdgpu_buffer_rsrc_t r = wave_rsrc(src + off, bytes);
        const uint32_t dst = (v ? vb_lds : kb_lds) + (u & 1) * TB, at = here(v ? dma_v : dma_k);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t x = v ? (uint32_t)v_swz<D>(RPL * i) : (uint32_t)k_swz<D>(RPL * i);
            load_lds16(r, at ^ (x * 16), 1024 * i, dst + 1024 * i);
        }
    };

    // Codes to LDS as they are, with K the slots' powers.
    constexpr int NCC = D / 16, RPC = 1024 / D;  // pieces of a row; rows of one load
    constexpr int NLC = LC ? LR / RPC : 1;       // a wave's loads of K (of V)
    const uint32_t dma_kc = (lane / NCC) * D + ((lane % NCC) ^ k8_swz<D>(wave * LR + lane / NCC)) * 16;
    const uint32_t dma_vc = (lane / NCC) * D + ((lane % NCC) ^ vt8_swz(wave * LR + lane / NCC)) * 16;
    auto slot_of = [&](int u) __attribute__((always_inline)) { return (uint32_t)(u - u0) % NST; };
    [[maybe_unused]] auto issue_codes = [&](int u, bool v) __attribute__((always_inline)) {
        if (u - pages0 >= 64) load_pages(u);
        const int page = __builtin_amdgcn_readlane(pages, u - pages0), p = unit_pos(u) + wave * LR;
        const int have = page < 0 ? 0 : max(0, min(LR, len - p));
        const int64_t at0 = ((int64_t)kvh << a.b.shift) + (p & ((1 << a.b.shift) - 1));
        if (!v) {
            uint32_t now = 0;
#pragma unroll
            for (int k = 0; k < NB; ++k) now |= (uint32_t)(gone[k] >> (u - pages0) & 1) << k;
            const int bit = NB * (u & 3);
            holes = (holes & ~(((1u << NB) - 1) << bit)) | (now << bit);
        }
        const uint8_t* src = v ? static_cast<const uint8_t*>(a.vpages) + max(page, 0) * a.v_stride
                               : static_cast<const uint8_t*>(a.kpages) + max(page, 0) * a.k_stride;
        const __amdgpu_buffer_rsrc_t r = wave_rsrc(src + at0 * D, have * D);
        const uint32_t slot = slot_of(u), dst = (v ? vb_lds : kb_lds) + slot * TC, at = here(v ? dma_vc : dma_kc);
#pragma unroll
        for (int i = 0; i < NLC; ++i) {
            const uint32_t x = v ? (uint32_t)vt8_swz(RPC * i) : (uint32_t)k8_swz<D>(RPC * i);
            load_lds16(r, at ^ (x * 16), 1024 * i, dst + 1024 * i);
        }
        if (!v)
            load_lds4<LR / 2>(wave_rsrc(a.scales + max(page, 0) * a.s_stride + 2 * at0, have > 0 ? 2 * LR : 0), lane * 4,
                              __builtin_amdgcn_readfirstlane(lds_addr(pow)) + (uint32_t)(u - u0) % kPowers * (2 * BN) + wave * (2 * LR));
    };

    // The last unit, u1 - 1, may end behind len: its powers there.
    [[maybe_unused]] const int tail = u1 > u0 ? len - unit_pos(u1 - 1) : BN;
    [[maybe_unused]] auto powers_end = [&](int u) __attribute__((always_inline)) {
        if (u + 1 == u1 && tail < BN) clear_powers<BN>(pow + (uint32_t)(u - u0) % kPowers * (2 * BN), tail);
    };

    // Or a wave's share of a unit goes through registers, where codes become bf16
    // times their power, so that what LDS holds and the products are the same.
    constexpr int NP = E8 ? LR * D / 1024 : 1;  // pieces of 16 codes of a lane, of K (of V)
    struct Codes {
        u32x4 c[NP];
        int e[NP];
    };
    [[maybe_unused]] auto fetch = [&](int u, bool v, Codes& x) __attribute__((always_inline)) {
        if (u - pages0 >= 64) load_pages(u);
        const int page = __builtin_amdgcn_readlane(pages, u - pages0), p = unit_pos(u) + wave * LR;
        const uint32_t have = page < 0 ? 0u : (uint32_t)max(0, min(LR, len - p));
        const int64_t slot = ((int64_t)kvh << a.b.shift) + (p & ((1 << a.b.shift) - 1));
        if (!v) {
            uint32_t now = 0;
#pragma unroll
            for (int k = 0; k < NB; ++k) now |= (uint32_t)(gone[k] >> (u - pages0) & 1) << k;
            const int at = NB * (u & 3);
            holes = (holes & ~(((1u << NB) - 1) << at)) | (now << at);
        }
        const uint8_t* src = v ? static_cast<const uint8_t*>(a.vpages) + max(page, 0) * a.v_stride
                               : static_cast<const uint8_t*>(a.kpages) + max(page, 0) * a.k_stride;
        const __amdgpu_buffer_rsrc_t r = wave_rsrc(src + slot * D, have * D);
        const __amdgpu_buffer_rsrc_t rs = wave_rsrc(a.scales + max(page, 0) * a.s_stride + 2 * slot, have * 2);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const uint32_t at = 64 * i + lane;
            x.c[i] = __builtin_amdgcn_raw_buffer_load_b128(r, 16 * at, 0, 0);
            x.e[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, at / (D / 16) * 2 + v, 0, 0);
        }
    };
    [[maybe_unused]] auto commit = [&](int u, bool v, const Codes& x) __attribute__((always_inline)) {
        unsigned char* buf = (v ? vbuf : kbuf) + (u & 1) * TB;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int at = 64 * i + lane, row = wave * LR + at / (D / 16), pc = 2 * (at % (D / 16));
            const int z = v ? v_swz<D>(row) : k_swz<D>(row);
            const float power = power_of_byte<0>(x.e[i]);
            const uint32_t c0 = x.c[i][0], c1 = x.c[i][1], c2 = x.c[i][2], c3 = x.c[i][3];
            *reinterpret_cast<bf16x8*>(buf + row * (2 * D) + (pc ^ z) * 16) = widen8(c0, c1, power);
            *reinterpret_cast<bf16x8*>(buf + row * (2 * D) + ((pc + 1) ^ z) * 16) = widen8(c2, c3, power);
        }
    };

    // The first units' way to LDS. (What is fetched is one unit ahead of what is in LDS, with
    // DS = 2 one phase.) It begins ahead of q's, a trip to memory less; but not for bf16 tiles
    // of D <= 256 without groups, where q's would return behind them and two workgroups
    // share a CU (three chunks of 1000 tokens in a 1024 window, 16 heads of 256 on 8,
    // 71.3 us against 69.9, of 128 45.2 against 45.0; 1024 tokens, 256, 41.7 against 40.7).
    [[maybe_unused]] Codes kx, vx;
    auto start = [&]() __attribute__((always_inline)) {
        if (u1 <= u0) return;
        load_pages(u0);
        if constexpr (LC) {
            // (DS = 1: three units ahead, of four; DS = 2: four phases, of three units)
            constexpr int ahead = DS == 1 ? 3 : 2;
#pragma unroll
            for (int i = 0; i < ahead; ++i)
                if (u0 + i < u1) {
                    issue_codes(u0 + i, false);
                    issue_codes(u0 + i, true);
                }
        } else if constexpr (E8) {
            fetch(u0, false, kx);
            fetch(u0, true, vx);
        } else {
            issue(u0, false);
            issue(u0, true);
        }
    };
    constexpr bool kAhead = E8 || MIX || DS == 2;
    if constexpr (kAhead) start();

    // This lane's row: column col of the wave's 32.
    const int r0 = rt * TR + 32 * rg;
    const int nrows = max(0, min(32, n * a.g - r0));
    const int row = r0 + min(col, max(nrows - 1, 0));
    const int tok = min(row / a.g, n - 1), head = kvh * a.g + row % a.g;
    bf16x8 q[DW / 16];
    {
        // (a lane's 16 bytes of codes are two operands: 16 columns of each 32)
        const uint16_t* qr = a.q + (int64_t)(first + tok) * a.ld_q + head * D + dh * DW + (LC ? 16 : 8) * h;
#pragma unroll
        for (int i = 0; i < DW / 16; ++i)
            q[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(qr + (LC ? 32 * (i / 2) + 8 * (i % 2) : 16 * i)));
    }
    int pos = len - n + tok, cap = pos;
    int wpos_lo = len - n + r0 / a.g;                        // lowest position up to which a row of the wave sees,
    int wpos_hi = len - n + (r0 + max(nrows, 1) - 1) / a.g;  // highest,
    int wpos_top = wpos_hi;                                  // and highest position of one
    if (pre) {
        const int one[1] = {first + tok};
        int p[1];
        row_positions<1>(a, seq, from, one, p);
        pos = p[0], cap = min(pos, len - 1);
        wpos_lo = min64(cap), wpos_hi = max64(cap), wpos_top = max64(pos);
    }
    const float c = fmaxf(a.scale * kLog2e, kMinScale);
    // Waited for here: the compiler would else wait at their first use, in
    // the loop, each time, for whatever is on its way to LDS by then.
#pragma unroll
    for (int i = 0; i < DW / 16; ++i) asm volatile("" : "+v"(q[i]));
    f32x16 o[DW / 32];
#pragma unroll
    for (int d = 0; d < DW / 32; ++d) o[d] = f32x16{};
    float m = kNoMax, l = 0.0f;

    const int vrow = LC ? 4 * h + ((lane >> 1) & 3) + 8 * ((lane >> 3) & 1) : 4 * h + ((lane & 15) >> 2);
    const uint32_t rd_k = LC ? col * D + (h ^ k8_swz<D>(col)) * 16 : col * (2 * D) + (h ^ k_swz<D>(col)) * 16;
    const uint32_t rd_v = LC ? vrow * D + (((lane >> 4) & 1) ^ vt8_swz(vrow)) * 16 + (lane & 1) * 8
                             : vrow * (2 * D) + ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ v_swz<D>(vrow)) * 16 + (lane & 1) * 8;

    // Rows that see nothing of 32 positions at p0 (or are none) are done with them.
    auto skip = [&](int p0) { return nrows == 0 || p0 > wpos_hi; };
    // K q of the 32 positions whose rows begin at ks, over this wave's columns.
    auto scores = [&](const unsigned char* ks, [[maybe_unused]] const unsigned char* pw) __attribute__((always_inline)) {
        f32x16 s{};
        const uint32_t at = here(rd_k);
        if constexpr (LC) {
            constexpr int NK = DW / 32, R = 3;  // pieces of two operands; on their way
            const float power = power_of_byte<0>(*reinterpret_cast<const uint16_t*>(pw + 2 * col));
            auto read_k = [&](int i) __attribute__((always_inline)) {
                return *reinterpret_cast<const u32x4*>(ks + (at ^ piece8<D>(2 * i)) + dh * DW);
            };
            u32x4 k[R];
#pragma unroll
            for (int i = 0; i < R; ++i) k[i] = read_k(i);
            if constexpr (DS == 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                const uint32_t c0 = k[i % R][0], c1 = k[i % R][1], c2 = k[i % R][2], c3 = k[i % R][3];
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen8(c0, c1, power), q[2 * i], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen8(c2, c3, power), q[2 * i + 1], s, 0, 0, 0);
                if (i + R < NK) k[i % R] = read_k(i + R);
            }
            if constexpr (DS == 1) __builtin_amdgcn_s_setprio(0);
            return s;
        }
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
    auto absorb = [&](const f32x16& sv, int p0, const unsigned char* vs, [[maybe_unused]] const unsigned char* pwr, uint32_t hole)
                      __attribute__((always_inline)) {
        hole &= 3;  // of its two blocks of 16
        float s[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = sv[i];
        const bool masked = hole || p0 + 31 > wpos_lo || (suf && p0 < from) ||
                            (a.window > 0 && p0 <= wpos_top - a.window && p0 + 31 >= a.sinks);
        if (masked) {
            // Relative to p0 + 4 h, so that positions are constants.
            const int at = cap - p0 - 4 * h, lo = a.window > 0 ? pos - p0 - 4 * h - a.window : INT_MIN, sk = a.sinks - p0 - 4 * h;
            [[maybe_unused]] const int begin = (suf ? from : 0) - p0 - 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int p = 8 * (i / 4) + i % 4, hi = hole >> (i / 8) & 1 ? -1 : at;
                bool seen = (p <= hi) & ((p > lo) | (p < sk));
                if constexpr (MIX) seen &= p >= begin;
                s[i] = seen ? s[i] : -__builtin_inff();
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
        if constexpr (LC) {  // times V's powers
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const i32x2 pairs = *reinterpret_cast<const i32x2*>(pwr + 16 * g + 8 * h);
                const uint32_t a0 = pairs[0], a1 = pairs[1];
                w[4 * g] *= power_of_byte<1>(a0);
                w[4 * g + 1] *= power_of_byte<3>(a0);
                w[4 * g + 2] *= power_of_byte<1>(a1);
                w[4 * g + 3] *= power_of_byte<3>(a1);
            }
        }
        bf16x8 pw[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) pw[i >> 3][i & 7] = (__bf16)w[i];
        // Columns 32 d .. of this wave, positions 16 k + 8 e + 4 h .. + 3.
        const uint32_t at = here(rd_v);
        auto read_v = [&](int d, int k) __attribute__((always_inline)) {
            if constexpr (LC) {
                return read_tr8(vs + (at ^ piece8<D>(2 * d)) + dh * DW + k * 16 * D);
            } else {
            const unsigned char* v = vs + (at ^ piece<D>(4 * d)) + piece_far<D>((dh * DW + 32 * d) / 8 & ~15) + k * 32 * D;
            const s16x4 lo = read_tr(v), hi = read_tr(v + 16 * D);
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            }
        };
        auto operand = [](auto v) __attribute__((always_inline)) {
            if constexpr (LC)
                return widen8(v[0], v[1], 1.0f);
            else
                return v;
        };
        // Operand j: two blocks of columns in turn, then their second 16 positions.
        constexpr int NV = DW / 16;
        auto blk = [](int j) { return (j & ~3) / 2 + (j & 1); };
        std::conditional_t<LC, i32x2, bf16x8> v[VR];
#pragma unroll
        for (int j = 0; j < VR; ++j) v[j] = read_v(blk(j), j >> 1 & 1);
        if constexpr (DS == 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            o[blk(j)] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(v[j % VR]), pw[j >> 1 & 1], o[blk(j)], 0, 0, 0);
            if (j + VR < NV) v[j % VR] = read_v(blk(j + VR), (j + VR) >> 1 & 1);
        }
        if constexpr (DS == 1) __builtin_amdgcn_s_setprio(0);
    };

    if constexpr (!kAhead) start();
    if constexpr (E8 && !LC)
        if (u1 > u0) {
            commit(u0, false, kx);
            if constexpr (DS == 1) {
                commit(u0, true, vx);
                if (u0 + 1 < u1) {
                    fetch(u0 + 1, false, kx);
                    fetch(u0 + 1, true, vx);
                }
            }
        }
    if constexpr (DS == 1) {
#pragma unroll 1
        for (int u = u0; u < u1; ++u) {
            if constexpr (LC) {
                if (u + 2 < u1)
                    wait_vm<2 * (2 * NLC + 1)>();
                else
                    wait_vm<0>();
            } else if constexpr (!E8) {
                wait_vm<0>();
            }
            __syncthreads();
            if constexpr (LC) {
                if (u + 3 < u1) {
                    issue_codes(u + 3, false);
                    issue_codes(u + 3, true);
                }
                powers_end(u);  // (each wave for itself)
            } else if (u + 1 < u1) {
                if constexpr (E8) {
                    commit(u + 1, false, kx);
                    commit(u + 1, true, vx);
                    if (u + 2 < u1) {
                        fetch(u + 2, false, kx);
                        fetch(u + 2, true, vx);
                    }
                } else {
                    issue(u + 1, false);
                    issue(u + 1, true);
                }
            }
            const int pt = unit_pos(u);
            const uint32_t slot = LC ? slot_of(u) : u & 1;
            const unsigned char* kt = kbuf + slot * (LC ? TC : TB);
            const unsigned char* vt = vbuf + slot * (LC ? TC : TB);
            const unsigned char* pw = pow + (uint32_t)(u - u0) % kPowers * (2 * BN);
#pragma unroll 1
            for (int sub = 0; sub < BN / 32 && !skip(pt + 32 * sub); ++sub)
                absorb(scores(kt + sub * 64 * D, pw), pt + 32 * sub, vt + sub * 64 * D, pw, holes >> (NB * (u & 3) + 2 * sub));
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
        // (codes become LDS's one phase ahead: phase + 1's buffer has had its last reader
        // two phases ago)
        auto begin = [&](int phase) __attribute__((always_inline)) {
            if constexpr (LC) {
                // Phases phase + 1 .. + 3 may still be on their way: two of K, one of V, or
                // the reverse. A buffer's last reader was two phases ago.
                if (phase + 3 < 2 * nu) {
                    if (phase & 1)
                        wait_vm<3 * NLC + 2>();
                    else
                        wait_vm<3 * NLC + 1>();
                } else {
                    wait_vm<0>();
                }
                __syncthreads();
                if (phase + 4 < 2 * nu) issue_codes(u0 + ((phase + 4) >> 1), phase & 1);
                return;
            }
            if constexpr (E8) {
                __syncthreads();
                if (phase + 1 < 2 * nu) commit(u0 + ((phase + 1) >> 1), (phase + 1) & 1, vx);
                if (phase + 2 < 2 * nu) fetch(u0 + ((phase + 2) >> 1), phase & 1, vx);
                return;
            }
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
            if constexpr (LC)
                if (wave == 0) powers_end(u);  // (for all: V's are read from the next phase on)
            if (!skip(p0)) {
                const uint32_t slot = LC ? slot_of(u) : u & 1;
                s = scores(kbuf + slot * (LC ? TC : TB), pow + (uint32_t)(u - u0) % kPowers * (2 * BN));
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
                const uint32_t slot = LC ? slot_of(u) : u & 1;
                absorb(s, p0, vbuf + slot * (LC ? TC : TB), pow + (uint32_t)(u - u0) % kPowers * (2 * BN), holes >> (NB * (u & 3)));
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
            const Sight at{__builtin_amdgcn_readlane(pos, r), __builtin_amdgcn_readlane(cap, r), suf ? from : 0};
            plain_row<D, E8>(a, seq, kvh, a.q + (int64_t)(first + tk) * a.ld_q + hd * D, at, sp.us, sp.ulo, BN, u0, u1, lane, acc,
                         mr, lr);
            if (nsplit == 1) {
                finish_row<D, MIX>(a, first + tk, hd, lane, acc, mr, lr, !pre, alone);
                continue;
            }
            float* pr = part + (32 * rg + r) * D + D / 64 * lane;
#pragma unroll
            for (int e = 0; e < D / 64; ++e) pr[e] = acc[e];
            if (lane == 0) {
                part[TR * D + 32 * rg + r] = mr;
                part[TR * (D + 1) + 32 * rg + r] = lr;
            }
        }
        return;
    }
    l += __shfl_xor(l, 32);
    if (col >= nrows) return;
    if (nsplit == 1) {
#pragma unroll
        for (int d = 0; d < DW / 32; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                finish4<D, MIX>(a, first + tok, head, dh * DW + 4 * h + 32 * d + 8 * k,
                                f32x4{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]}, m, l, !pre, alone);
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

template <int D, bool E8, bool MIX>
__global__ void __launch_bounds__((64 * tile_waves(D)), 2) attn_paged_tile_kernel(PagedAttnArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int TR = tile_rows(D), BN = tile_bn(D);
    static_assert(tile_lds(D, E8) >= 4 * kSplitTiles, "the tiles' units");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    TileSteps steps;
    steps.s0 = tile_scan<TR, MIX>(a, 0, lane);
    if (MIX && seq_count<MIX>(a) > 64) steps.s1 = tile_scan<TR, MIX>(a, 64, lane, &steps.s0.s);
    const int tiles = tile_count<TR, MIX>(a, steps, lane), items = tiles * a.kv_heads;
    const bool split = items <= a.max_items;
    if (a.tab && blockIdx.x == 0 && tid == 0) a.tab[0] = split ? items : 0;
    if (items == 0) return;  // (the streaming kernel's all; there may be no slots to plan for)
    int gt, kvh, part = 0, parts = 1, entry = 0;
    if (split) {
        int* nu = reinterpret_cast<int*>(smem);
        tile_units<TR, BN, tile_waves(D), MIX>(a, steps, tiles, lane, wave, nu);
        int all;
        const int cap = tile_cap<MIX>(a, nu, tiles, lane, all);
        // (MIX: groups' parts before sequences'; else a prompt's last tiles before its first)
        const int e = MIX ? (int)blockIdx.x : all * a.kv_heads - 1 - (int)blockIdx.x;
        if (e < 0 || e >= all * a.kv_heads) return;
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
    tile_item<D, E8, MIX>(a, steps, uniform(gt), uniform(kvh), uniform(part), uniform(parts), uniform(entry),
                          split ? a.tab : nullptr, smem);
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
            const int rr = rt * TR + r0 + r, tok = per_head(a, rr), head = kvh * a.g + rr % a.g;
            store4(a.out + (int64_t)(first + tok) * a.ld_out + head * D + 4 * c, acc, inv[r]);
        }
        __syncthreads();
    }
}

// How a call's work is spread.
struct AttnPlan {
    int qt;              // row tiles of 16 in the streaming kernel (0: not launched)
    int64_t row_limit;   // sequences of at most this many rows are its, the others the tile kernel's
    int grid;            // its workgroups
    int64_t grid_tiles;  // tiles times kv heads of the tile kernel at most (0: not launched),
    int64_t tiles;       // and at most as far as max_q tells
    int slots;           // parts of tiles; 0: none is split
    uint64_t cuts_bytes, rows_bytes, tab_bytes, part_bytes;
};

__attribute__((unused)) AttnPlan attn_plan(int heads, int kv_heads, int D, int B, int T, int max_q, bool e8) {
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
        p.grid = device_cus() * (rows_two(D, p.qt, e8) ? 2 : 1);
        p.cuts_bytes = (uint64_t)p.grid * kTabInts * sizeof(int);
        p.rows_bytes = p.cuts_bytes + (uint64_t)p.grid * 2 * 16 * p.qt * (D + 2) * sizeof(float);
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

// How the work of groups and sequences together (MIX) is spread: groups of few rows and
// the sequences' own rows are streamed, more rows are tiles, which read K and V once for
// 128 rows. (A streaming tile of more than 32 rows is bound by its products: 64 sequences
// of three prompts, 88 rows of a group and kv head, 95 us streamed, 49 + 20 with tiles.)
__attribute__((unused)) AttnPlan mix_plan(int heads, int kv_heads, int D, int B, int T, int max_q, int groups, bool e8) {
    AttnPlan p{};
    const int64_t g = heads / kv_heads, all = T * g;
    max_q = std::min(max_q, T);
    const int qt_max = D <= 128 ? 4 : (D == 256 ? 2 : 1);
    const int64_t rows = (max_q > 0 ? max_q : ((int64_t)T + B - 1) / B) * g;  // of a sequence, as far as is known
    const int64_t group_rows = ((int64_t)T + groups - 1) / groups * g;
    const int64_t slots = (int64_t)device_cus() * (D == 512 ? 1 : 2), tr = 128;
    auto tiles_of = [&](int64_t n, int64_t row_limit) { return (all / tr + std::min(n, all / (row_limit + 1) + 1)) * kv_heads; };
    auto tiles_known = [&](int64_t n) { return max_q > 0 ? std::min(n, (int64_t)B * ((max_q * g + tr - 1) / tr) * kv_heads) : n; };
    // (the sequences' rules are attn_plan's)
    const bool few = tiles_known(tiles_of(B, 0)) <= slots / 2;
    const bool seq_tiles = rows > (few ? (D == 512 ? 15 : 16) : 16 * qt_max);
    const bool group_tiles = seq_tiles || group_rows > 16 * std::min(qt_max, 2);
    if (!seq_tiles) {
        const int64_t r = group_tiles ? rows : std::max(rows, group_rows);
        p.qt = std::min(qt_max, r <= 16 ? 1 : (r <= 32 ? 2 : 4));
        p.row_limit = group_tiles ? 16 * p.qt : INT64_MAX;
        p.grid = device_cus() * (rows_two(D, p.qt, e8) ? 2 : 1);
        p.rows_bytes = (uint64_t)p.grid * 2 * 16 * p.qt * (D + 2) * sizeof(float);
    }
    p.part_bytes = p.rows_bytes;
    if (group_tiles) {
        p.grid_tiles = tiles_of(groups, p.row_limit) + tiles_of(B, p.row_limit);
        const bool own = seq_tiles || max_q == 0 || max_q * g > p.row_limit;  // sequences that are tiles
        p.tiles = std::min(p.grid_tiles, tiles_of(groups, p.row_limit) + (own ? tiles_known(tiles_of(B, p.row_limit)) : 0));
        if (p.tiles <= slots / 2 && p.tiles <= kSplitTiles) {
            p.slots = (int)slots;
            p.part_bytes += std::min((uint64_t)slots * 2, (uint64_t)p.tiles * kMaxParts) * tr * (D + 2) * sizeof(float);
        }
    }
    return p;
}

// Dynamic LDS past 64 KiB, asked for once per kernel and device.
__attribute__((unused)) int allow_lds(const void* k, int lds, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (int rc = hip_check(hipGetDevice(&dev), "hipGetDevice")) return rc;
    if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return ALV_OK;
    if (int rc = hip_check(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute"))
        return rc;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return ALV_OK;
}

template <int D, int QT, bool E8, bool MIX>
int launch_rows(const PagedAttnArgs& a, const AttnPlan& p, hipStream_t s) {
    constexpr bool TWO = rows_two(D, QT, E8);
    constexpr int lds = rows_lds(D, QT, E8, TWO);
    static_assert(lds <= kCuLds, "LDS of a CU");
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_lds(reinterpret_cast<const void*>(&attn_paged_rows_kernel<D, QT, E8, MIX>), lds, done)) return rc;
    hipLaunchKernelGGL((attn_paged_rows_kernel<D, QT, E8, MIX>), dim3(p.grid), dim3(64 * rows_waves(D, TWO)), lds, s, a);
    if (int rc = hip_check(hipGetLastError(), "attn_paged_rows_kernel launch")) return rc;
    if (MIX) return ALV_OK;
    hipLaunchKernelGGL((attn_paged_rows_merge_kernel<D, QT>), dim3(p.grid - 1, 4 * QT), dim3(256), 0, s, a);
    return hip_check(hipGetLastError(), "attn_paged_rows_merge_kernel launch");
}

template <int D, bool E8, bool MIX>
int launch_tiles(const PagedAttnArgs& a, const AttnPlan& p, hipStream_t s) {
    constexpr int lds = tile_lds(D, E8);
    static_assert(lds <= kCuLds, "LDS of a CU");
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_lds(reinterpret_cast<const void*>(&attn_paged_tile_kernel<D, E8, MIX>), lds, done)) return rc;
    hipLaunchKernelGGL((attn_paged_tile_kernel<D, E8, MIX>), dim3((uint32_t)std::max(p.grid_tiles, (int64_t)p.slots * 2)), dim3(64 * tile_waves(D)), lds, s, a);
    if (int rc = hip_check(hipGetLastError(), "attn_paged_tile_kernel launch")) return rc;
    if (MIX || p.slots == 0) return ALV_OK;
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

template <int D, bool E8, bool MIX>
int launch_d(PagedAttnArgs a, const AttnPlan& p, hipStream_t s) {
    a.grid = p.grid;
    a.tile_places = p.slots ? (int)std::min((int64_t)p.slots * 2, p.tiles * kMaxParts) : 0;
    a.row_limit = p.row_limit;
    a.slots = p.slots;
    a.max_items = p.slots ? (int)p.tiles : 0;
    a.max_tiles = (int)(p.grid_tiles / a.kv_heads);
    float* part = a.part;
    a.tile_part = part + (p.rows_bytes + p.tab_bytes) / sizeof(float);
    if (p.grid_tiles) {
        if (!MIX && p.slots) a.tab = reinterpret_cast<int*>(part + p.rows_bytes / sizeof(float));
        a.part = a.tile_part;
        if (int rc = launch_tiles<D, E8, MIX>(a, p, s)) return rc;
    }
    a.cuts = reinterpret_cast<int*>(part);
    a.part = part + p.cuts_bytes / sizeof(float);
    auto join = [&](auto qt) {
        if constexpr (!MIX) return ALV_OK;
        // Four waves to a row where rows are few (8 samples of one prompt, 32 rows: 11 us, 6).
        const int64_t rows = (int64_t)a.b.T * a.heads;
        constexpr int QT = decltype(qt)::value;
        if (rows <= 1024)
            hipLaunchKernelGGL((attn_paged_join_kernel<D, QT, 4>), dim3((uint32_t)rows), dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL((attn_paged_join_kernel<D, QT, 1>), dim3((uint32_t)std::min((rows + 3) / 4, (int64_t)1 << 22)),
                               dim3(256), 0, s, a);
        return hip_check(hipGetLastError(), "attn_paged_join_kernel launch");
    };
    auto rows_run = [&](auto qt) {
        if (p.qt)
            if (int rc = launch_rows<D, decltype(qt)::value, E8, MIX>(a, p, s)) return rc;
        return join(qt);
    };
    if constexpr (D <= 256)
        if (p.qt == 2) return rows_run(std::integral_constant<int, 2>());
    if constexpr (D <= 128)
        if (p.qt == 4) return rows_run(std::integral_constant<int, 4>());
    return rows_run(std::integral_constant<int, 1>());
}

// The arguments' checks that all attention entries share, and what they fill in of
// `a` (which holds pools, strides, heads, window, sinks, scale, out and, of 8-bit pages, scales).
__attribute__((unused)) int attn_check(PagedAttnArgs* a, int D, const int32_t* page_table, int64_t ld_table, int max_pages,
                                       const int32_t* q_start, const int32_t* kv_len, int B, int T, int pages, int page_size,
                                       int max_q) {
    if (int rc = paged_batch(page_table, ld_table, max_pages, q_start, kv_len, B, T, pages, page_size, &a->b)) return rc;
    const int heads = a->heads, kv_heads = a->kv_heads;
    if (!a->kpages || !a->vpages || (T > 0 && (!a->q || !a->out))) return fail(ALV_ERR_ARG, "null pointer");
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || (D != 64 && D != 128 && D != 256 && D != 512) || a->window < 0 ||
        a->sinks < 0 || max_q < 0 || a->ld_q < (int64_t)heads * D || a->ld_out < (int64_t)heads * D)
        return fail(ALV_ERR_ARG, "bad attention shape heads=%d kv_heads=%d D=%d window=%d sinks=%d ld_q=%lld ld_out=%lld "
                    "(D one of 64, 128, 256, 512)", heads, kv_heads, D, a->window, a->sinks, (long long)a->ld_q,
                    (long long)a->ld_out);
    if (heads > kMaxHeads) return fail(ALV_ERR_RANGE, "%d heads (at most %d)", heads, kMaxHeads);
    if (!(a->scale >= 0.0f) || a->scale > 3e38f) return fail(ALV_ERR_ARG, "scale %g: finite and not negative", (double)a->scale);
    const int64_t page_values = (int64_t)kv_heads * page_size * D;
    if (a->k_stride < page_values || a->v_stride < page_values)
        return fail(ALV_ERR_ARG, "page strides %lld and %lld hold fewer than the page's %lld values", (long long)a->k_stride,
                    (long long)a->v_stride, (long long)page_values);
    if (a->scales && a->s_stride < 2 * (int64_t)kv_heads * page_size)
        return fail(ALV_ERR_ARG, "scales %lld apart hold fewer than a page's %lld", (long long)a->s_stride,
                    2ll * kv_heads * page_size);
    const int per = a->scales ? 16 : 8;  // values of 16 bytes
    if (a->scales && (reinterpret_cast<uintptr_t>(a->scales) % 16 || a->s_stride % 16))
        return fail(ALV_ERR_ALIGN, "scales and their pages need 16-byte alignment");
    if (reinterpret_cast<uintptr_t>(a->kpages) % 16 || reinterpret_cast<uintptr_t>(a->vpages) % 16 || a->k_stride % per ||
        a->v_stride % per || reinterpret_cast<uintptr_t>(a->q) % 16 || a->ld_q % 8 || reinterpret_cast<uintptr_t>(a->out) % 8 ||
        a->ld_out % 4)
        return fail(ALV_ERR_ALIGN, "q, kpages and vpages and their rows need 16-byte alignment, out and its rows 8-byte");
    if (T == 0) return ALV_OK;
    a->g = heads / kv_heads;
    a->g_shift = a->g & (a->g - 1) ? -1 : __builtin_ctz((unsigned)a->g);
    a->window = a->window < a->b.max_pos ? a->window : 0;  // (all positions are within it)
    if ((int64_t)T * heads > (int64_t)1 << 30)  // (the largest launch: 2^32 threads)
        return fail(ALV_ERR_RANGE, "%d rows of %d heads in one call (at most 2^30 rows times heads)", T, heads);
    return ALV_OK;
}

__attribute__((unused)) int attn_fits(const AttnPlan& p, int T, int heads, int B) {
    if (p.grid_tiles * 512 > (int64_t)UINT32_MAX)
        return fail(ALV_ERR_RANGE, "%d rows of %d heads in %d sequences: too many tiles for one call", T, heads, B);
    return ALV_OK;
}

__attribute__((unused)) int attn_workspace(const void* workspace, uint64_t have, uint64_t need) {
    if (need && (!workspace || have < need))
        return fail(ALV_ERR_ARG, "workspace of %llu bytes, %llu needed", (unsigned long long)have, (unsigned long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(ALV_ERR_ALIGN, "workspace needs 16-byte alignment");
    return ALV_OK;
}

template <bool E8, bool MIX>
int attn_launch(const PagedAttnArgs& a, int D, const AttnPlan& p, hipStream_t s) {
    switch (D) {
        case 64: return launch_d<64, E8, MIX>(a, p, s);
        case 128: return launch_d<128, E8, MIX>(a, p, s);
        case 256: return launch_d<256, E8, MIX>(a, p, s);
        default: return launch_d<512, E8, MIX>(a, p, s);
    }
}

}  // namespace
}  // namespace alv

