// The paged KV cache and the batch of sequences that the paged kernels share.
//
// Pages are (page, kv head, slot, column) bf16, consecutive pages `k_stride` /
// `v_stride` values apart; position p of sequence b is slot p % S of page
// table[b * ld_table + p / S] (S a power of two). An entry outside [0, pages)
// holds no positions: nothing is read from it or written to it.
//
// Sequence b owns the packed rows [q_start[b], q_start[b + 1]); they are the
// last of its kv_len[b] positions. A sequence whose rows do not fit its length,
// or whose length does not fit its table row, is malformed: its rows get zeros.
// Rows outside every sequence or past the batch's T are never touched, so any
// contents of q_start, kv_len and the table stay in bounds.
#pragma once

#include <stdint.h>

#include "q4_host.h"

namespace alv {

struct PagedBatch {
    const int32_t* table;
    const int32_t* q_start;  // B + 1
    const int32_t* kv_len;   // B
    int64_t ld_table;
    int B, T, max_pages, pages, shift;  // shift: log2 of the page size
    int max_pos;                        // positions a table row takes
};

constexpr int kPageMin = 16, kPageMax = 1024;
constexpr int kMaxRows = 1 << 22;  // 512 threads a row stay within a launch's 2^32 threads

constexpr int kMaxHeads = 1 << 16;  // a row's offsets stay within 32 bits

inline int page_shift(int page_size) { return 31 - __builtin_clz((unsigned)page_size); }

// Checks of the arguments every paged entry point shares, and the batch.
inline int paged_batch(const int32_t* table, int64_t ld_table, int max_pages, const int32_t* q_start,
                       const int32_t* kv_len, int B, int T, int pages, int page_size, PagedBatch* out) {
    if (!table || !q_start || !kv_len) return fail(ALV_ERR_ARG, "null pointer");
    if (page_size < kPageMin || page_size > kPageMax || (page_size & (page_size - 1)))
        return fail(ALV_ERR_ARG, "page size %d: a power of two from %d to %d", page_size, kPageMin, kPageMax);
    if (B < 1 || T < 0 || pages < 1 || max_pages < 1 || ld_table < max_pages)
        return fail(ALV_ERR_ARG, "bad batch B=%d T=%d pages=%d max_pages=%d ld_table=%lld", B, T, pages, max_pages,
                    (long long)ld_table);
    if (T > kMaxRows) return fail(ALV_ERR_RANGE, "%d rows in one call (at most %d)", T, kMaxRows);
    if ((int64_t)max_pages * page_size > (int64_t)1 << 30)
        return fail(ALV_ERR_RANGE, "%d pages of %d positions per sequence (at most 2^30 positions)", max_pages, page_size);
    if (reinterpret_cast<uintptr_t>(table) % 4 || reinterpret_cast<uintptr_t>(q_start) % 4 ||
        reinterpret_cast<uintptr_t>(kv_len) % 4)
        return fail(ALV_ERR_ALIGN, "page_table, q_start and kv_len need 4-byte alignment");
    *out = PagedBatch{table, q_start, kv_len, ld_table, B, T, max_pages, pages, page_shift(page_size),
                      max_pages * page_size};
    return ALV_OK;
}

#ifdef __HIPCC__
namespace {

struct SeqRows {
    int seq;   // -1: the row belongs to no sequence
    int first; // its first packed row
    int n;     // its rows
    int len;   // its positions
    bool ok;   // well formed
};

__device__ __forceinline__ bool seq_ok(const PagedBatch& a, int first, int n, int len) {
    return first >= 0 && n >= 0 && first + (int64_t)n <= a.T && n <= len && len <= a.max_pos;
}

// The sequence that owns packed row t, by the whole wave (t uniform): each lane
// looks at one sequence per step, so a batch of up to 64 costs one round of
// loads.
__device__ __forceinline__ SeqRows find_row(const PagedBatch& a, int t, int lane) {
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = b0 + lane;
        int lo = 0, hi = 0, len = 0;
        if (b < a.B) {
            lo = a.q_start[b];
            hi = a.q_start[b + 1];
            len = a.kv_len[b];
        }
        const uint64_t m = __ballot(b < a.B && lo <= t && t < hi);
        if (m) {
            const int l = __builtin_ctzll(m);
            SeqRows r;
            r.seq = b0 + l;
            r.first = __builtin_amdgcn_readlane(lo, l);
            r.n = __builtin_amdgcn_readlane(hi, l) - r.first;
            r.len = __builtin_amdgcn_readlane(len, l);
            r.ok = seq_ok(a, r.first, r.n, r.len);
            return r;
        }
    }
    return SeqRows{-1, 0, 0, 0, false};
}

// The page of position p (0 <= p < max_pos) of sequence b, or -1.
__device__ __forceinline__ int page_of(const PagedBatch& a, int b, int p) {
    const int e = a.table[(int64_t)b * a.ld_table + (p >> a.shift)];
    return (unsigned)e < (unsigned)a.pages ? e : -1;
}

}  // namespace
#endif

}  // namespace alv
