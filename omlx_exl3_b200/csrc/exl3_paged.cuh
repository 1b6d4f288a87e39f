// The paged batch as the kernels see it: which sequence a row belongs to, and where a position lives.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "exl3_b200.h"
#include "exl3_common.cuh"

namespace exl3 {

// A row or position that the batch's tables do not cover (a page outside the pool, a position past the
// page table's columns or the rotation table): the row or page is left out and this bit is set.
enum : uint32_t { kStatusPagedRange = 8u };

// The first s with x < cu_rows[s + 1] - skip * (s + 1), found by the whole warp with 32 probes a round (one round up to
// 32 sequences, two up to 1024). skip 0: the sequence of row x; skip 1: that of draft x, where every sequence has a draft for each
// row but its last. seqs >= 1; x at or past the end gives the last sequence.
template <int skip = 0>
__device__ __forceinline__ int seq_of_row(const int32_t* cu_rows, int seqs, int x, int lane)
{
    int lo = 0, n = seqs;                                // the answer is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) >> 5;                  // probe the last sequence of each of 32 parts
        const int probe = min(lo + (lane + 1) * step, lo + n);
        const unsigned past = __ballot_sync(0xffffffffu, cu_rows[probe] - skip * probe <= x);
        const int part = min(__popc(past), 31);
        const int end = lo + n;
        lo = min(lo + part * step, end - 1);
        n = min(step, end - lo);
    }
    return lo;
}

// Page of position `pos` of sequence s; -1 where the table has none or names one outside the pool.
__device__ __forceinline__ int page_of(const exl3_paged_desc& b, int s, int pos)
{
    const int col = pos >> (31 - __clz(b.page_size));    // a power of two
    if (pos < 0 || col >= b.table_cols) return -1;
    const int page = b.page_table[(size_t)s * b.table_cols + col];
    return page >= 0 && page < b.num_pages ? page : -1;
}

}  // namespace exl3

// Host-side check of a descriptor (EXL3_OK or a status).
int exl3_check_paged(const exl3_paged_desc* b);
