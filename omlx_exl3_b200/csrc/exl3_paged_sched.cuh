// Work list of the paged attention kernels, worked out by each warp from the batch's device tables.
//
// An item is `span` packed query rows (row = token * group + head) of one (sequence, kv head); its units are steps of
// 128 positions up to the last position any of its rows sees. All items' units form one list (sequence, kv head,
// item) and every CTA takes an equal contiguous share of it, so ragged batches load all SMs evenly and the host needs to
// know no length. A share's end may cut an item: the CTAs that share one leave fp32 partials (m, l, O) in the
// workspace, and a second small kernel merges them in CTA order (exl3_paged_merge.cu). Every CTA records the item
// that starts in its share and leaves it, if one does; nothing in the workspace needs a value from before the call.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "exl3_b200.h"
#include "exl3_common.cuh"
#include "exl3_paged.cuh"
#include "exl3_paged_math.cuh"

namespace exl3 {

constexpr int kPaStep = 128;                          // positions of a unit
constexpr int kPaRows = 128;                          // packed rows of a tensor-core tile
constexpr int kPaFew = 16;                            // packed rows that the kernel for few rows takes at once
constexpr float kPaSlack = 8.0f;                      // log2 growth of a row's maximum before its accumulator is rescaled

struct PaArgs {
    exl3_paged_desc b;
    const void* q;
    long long q_stride;
    void* out;
    struct PaItem* items;                             // [CTAs] the item that starts in the CTA's share and leaves it
    uint8_t* parts;                                   // [CTAs][2: began before this CTA, begins in it][tiles]
    uint32_t* status;
    float scale_log2;
    int hq, grp, span, item;
    uint32_t grp_magic;                               // ceil(2^32 / grp): x / grp = umulhi(x, grp_magic) for x < 2^25 (0: grp is 1)
    int behind;                                       // launched behind the tile kernel, which it need not wait for to begin
    int lo, hi;                                       // sequences of lo < rows * grp <= hi are this kernel's
};

// An item whose parts are to be merged; parts 0: none; -1: cu_rows is no list of rows, and nothing was computed.
struct PaItem {
    int parts, c0, h, start, p0, used, gap, pad;      // first packed row, packed rows; rows of tile 1 follow `gap` after p0
};

// One partial of up to ROWS packed rows: O as [column quad][used row][4], then (m, l) per row.
template <int HD, int ROWS>
struct PaPart {
    static constexpr size_t kMl = (size_t)ROWS * HD * 4;
    static constexpr size_t kBytes = kMl + ROWS * 8;
};

struct PaSeg {
    int s, h, p0;                                     // sequence, kv head, first packed row
    int start, rows, ctx;                             // the sequence's first row, its rows, position of its first row
    int j0, j1, units, end;                           // this CTA's units of the item, all of them, positions its last row sees
    int c0, c1;                                       // the CTAs that share the item
};

__device__ __forceinline__ int by_grp(const PaArgs& a, int x) { return a.grp_magic ? (int)__umulhi((uint32_t)x, a.grp_magic) : x; }

// The list is laid out in units with `item` more in front of every item (what its start and end cost beside its steps):
// short contexts would otherwise pile up in one share. A share is ceil(length / CTAs) units. All of it is 32-bit and nearly
// free of divisions (the host has checked that the list is short enough): this runs before the first load of a call.
struct PaSched {
    const PaArgs& a;
    int share, begin, until;                          // a share's length, the current item's place in the list, this share's end
    int s, h, t, j, cap;
    int rows, len;                                    // of sequence s
    bool bad;                                         // cu_rows falls somewhere, or leaves 0 .. b.rows

    __device__ __forceinline__ explicit PaSched(const PaArgs& args) : a(args) {}

    __device__ __forceinline__ bool takes(int r) const { return r > 0 && r * a.grp > a.lo && r * a.grp <= a.hi; }
    // Positions the last row of item i sees, 0 .. the page table's reach.
    __device__ __forceinline__ int item_end(int r, int n, int i) const
    {
        const int e = n - r + by_grp(a, min(r * a.grp, (i + 1) * a.span) - 1) + 1;
        return max(0, min(e, cap));
    }
    __device__ __forceinline__ static int units_of(int end) { return max(1, (end + kPaStep - 1) / kPaStep); }

    // Rows and length of sequence q: a length that could not be one is taken as the nearest that could. False where the rows are out
    // of order or of range; all three words are asked for before any is looked at.
    __device__ __forceinline__ bool load(int q, int& r, int& n) const
    {
        const int lo = a.b.cu_rows[q], hi = a.b.cu_rows[q + 1], len = a.b.lens[q];
        r = hi - lo;
        n = max(0, min(len, cap + a.b.rows));
        return (lo >= 0) & (hi >= lo) & (hi <= a.b.rows);
    }

    // Length of sequence q in the list, for one kv head; -1: its rows are out of order or out of range.
    __device__ __forceinline__ int head_length(int q) const
    {
        if (q >= a.b.seqs) return 0;
        int r, n, sum = 0;
        if (!load(q, r, n)) return -1;
        if (!takes(r)) return 0;
        for (int i = 0; i * a.span < r * a.grp; ++i) sum += units_of(item_end(r, n, i)) + a.item;
        return sum;
    }

    // All lanes of the warp. This CTA's share of the list, and where it starts. Rows that rise from sequence to sequence within
    // 0 .. b.rows are no more than b.rows in all, which is what the list's 32 bits and every row index below rest on; any other
    // cu_rows gives an empty list.
    __device__ __forceinline__ void start(int cta, int grid, int lane)
    {
        cap = a.b.table_cols * a.b.page_size;
        int first = 0, total = 0;                     // first: this lane's part of the first 32 sequences
        bad = false;
        for (int q0 = 0; q0 < a.b.seqs; q0 += 32) {
            const int n = head_length(q0 + lane);
            if (q0 == 0) first = n;
            bad |= __any_sync(0xffffffffu, n < 0);
            total += __reduce_add_sync(0xffffffffu, n) * a.b.hkv;
        }
        s = h = t = j = 0;
        begin = until = 0;
        if (bad) total = 0;
        share = (total + grid - 1) / grid;
        const int u = cta * share;
        if (u >= total) return;
        until = min(total, u + share);
        int before = 0, at = 0;
        for (int q0 = 0; q0 < a.b.seqs; q0 += 32) {
            const int n = q0 == 0 ? first : head_length(q0 + lane);
            int sum = n;                              // inclusive prefix
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            const int k = __popc(__ballot_sync(0xffffffffu, before + sum * a.b.hkv <= u));
            if (k < 32) {
                const int per = __shfl_sync(0xffffffffu, n, k);
                s = q0 + k;
                at = u - before - (__shfl_sync(0xffffffffu, sum, k) - per) * a.b.hkv;
                h = at / per;
                at -= per * h;
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31) * a.b.hkv;
        }
        load(s, rows, len);
        for (;;) {
            const int n = units_of(item_end(rows, len, t)) + a.item;
            if (at < n) break;
            at -= n;
            ++t;
        }
        begin = u - at;
        j = max(0, at - a.item);                      // at < n: one of the item's units
    }

    // The next segment of this CTA's share; false when it is done.
    __device__ __forceinline__ bool next(PaSeg& g)
    {
        if (begin + a.item >= until) return false;    // no unit of the current item is in the share
        g.s = s;
        g.h = h;
        g.p0 = t * a.span;
        g.start = a.b.cu_rows[s];
        g.rows = rows;
        g.ctx = len - rows;
        g.end = item_end(rows, len, t);
        g.units = units_of(g.end);
        g.j0 = j;
        g.j1 = min(g.units, until - begin - a.item);
        g.c0 = g.c1 = 0;
        if (j > 0 || g.j1 < g.units) {
            g.c0 = (begin + a.item) / share;
            g.c1 = (begin + a.item + g.units - 1) / share;
        }
        j = 0;
        begin += a.item + g.units;
        if (begin < until) {
            if ((t + 1) * a.span < rows * a.grp) {
                ++t;
            } else {
                t = 0;
                if (++h == a.b.hkv) {
                    h = 0;
                    do load(++s, rows, len);
                    while (s < a.b.seqs - 1 && !takes(rows));
                }
            }
        }
        return true;
    }
};

// exp2((m - top) * c), 0 for a row that has seen nothing (m = -inf).
__device__ __forceinline__ float pa_weight(float m, float top, float c)
{
    return m == -INFINITY ? 0.f : ex2((m - top) * c);
}

template <typename C>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint32_t r;
    if constexpr (sizeof(C) == 2 && __is_same(C, __half)) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The partial that CTA `cta` leaves of an item that starts in CTA c0.
template <int HD, int ROWS, int TILES>
__device__ __forceinline__ uint8_t* pa_part(uint8_t* parts, int c0, int cta, int tile)
{
    return parts + ((size_t)(cta * 2 + (cta == c0 ? 1 : 0)) * TILES + tile) * PaPart<HD, ROWS>::kBytes;
}

// After its last segment g (any == false: it had none) a CTA records the item that it starts and does not finish.
__device__ __forceinline__ void pa_record(const PaArgs& a, bool bad, bool any, const PaSeg& g, int used, int gap)
{
    PaItem it{};
    if (bad) {
        it.parts = -1;
        if (blockIdx.x == 0) atomicOr(a.status, kStatusPagedRange);
    }
    if (any && g.j0 == 0 && g.j1 < g.units) {
        it.parts = g.c1 - g.c0 + 1;
        it.c0 = g.c0;
        it.h = g.h;
        it.start = g.start;
        it.p0 = g.p0;
        it.used = used;
        it.gap = gap;
    }
    a.items[blockIdx.x] = it;
}

// Whether every batch of these sizes has a list that 32 bits hold (and rows that by_grp divides); items of `span` rows.
inline bool pa_list_fits(const PaArgs& a, int span)
{
    const long long packed = (long long)a.b.rows * a.grp;
    const long long steps = ((long long)a.b.table_cols * a.b.page_size + kPaStep - 1) / kPaStep + 8;
    return packed < (1 << 25) && (packed / span + a.b.seqs) * a.b.hkv < 0x7fffffffll / steps;
}

// One launch over the sequences a.lo < rows * grp <= a.hi. Both set a.span and a.item.
int pa_launch_tiles(const PaArgs& a, cudaStream_t s);     // exl3_paged_attn.cu: tensor-core tiles of 256 packed rows
int pa_launch_few(const PaArgs& a, cudaStream_t s);       // exl3_paged_few.cu: up to 16 packed rows at a time

// Merges what either or both left in parts (exl3_paged_merge.cu).
int pa_launch_merge(const PaArgs* tiles, const PaArgs* few, int ctas, cudaStream_t s);

}  // namespace exl3
