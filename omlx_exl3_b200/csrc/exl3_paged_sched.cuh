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
    int lo, hi;                                       // sequences of lo < rows * grp <= hi are this kernel's
};

// An item whose parts are to be merged; parts 0: none.
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

// The list is laid out in units with `item` more in front of every item (what its start and end cost beside its steps):
// short contexts would otherwise pile up in one share.
struct PaSched {
    const PaArgs& a;
    long long total, begin, until;                    // the list's length, the current item's place in it, this share's end
    int ctas, s, h, t, j, cap;

    __device__ __forceinline__ explicit PaSched(const PaArgs& args) : a(args) {}

    __device__ __forceinline__ int rows_of(int q) const { return a.b.cu_rows[q + 1] - a.b.cu_rows[q]; }
    __device__ __forceinline__ bool takes(int rows) const
    {
        const long long packed = (long long)rows * a.grp;
        return rows > 0 && packed > a.lo && packed <= a.hi;
    }
    // Positions the last row of item i sees, 0 .. the page table's reach.
    __device__ __forceinline__ int item_end(int rows, int len, int i) const
    {
        const int last = min(rows * a.grp, (i + 1) * a.span) - 1;
        const long long e = (long long)len - rows + last / a.grp + 1;
        return (int)max(0ll, min(e, (long long)cap));
    }
    __device__ __forceinline__ static int units_of(int end) { return max(1, (end + kPaStep - 1) / kPaStep); }

    __device__ __forceinline__ long long seq_length(int q) const
    {
        const int rows = q < a.b.seqs ? rows_of(q) : 0;
        if (!takes(rows)) return 0;
        const int len = a.b.lens[q];
        long long n = 0;
        for (int i = 0; i * a.span < rows * a.grp; ++i) n += units_of(item_end(rows, len, i)) + a.item;
        return n * a.b.hkv;
    }

    // All lanes of the warp. This CTA's share of the list, and where it starts.
    __device__ __forceinline__ void start(int cta, int grid, int lane)
    {
        cap = a.b.table_cols * a.b.page_size;
        long long first = 0;                          // this lane's part of the first 32 sequences
        total = 0;
        for (int q0 = 0; q0 < a.b.seqs; q0 += 32) {
            long long n = seq_length(q0 + lane);
            if (q0 == 0) first = n;
#pragma unroll
            for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
            total += n;
        }
        s = h = t = j = 0;
        begin = until = 0;
        ctas = (int)min((long long)grid, total);
        if (cta >= ctas) return;
        const long long u = total * cta / ctas;
        until = total * (cta + 1) / ctas;
        long long before = 0, at = 0;
        for (int q0 = 0; q0 < a.b.seqs; q0 += 32) {
            const long long n = q0 == 0 ? first : seq_length(q0 + lane);
            long long sum = n;                        // inclusive prefix
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            const int k = __popc(__ballot_sync(0xffffffffu, before + sum <= u));
            if (k < 32) {
                s = q0 + k;
                at = u - before - (__shfl_sync(0xffffffffu, sum, k) - __shfl_sync(0xffffffffu, n, k));
                const long long per = __shfl_sync(0xffffffffu, n, k) / a.b.hkv;
                h = (int)(at / per);
                at -= per * h;
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        const int rows = rows_of(s), len = a.b.lens[s];
        for (;;) {
            const int n = units_of(item_end(rows, len, t)) + a.item;
            if (at < n) break;
            at -= n;
            ++t;
        }
        begin = u - at;
        j = max(0, (int)at - a.item);                 // at < n: one of the item's units
    }

    __device__ __forceinline__ int cta_of(long long place) const { return (int)(((place + 1) * ctas - 1) / total); }

    // The next segment of this CTA's share; false when it is done.
    __device__ __forceinline__ bool next(PaSeg& g)
    {
        if (begin + a.item >= until) return false;    // no unit of the current item is in the share
        const int rows = rows_of(s), len = a.b.lens[s];
        g.s = s;
        g.h = h;
        g.p0 = t * a.span;
        g.start = a.b.cu_rows[s];
        g.rows = rows;
        g.ctx = (int)max(-(1ll << 30), (long long)len - rows);
        g.end = item_end(rows, len, t);
        g.units = units_of(g.end);
        g.j0 = j;
        g.j1 = (int)min((long long)g.units, until - begin - a.item);
        const bool cut = j > 0 || g.j1 < g.units;
        g.c0 = cut ? cta_of(begin + a.item) : 0;
        g.c1 = cut ? cta_of(begin + a.item + g.units - 1) : 0;
        j = 0;
        begin += a.item + g.units;
        if (begin < until) {
            if ((t + 1) * a.span < rows * a.grp) {
                ++t;
            } else {
                t = 0;
                if (++h == a.b.hkv) {
                    h = 0;
                    do ++s;
                    while (s < a.b.seqs - 1 && !takes(rows_of(s)));
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
__device__ __forceinline__ void pa_record(const PaArgs& a, bool any, const PaSeg& g, int used, int gap)
{
    PaItem it{};
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

// One launch over the sequences a.lo < rows * grp <= a.hi. Both set a.span and a.item.
int pa_launch_tiles(const PaArgs& a, cudaStream_t s);     // exl3_paged_attn.cu: tensor-core tiles of 256 packed rows
int pa_launch_few(const PaArgs& a, cudaStream_t s);       // exl3_paged_few.cu: up to 16 packed rows at a time

// Merges what either or both left in parts (exl3_paged_merge.cu).
int pa_launch_merge(const PaArgs* tiles, const PaArgs* few, int ctas, cudaStream_t s);

}  // namespace exl3
