// Attention of a batch's new rows over paged keys and values (fp16 / bf16, head_dim 64 or 128, grouped heads),
// for chunks of thousands of rows and single decoded tokens alike.
//
//   out[r, h] = sum_j p_j V[j, h / g] / sum_j p_j,  p_j = exp(scale q[r, h] . K[j, h / g] - m),  j <= pos(r)
//
// Tiles. The g query heads of a kv head are packed with T = 128 / g consecutive rows of a sequence into the 128
// rows of a tile (row = token * g + head), so a kv head's keys and values are read once for its whole group. One
// work item is two such tiles (2 T tokens) of one (sequence, kv head); an item of T tokens or fewer has one tile.
// Per step of 128 positions, tcgen05.mma computes S = Q K^T into tensor memory (fp32), one softmax thread per row
// reads its row, keeps the running maximum and sum in registers, writes P back over S in the 16-bit type, and a
// second tcgen05.mma adds P V to the accumulator in tensor memory.
//
// Roles of a CTA (one per SM, persistent): two softmax warpgroups, one warp that loads with TMA, one that
// issues the MMAs. The tensor core alternates between two slots (S, P and O of their own) and works on one while the
// other slot's softmax runs. In a two-tile item slot = tile; in a one-tile item the slots take alternate steps of the
// same rows and are merged at its end. The accumulator is rescaled only when a row's maximum grows by more than 2^8
// (P <= 256 is exact enough in either type, and the sum is fp32 of the unrounded p), by the softmax thread itself: S of
// step j is only complete when P V of step j - 1 is, so nothing else touches the accumulator then.
//
// Split. All items' steps form one list (sequence, kv head, tile); each CTA takes an equal contiguous share of it,
// computed by every warp from the device tables, so ragged batches and long contexts load all SMs evenly without
// the host knowing a length. An item cut by a share's end leaves fp32 partials (m, l, O) in the workspace; the CTA that
// arrives last on the item's counter merges them in CTA order: the result does not depend on who was last,
// and no CTA waits for another.
//
// Positions are gathered by page: a step's tile is 128 / page_size TMA boxes per 64 columns (one for larger pages), pages
// past the sequence's end are not read (zero fill), and what lies behind the end in its last page is masked in S and
// zeroed in V's tile, since 0 * NaN would pass through the product.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "exl3_b200.h"
#include "exl3_common.cuh"
#include "exl3_host.h"
#include "exl3_paged.cuh"
#include "exl3_tc.cuh"

namespace exl3 {

constexpr int kPaRows = 128;                          // packed query rows of a tile, and TMEM lanes
constexpr int kPaStep = 128;                          // positions of a step
constexpr int kPaThreads = 384;                       // two softmax warpgroups; one with the load and the MMA warp
// Registers of a softmax thread (a row's 128 scores stay in registers) and of the others: 2 x 200 + 104 = 3 x 168, what the
// launch gives the three warpgroups together.
constexpr int kPaSoftmaxRegs = 200, kPaOtherRegs = 104;
constexpr int kPaBarBytes = 512;
constexpr uint64_t kPaExitNs = 100000000ull;          // wait for a CTA's own copies and MMAs before it exits
constexpr float kPaSlack = 8.0f;                      // log2 growth of a row's maximum before its accumulator is rescaled

template <int HD>
struct PaShape {
    static constexpr int kPanels = HD / 64;           // 128-byte swizzled panels of a tile
    static constexpr int kTile = kPaRows * HD * 2;    // bytes of a Q, K or V tile
    static constexpr int kPanel = kPaRows * 128;
    static constexpr int kStages = HD == 128 ? 5 : 8;
    static constexpr int kMl = kPaRows * 8;           // slot 1's (m, l) for the merge of a one-tile item
    static constexpr int kSmem = 1024 + 2 * kTile + kStages * kTile + kMl + kPaBarBytes;
    static constexpr size_t kPart = (size_t)kPaRows * HD * 4 + kPaRows * 8;   // partial O and (m, l) of one tile
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct PaArgs {
    exl3_paged_desc b;
    void* out;
    uint32_t* counters;                               // [CTAs][2] arrivals of the item that starts in the CTA and leaves it
    uint8_t* parts;                                   // [CTAs][2: began before this CTA, begins in it][2 tiles]
    uint32_t* status;
    float scale_log2;
    int hq, grp, tokens;                              // tokens of a tile
};

// ------------------------------------------------------------------------------ schedule
struct PaSeg {
    int s, h, row0, pos0, ntok[2], rows_used[2];      // sequence, kv head, first row and its position, tokens / rows of the tiles
    int j0, j1, units, end;                           // this CTA's steps of the item, all of them, first position past the last row
    bool dual;
    int c0, c1;                                       // the CTAs that share the item
};

struct PaSched {
    const PaArgs& a;
    long long total, u, left;
    int ctas, s, h, t, j, cap;

    __device__ __forceinline__ explicit PaSched(const PaArgs& args) : a(args) {}

    __device__ __forceinline__ int item_end(int rows, int len, int t) const
    {
        const long long e = (long long)len - rows + min(rows, (t + 1) * 2 * a.tokens);
        return (int)max(0ll, min(e, (long long)cap));
    }
    __device__ __forceinline__ static int units_of(int end) { return max(1, (end + kPaStep - 1) / kPaStep); }

    __device__ __forceinline__ long long seq_units(int q) const
    {
        const int rows = q < a.b.seqs ? a.b.cu_rows[q + 1] - a.b.cu_rows[q] : 0;
        if (rows <= 0) return 0;
        const int len = a.b.lens[q];
        long long n = 0;
        const int items = (rows + 2 * a.tokens - 1) / (2 * a.tokens);
        for (int i = 0; i < items; ++i) n += units_of(item_end(rows, len, i));
        return n * a.b.hkv;
    }

    // All lanes of the warp. This CTA's share of the list, and where it starts.
    __device__ __forceinline__ void start(int cta, int grid, int lane)
    {
        cap = a.b.table_cols * a.b.page_size;
        long long first = 0;                          // this lane's units of the first 32 sequences
        total = 0;
        for (int q0 = 0; q0 < a.b.seqs; q0 += 32) {
            long long n = seq_units(q0 + lane);
            if (q0 == 0) first = n;
#pragma unroll
            for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
            total += n;
        }
        s = h = t = j = 0;
        left = 0;
        u = 0;
        ctas = (int)min((long long)grid, total);
        if (cta >= ctas) return;
        u = total * cta / ctas;
        left = total * (cta + 1) / ctas - u;
        long long before = 0, at = 0;
        for (int q0 = 0; q0 < a.b.seqs; q0 += 32) {
            const long long n = q0 == 0 ? first : seq_units(q0 + lane);
            long long sum = n;                        // inclusive prefix
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + sum <= u);
            const int k = __popc(past);
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
        const int rows = a.b.cu_rows[s + 1] - a.b.cu_rows[s], len = a.b.lens[s];
        for (;;) {
            const int n = units_of(item_end(rows, len, t));
            if (at < n) break;
            at -= n;
            ++t;
        }
        j = (int)at;
    }

    __device__ __forceinline__ int cta_of(long long unit) const { return (int)(((unit + 1) * ctas - 1) / total); }

    // The next segment of this CTA's share; false when it is done.
    __device__ __forceinline__ bool next(PaSeg& g)
    {
        if (left <= 0) return false;
        const int start_row = a.b.cu_rows[s];
        const int rows = a.b.cu_rows[s + 1] - start_row, len = a.b.lens[s];
        const int tok0 = t * 2 * a.tokens, ntok = min(rows - tok0, 2 * a.tokens);
        g.s = s;
        g.h = h;
        g.row0 = start_row + tok0;
        g.pos0 = (int)max(-(1ll << 30), (long long)len - rows + tok0);
        g.dual = ntok > a.tokens;
        g.ntok[0] = min(ntok, a.tokens);
        g.ntok[1] = ntok - g.ntok[0];
        g.rows_used[0] = g.ntok[0] * a.grp;
        g.rows_used[1] = g.ntok[1] * a.grp;
        g.end = item_end(rows, len, t);
        g.units = units_of(g.end);
        g.j0 = j;
        g.j1 = (int)min((long long)g.units, j + left);
        g.c0 = cta_of(u - j);
        g.c1 = cta_of(u - j + g.units - 1);
        const int n = g.j1 - g.j0;
        left -= n;
        u += n;
        j = 0;
        if (left > 0) {
            if (tok0 + 2 * a.tokens < rows) {
                ++t;
            } else {
                t = 0;
                if (++h == a.b.hkv) {
                    h = 0;
                    do ++s;
                    while (s < a.b.seqs - 1 && a.b.cu_rows[s + 1] <= a.b.cu_rows[s]);
                }
            }
        }
        return true;
    }
};

// ------------------------------------------------------------------------------ instructions
template <typename C>
constexpr uint32_t pa_idesc(int n, bool v_major)
{
    const uint32_t fmt = std::is_same<C, __nv_bfloat16>::value ? 1u : 0u;     // both operands of one type
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (v_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kPaRows >> 4) << 24);
}

// V's tile as the B operand of P V: stored position by position, so its N (column) axis is the contiguous one.
// 128-byte swizzle; panels of 64 columns `panel` bytes apart, groups of 8 positions 1024 bytes apart.
__device__ __forceinline__ uint64_t pa_desc_v(const void* p, uint32_t panel)
{
    const uint64_t addr = smem_addr(p);
    return ((addr >> 4) & 0x3FFFull) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename C>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint32_t r;
    if constexpr (std::is_same<C, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Bounded wait of a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns = 2000000000ull)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, limit_ns));
}

// exp2((m - top) * c), 0 for a row that has seen nothing (m = -inf).
__device__ __forceinline__ float pa_weight(float m, float top, float c)
{
    return m == -INFINITY ? 0.f : ex2((m - top) * c);
}

// ------------------------------------------------------------------------------ kernel
template <typename C, int HD>
__global__ void __launch_bounds__(kPaThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PaArgs a)
{
    using P = PaShape<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_s = smem;                              // two tiles; the second is the merge buffer of one-tile items
    uint8_t* kv_s = smem + 2 * P::kTile;
    float2* ml_s = reinterpret_cast<float2*>(kv_s + P::kStages * P::kTile);
    uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(ml_s) + P::kMl);
    uint64_t* full = bars;                            // [stages] a K or V tile has landed
    uint64_t* empty = full + P::kStages;              // [stages] its MMAs are done
    uint64_t* q_full = empty + P::kStages;
    uint64_t* q_empty = q_full + 1;                   // the item's S are done and its merge buffer is read
    uint64_t* s_full = q_empty + 1;                   // [2] S of the slot is complete (and the P V before it)
    uint64_t* p_full = s_full + 2;                    // [2] P of the slot is written
    uint64_t* o_full = p_full + 2;                    // [2] the slot's accumulator is complete
    uint64_t* o_empty = o_full + 2;                   // [2] it has been read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_empty + 2);
    uint32_t* last_flag = tmem_slot + 1;              // [2]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < P::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1 + 8);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
            mbar_init(&o_empty[i], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;                 // S of slot i at column 128 i, O at 256 + HD i
    pdl_trigger();
    pdl_wait();

    PaSched sched(a);
    PaSeg g{};
    bool ok = true;

    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPaOtherRegs));
      if (warp == 8) {
        sched.start(blockIdx.x, gridDim.x, lane);
        // ---------------------------------------------------------------- loads
        const int ps = a.b.page_size;
        const int boxes = ps >= kPaStep ? 1 : kPaStep / ps;            // TMA boxes of a panel
        const int box_rows = min(ps, kPaStep);
        uint32_t n_seg = 0, it = 0;
        // this lane's page of a step (lanes past the boxes have none)
        auto page_at = [&](int step) {
            const int pos = step * kPaStep + lane * box_rows;
            if (lane >= boxes || step >= g.j1 || pos >= g.end) return -1;
            const int page = page_of(a.b, g.s, pos);
            if (page < 0) atomicOr(a.status, kStatusPagedRange);
            return page;
        };
        auto load = [&](const CUtensorMap* map, int step, int page) {
            const int st = it % P::kStages;
            if (it >= (uint32_t)P::kStages && !pa_wait(&empty[st], ((it / P::kStages) - 1) & 1)) ok = false;
            if (!ok) return;
            if (lane == 0) mbar_arrive_expect_tx(&full[st], P::kTile);
            __syncwarp();
            if (lane < boxes) {
                uint8_t* dst = kv_s + st * P::kTile + lane * box_rows * 128;
                const int y = (step * kPaStep) & (ps - 1);
#pragma unroll
                for (int p = 0; p < P::kPanels; ++p)
                    tma_load_4d(dst + p * P::kPanel, map, p * 64, boxes == 1 ? y : 0, g.h, page, &full[st]);
            }
            ++it;
        };
        while (ok && sched.next(g)) {
            if (n_seg > 0 && !pa_wait(q_empty, (n_seg - 1) & 1)) { ok = false; break; }
            if (lane == 0) {
                if ((long long)g.pos0 + g.ntok[0] + g.ntok[1] > sched.cap) atomicOr(a.status, kStatusPagedRange);
                const int tiles = g.dual ? 2 : 1;
                mbar_arrive_expect_tx(q_full, tiles * P::kPanels * a.tokens * a.grp * 128);
                for (int i = 0; i < tiles; ++i)
                    for (int p = 0; p < P::kPanels; ++p)
                        tma_load_3d(q_s + i * P::kTile + p * P::kPanel, &qmap, p * 64, g.h * a.grp, g.row0 + i * a.tokens,
                                    q_full);
            }
            __syncwarp();
            ++n_seg;
            const int n = g.j1 - g.j0, ahead = g.dual ? 1 : 2;
            int pg0 = page_at(g.j0), pg1 = page_at(g.j0 + 1), pg2 = page_at(g.j0 + 2);   // of steps m, m + 1, m + 2
            load(&kmap, g.j0, pg0);
            if (ahead == 2 && n > 1) load(&kmap, g.j0 + 1, pg1);
            for (int m = 0; m < n && ok; ++m) {
                const int pg3 = page_at(g.j0 + m + 3);
                load(&vmap, g.j0 + m, pg0);
                if (m + ahead < n) load(&kmap, g.j0 + m + ahead, ahead == 1 ? pg1 : pg2);
                pg0 = pg1;
                pg1 = pg2;
                pg2 = pg3;
            }
        }
        // nothing of this CTA may still be landing when it exits
        for (uint32_t i = it > (uint32_t)P::kStages ? it - P::kStages : 0; i < it; ++i)
            if (!pa_wait(&full[i % P::kStages], (i / P::kStages) & 1, kPaExitNs)) ok = false;
        if (n_seg > 0 && !pa_wait(q_full, (n_seg - 1) & 1, kPaExitNs)) ok = false;
      } else if (warp == 9) {
        sched.start(blockIdx.x, gridDim.x, lane);
        // ---------------------------------------------------------------- MMAs (lane 0 issues)
        constexpr uint32_t idesc_s = pa_idesc<C>(kPaStep, false), idesc_o = pa_idesc<C>(HD, true);
        uint32_t n_seg = 0, it = 0, n_p[2] = {0, 0}, n_o[2] = {0, 0};
        auto stage_wait = [&](uint32_t i) {
            if (ok && !pa_wait(&full[i % P::kStages], (i / P::kStages) & 1)) ok = false;
            tc_fence_after();
            return kv_s + (i % P::kStages) * P::kTile;
        };
        auto mma_s = [&](int slot, int tile, const uint8_t* k) {
            if (!ok || lane != 0) return;
            const uint64_t qd = smem_desc_sw128(q_s + tile * P::kTile), kd = smem_desc_sw128(k);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                const int off = ((kk / 4) * P::kPanel + (kk % 4) * 32) >> 4;
                tc_mma_f16(tmem + slot * kPaStep, qd + off, kd + off, idesc_s, kk > 0);
            }
            tc_commit(&s_full[slot]);
        };
        auto mma_o = [&](int slot, const uint8_t* v, bool first) {
            if (ok && !pa_wait(&p_full[slot], n_p[slot] & 1)) ok = false;
            ++n_p[slot];
            if (first) {
                if (n_o[slot] > 0 && ok && !pa_wait(&o_empty[slot], (n_o[slot] - 1) & 1)) ok = false;
                ++n_o[slot];
            }
            tc_fence_after();
            if (!ok || lane != 0) return;
            const uint64_t vd = pa_desc_v(v, P::kPanel);
#pragma unroll
            for (int kk = 0; kk < kPaStep / 16; ++kk)
                tc_mma_f16_ts(tmem + 256 + slot * HD, tmem + slot * kPaStep + kk * 8, vd + kk * (2048 >> 4), idesc_o,
                              (first && kk == 0) ? 0u : 1u);
        };
        auto commit = [&](uint64_t* bar) {
            if (ok && lane == 0) tc_commit(bar);
        };
        // positions past the sequence's end: their V rows become zero
        auto clean = [&](uint8_t* v, int step) {
            const int valid = g.end - step * kPaStep;
            if (valid >= kPaStep) return;
            const int lo = max(valid, 0) * 8;
            for (int i = lo + lane; i < kPaStep * 8; i += 32)
#pragma unroll
                for (int p = 0; p < P::kPanels; ++p)
                    *reinterpret_cast<uint4*>(v + p * P::kPanel + i * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
        };
        while (ok && sched.next(g)) {
            if (!pa_wait(q_full, n_seg & 1)) { ok = false; break; }
            ++n_seg;
            const int n = g.j1 - g.j0;
            if (g.dual) {
                const uint8_t* k = stage_wait(it);
                mma_s(0, 0, k);
                mma_s(1, 1, k);
                commit(&empty[it % P::kStages]);
                ++it;
                if (n == 1) commit(q_empty);
                for (int m = 0; m < n && ok; ++m) {
                    const uint32_t vi = it, ki = it + 1;
                    uint8_t* v = stage_wait(vi);
                    clean(v, g.j0 + m);
                    const bool more = m + 1 < n;
                    mma_o(0, v, m == 0);
                    if (more) {
                        k = stage_wait(ki);
                        mma_s(0, 0, k);
                    } else {
                        commit(&o_full[0]);
                    }
                    mma_o(1, v, m == 0);
                    commit(&empty[vi % P::kStages]);
                    if (more) {
                        mma_s(1, 1, k);
                        commit(&empty[ki % P::kStages]);
                        if (m + 2 == n) commit(q_empty);
                    } else {
                        commit(&o_full[1]);
                    }
                    it += more ? 2 : 1;
                }
            } else {
                for (int i = 0; i < min(n, 2); ++i, ++it) {
                    mma_s(i, 0, stage_wait(it));
                    commit(&empty[it % P::kStages]);
                }
                if (n <= 2) commit(q_empty);
                for (int m = 0; m < n && ok; ++m) {
                    const int slot = m & 1;
                    uint8_t* v = stage_wait(it);
                    clean(v, g.j0 + m);
                    mma_o(slot, v, m < 2);
                    commit(&empty[it % P::kStages]);
                    ++it;
                    if (m + 2 < n) {
                        mma_s(slot, 0, stage_wait(it));
                        commit(&empty[it % P::kStages]);
                        ++it;
                        if (m + 3 == n) commit(q_empty);
                    } else {
                        commit(&o_full[slot]);
                    }
                }
            }
        }
        // the MMAs' last reads and commits before the CTA's memory goes
        for (uint32_t i = it > (uint32_t)P::kStages ? it - P::kStages : 0; i < it; ++i)
            if (!pa_wait(&empty[i % P::kStages], (i / P::kStages) & 1, kPaExitNs)) ok = false;
      }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPaSoftmaxRegs));
        sched.start(blockIdx.x, gridDim.x, lane);
        // ---------------------------------------------------------------- softmax and epilogue
        const int slot = warp >> 2, quarter = warp & 3;
        const int r = quarter * 32 + lane;                             // this thread's row and TMEM lane
        const int wtid = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_t = tmem + lanes + slot * kPaStep, o_t = tmem + lanes + 256 + slot * HD;
        const float c = a.scale_log2;
        uint32_t n_s = 0, n_o = 0;
        // A wait that gave up only clears ok: the warps stay in step with each other, since they meet at barriers.
        while (sched.next(g)) {
            const int tile = g.dual ? slot : 0;
            const int used = g.rows_used[tile];
            const int tok = r / a.grp;
            const int pos = g.pos0 + tile * a.tokens + tok;
            const int limit = r < used ? min(pos + 1, g.end) : 0;      // positions this row sees
            const bool idle = quarter * 32 >= used;                    // no row of this warp is used
            float m = -INFINITY, l = 0.f;
            const int n = g.j1 - g.j0;
            const int mine = g.dual ? n : (n + 1 - slot) / 2;
            for (int i = 0; i < mine; ++i) {
                if (ok && !pa_wait(&s_full[slot], n_s & 1)) ok = false;
                ++n_s;
                tc_fence_after();
                if (!idle) {
                    const int step = g.j0 + (g.dual ? i : 2 * i + slot);
                    float x[kPaStep];
#pragma unroll
                    for (int q = 0; q < 4; ++q) tc_ld32(s_t + q * 32, *reinterpret_cast<float(*)[32]>(x + q * 32));
                    tc_wait_ld();
                    const int see = limit - step * kPaStep;
                    if (__any_sync(0xffffffffu, see < kPaStep)) {
#pragma unroll
                        for (int q = 0; q < kPaStep; ++q) x[q] = q < see ? x[q] : -INFINITY;
                    }
                    float t0 = x[0], t1 = x[1], t2 = x[2], t3 = x[3];
#pragma unroll
                    for (int q = 4; q < kPaStep; q += 4) {
                        t0 = fmaxf(t0, x[q]);
                        t1 = fmaxf(t1, x[q + 1]);
                        t2 = fmaxf(t2, x[q + 2]);
                        t3 = fmaxf(t3, x[q + 3]);
                    }
                    const float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
                    const bool grow = (top - m) * c > kPaSlack;        // false for a row that has seen nothing yet
                    if (__any_sync(0xffffffffu, grow)) {
                        const float f = grow ? pa_weight(m, top, c) : 1.f;
                        if (grow) m = top;
                        l *= f;
                        if (i > 0) {
#pragma unroll 1
                            for (int q = 0; q < HD; q += 16) {
                                float o[16];
                                uint32_t w[16];
                                tc_ld16(o_t + q, o);
                                tc_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * f);
                                tc_st16(o_t + q, w);
                            }
                            tc_wait_st();
                        }
                    }
                    const float mc = m == -INFINITY ? 0.f : m * c;
                    float l0 = 0.f, l1 = 0.f, l2 = 0.f, l3 = 0.f;
#pragma unroll
                    for (int part = 0; part < 4; ++part) {
                        uint32_t pk[16];
#pragma unroll
                        for (int q = 0; q < 32; q += 4) {
                            const float* y = x + part * 32 + q;
                            const float e0 = ex2(fmaf(y[0], c, -mc)), e1 = ex2(fmaf(y[1], c, -mc));
                            const float e2 = ex2(fmaf(y[2], c, -mc)), e3 = ex2(fmaf(y[3], c, -mc));
                            l0 += e0;
                            l1 += e1;
                            l2 += e2;
                            l3 += e3;
                            pk[q / 2] = pack2<C>(e0, e1);
                            pk[q / 2 + 1] = pack2<C>(e2, e3);
                        }
                        tc_st16(s_t + part * 16, pk);
                    }
                    l += (l0 + l1) + (l2 + l3);
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[slot]);
            }
            if (mine > 0) {
                if (ok && !pa_wait(&o_full[slot], n_o & 1)) ok = false;
                ++n_o;
                tc_fence_after();
            }
            // The accumulator, 32 columns at a time. In a one-tile item slot 1's steps of the same rows join slot 0's
            // through the free Q tile, half of the columns at a time.
            float4* buf = reinterpret_cast<float4*>(q_s + P::kTile) + r;
            const bool whole = g.c0 == g.c1;                           // the whole item is this CTA's
            const int row = g.row0 + tile * a.tokens + tok;
            const bool live = r < used && row < a.b.rows;
            C* dst = static_cast<C*>(a.out) + ((size_t)row * a.hq + g.h * a.grp + (r - tok * a.grp)) * HD;
            // this CTA's part of a shared item: [column quad][used row], then (m, l) per row
            auto part = [&](int cta) { return a.parts + ((size_t)(cta * 2 + (cta == g.c0 ? 1 : 0)) * 2 + tile) * P::kPart; };
            float4* pdst = reinterpret_cast<float4*>(part(blockIdx.x)) + r;
            const bool joins = !g.dual && n > 1;                       // slot 1 had steps
            if (!g.dual && slot == 1) ml_s[r] = make_float2(m, l);
            float f0 = 1.f, f1 = 0.f, inv = 0.f;
#pragma unroll 1
            for (int ch = 0; ch < HD / 32; ++ch) {
                constexpr int kHalf = HD / 64;                         // chunks of a half
                const bool sends = !g.dual && slot == 1;
                if (!g.dual && slot == 0 && ch % kHalf == 0) named_bar_sync(1, 256);
                if (slot == 0 && joins && ch == 0) {
                    const float2 w = ml_s[r];
                    const float top = fmaxf(m, w.x);
                    if (top > -INFINITY) {
                        f0 = pa_weight(m, top, c);
                        f1 = pa_weight(w.x, top, c);
                    }
                    l = l * f0 + w.y * f1;
                    m = top;
                }
                if (ch == 0) inv = 1.f / l;
                float o[32];
                if (mine > 0) {
                    tc_ld32(o_t + ch * 32, o);
                    tc_wait_ld();
                    if (sends) {
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            buf[(ch % kHalf * 8 + q) * kPaRows] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
                    } else {
                        if (joins) {
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                const float4 w = buf[(ch % kHalf * 8 + q) * kPaRows];
                                o[4 * q] = o[4 * q] * f0 + w.x * f1;
                                o[4 * q + 1] = o[4 * q + 1] * f0 + w.y * f1;
                                o[4 * q + 2] = o[4 * q + 2] * f0 + w.z * f1;
                                o[4 * q + 3] = o[4 * q + 3] * f0 + w.w * f1;
                            }
                        }
                        if (whole && live) {
#pragma unroll
                            for (int q = 0; q < 32; q += 8) {
                                uint4 w;
                                w.x = pack2<C>(o[q] * inv, o[q + 1] * inv);
                                w.y = pack2<C>(o[q + 2] * inv, o[q + 3] * inv);
                                w.z = pack2<C>(o[q + 4] * inv, o[q + 5] * inv);
                                w.w = pack2<C>(o[q + 6] * inv, o[q + 7] * inv);
                                *reinterpret_cast<uint4*>(dst + ch * 32 + q) = l == 0.f ? make_uint4(0, 0, 0, 0) : w;
                            }
                        } else if (!whole && r < used) {
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                __stcg(pdst + (ch * 8 + q) * used, make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]));
                        }
                    }
                }
                if (sends && ch % kHalf == kHalf - 1) named_bar_sync(1, 256);
                if (!g.dual && ch % kHalf == kHalf - 1) named_bar_sync(2, 256);
            }
            tc_fence_before();
            fence_proxy_async_smem();                                  // the merge buffer is a TMA destination again
            __syncwarp();
            if (lane == 0) {
                if (mine > 0) mbar_arrive(&o_empty[slot]);
                mbar_arrive(q_empty);
            }
            if (whole || (!g.dual && slot == 1)) continue;
            if (r < used) __stcg(reinterpret_cast<float2*>(part(blockIdx.x) + (size_t)kPaRows * HD * 4) + r, make_float2(m, l));
            __threadfence();
            named_bar_sync(3 + slot, 128);
            if (wtid == 0) {
                uint32_t* cnt = a.counters + g.c0 * 2 + tile;
                const bool last = atomicAdd(cnt, 1u) == (uint32_t)(g.c1 - g.c0);
                if (last) *cnt = 0u;                                   // zero at rest
                __threadfence();
                last_flag[slot] = last;
            }
            named_bar_sync(3 + slot, 128);
            const bool last = last_flag[slot] != 0u;
            named_bar_sync(3 + slot, 128);                             // read before the next item writes it
            if (!last) continue;
            __threadfence();
            for (int e = wtid; e < used * (HD / 4); e += 128) {
                const int er = e % used, q = e / used;
                float top = -INFINITY;
                for (int k = g.c0; k <= g.c1; ++k)
                    top = fmaxf(top, __ldcg(reinterpret_cast<const float2*>(part(k) + (size_t)kPaRows * HD * 4) + er).x);
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                float sum = 0.f;
#pragma unroll 4
                for (int k = g.c0; k <= g.c1; ++k) {
                    const uint8_t* pt = part(k);
                    const float2 w = __ldcg(reinterpret_cast<const float2*>(pt + (size_t)kPaRows * HD * 4) + er);
                    const float4 y = __ldcg(reinterpret_cast<const float4*>(pt) + e);
                    const float f = pa_weight(w.x, top, c);
                    sum += w.y * f;
                    acc.x += y.x * f;
                    acc.y += y.y * f;
                    acc.z += y.z * f;
                    acc.w += y.w * f;
                }
                const int et = er / a.grp, erow = g.row0 + tile * a.tokens + et;
                if (erow < a.b.rows) {
                    const float einv = 1.f / sum;
                    uint2 w = make_uint2(pack2<C>(acc.x * einv, acc.y * einv), pack2<C>(acc.z * einv, acc.w * einv));
                    if (sum == 0.f) w = make_uint2(0, 0);
                    *reinterpret_cast<uint2*>(static_cast<C*>(a.out) +
                                              ((size_t)erow * a.hq + g.h * a.grp + (er - et * a.grp)) * HD + q * 4) = w;
                }
            }
        }
    }
    if (!ok && lane == 0) atomicOr(a.status, kStatusPipeTimeout);
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// ------------------------------------------------------------------------------ host
static CUtensorMapDataType pa_type(int dtype)
{
    return dtype == EXL3_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// Pages as (head_dim, page_size, hkv, num_pages): a box is 64 columns of up to 128 positions of one page and head.
static bool pa_map_pages(PFN_cuTensorMapEncodeTiled_v12000 encode, CUtensorMap* map, const void* base, const exl3_paged_desc& b)
{
    const cuuint64_t dims[4] = {(cuuint64_t)b.head_dim, (cuuint64_t)b.page_size, (cuuint64_t)b.hkv, (cuuint64_t)b.num_pages};
    const cuuint64_t row = (cuuint64_t)b.head_dim * 2;
    const cuuint64_t strides[3] = {row, row * b.page_size, row * b.page_size * b.hkv};
    const cuuint32_t box[4] = {64, (cuuint32_t)(b.page_size < kPaStep ? b.page_size : kPaStep), 1, 1};
    const cuuint32_t one[4] = {1, 1, 1, 1};
    return encode(map, pa_type(b.dtype), 4, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
           CUDA_SUCCESS;
}

// Queries as (head_dim, hq, rows): a box is 64 columns of one kv head's group for a tile's tokens, which lands as the
// tile's packed rows.
static bool pa_map_q(PFN_cuTensorMapEncodeTiled_v12000 encode, CUtensorMap* map, const void* base, long long stride,
                     const exl3_paged_desc& b, int hq, int grp, int tokens)
{
    const cuuint64_t dims[3] = {(cuuint64_t)b.head_dim, (cuuint64_t)hq, (cuuint64_t)b.rows};
    const cuuint64_t strides[2] = {(cuuint64_t)b.head_dim * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)grp, (cuuint32_t)tokens};
    const cuuint32_t one[3] = {1, 1, 1};
    return encode(map, pa_type(b.dtype), 3, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
           CUDA_SUCCESS;
}

static int check_attn(const exl3_paged_desc* b, int hq)
{
    if (int e = exl3_check_paged(b)) return e;
    if (hq < 1 || hq % b->hkv || hq / b->hkv > kPaRows) return EXL3_E_SHAPE;
    return EXL3_OK;
}

static int attn_ctas() { return std::min(device_sm_count(), EXL3_PAGED_HEADER_BYTES / 8); }

template <int HD>
static size_t attn_bytes() { return EXL3_PAGED_HEADER_BYTES + (size_t)attn_ctas() * 4 * PaShape<HD>::kPart; }

template <typename C, int HD>
static int launch_attn(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const PaArgs& a, cudaStream_t s)
{
    static bool attr_set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return EXL3_E_CUDA;
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        if (cudaFuncSetAttribute(paged_attn_kernel<C, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, PaShape<HD>::kSmem) !=
            cudaSuccess)
            return EXL3_E_CUDA;
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    return launch_pdl(paged_attn_kernel<C, HD>, dim3(attn_ctas()), dim3(kPaThreads), PaShape<HD>::kSmem, s, qm, km, vm, a);
}

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_paged_attn_workspace(const exl3_paged_desc* batch, int hq, size_t* bytes)
{
    if (!bytes) return EXL3_E_NULL;
    if (int e = check_attn(batch, hq)) return e;
    *bytes = batch->head_dim == 128 ? attn_bytes<128>() : attn_bytes<64>();
    return EXL3_OK;
}

extern "C" int exl3_paged_attn(const exl3_paged_desc* batch, const void* q, long long q_stride, int hq, float scale,
                               void* out, void* workspace, size_t workspace_bytes, uint32_t* status, void* stream)
{
    if (int e = check_attn(batch, hq)) return e;
    if (batch->rows == 0) return EXL3_OK;
    if (!q || !out || !status || !workspace) return EXL3_E_NULL;
    if (q_stride < (long long)hq * batch->head_dim || !(scale > 0.f)) return EXL3_E_SHAPE;
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(status, 4) || !aligned(workspace, 16) || q_stride % 8)
        return EXL3_E_ALIGN;
    if (int e = check_device()) return e;
    if (workspace_bytes < (batch->head_dim == 128 ? attn_bytes<128>() : attn_bytes<64>())) return EXL3_E_WORKSPACE;
    auto encode = exl3_get_tensormap_encoder();
    if (!encode) return EXL3_E_CUDA;
    PaArgs a{};
    a.b = *batch;
    a.out = out;
    a.counters = static_cast<uint32_t*>(workspace);
    a.parts = static_cast<uint8_t*>(workspace) + EXL3_PAGED_HEADER_BYTES;
    a.status = status;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.hq = hq;
    a.grp = hq / batch->hkv;
    a.tokens = kPaRows / a.grp;
    CUtensorMap qm, km, vm;
    if (!pa_map_q(encode, &qm, q, q_stride, *batch, hq, a.grp, a.tokens) || !pa_map_pages(encode, &km, batch->k_pages, *batch) ||
        !pa_map_pages(encode, &vm, batch->v_pages, *batch))
        return EXL3_E_CUDA;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (batch->dtype == EXL3_F16)
        return batch->head_dim == 128 ? launch_attn<__half, 128>(qm, km, vm, a, s) : launch_attn<__half, 64>(qm, km, vm, a, s);
    return batch->head_dim == 128 ? launch_attn<__nv_bfloat16, 128>(qm, km, vm, a, s)
                                  : launch_attn<__nv_bfloat16, 64>(qm, km, vm, a, s);
}
