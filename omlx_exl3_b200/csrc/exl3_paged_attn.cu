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
// Roles of a CTA (one per SM, persistent): two softmax warpgroups, one warp that loads with TMA, two that issue the
// MMAs, one that cleans a tile's end. There are two slots (S, P and O of their own, a warpgroup and an issuing warp each). In a
// two-tile item slot = tile; in a one-tile item the slots take alternate steps of the same rows and are merged at its
// end. Within a slot a step goes by halves of 64 positions: while the softmax works on one half of S, the tensor core does
// the other half's P V and then its S of the next step, in that order from one warp, so S may overwrite P. The
// accumulator is rescaled only when a row's maximum grows by more than 2^8 (P <= 256 is exact enough in either type, and
// the sum is fp32 of the unrounded p), by the softmax thread itself, once the P V issued last is complete.
//
// Bound by the softmax (ex2: 128 x 128 of a tile step take 1024 cycles of the special function unit, as long as its 2 x 128^3
// MMAs) and by what lies between (both are busy 54 % of the time): 4096 rows over 8192 positions of 40 / 8 heads of 128 in bf16 take
// 486 us in short runs, 1.06 PFLOP/s, 0.65 of a measured library GEMM's burst, and 556 us in a long loop, where the power cap lowers
// the clocks: 0.93 PFLOP/s, 0.68 of its sustained rate; an exponent polynomial on the FMA pipe for a quarter of the ex2 (553 against 507
// us at that stage), four softmax warpgroups with a row's halves in two threads (589), and whole steps with an enforced
// alternation of the slots' MMAs (497) were measured slower.
//
// Split: exl3_paged_sched.cuh; the parts of cut items are merged by exl3_paged_merge.cu.
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
#include "exl3_paged_sched.cuh"
#include "exl3_tc.cuh"

namespace exl3 {

constexpr int kPaThreads = 384;                       // two softmax warpgroups; one with the load, clean and MMA warps
constexpr int kPaBarBytes = 512;
constexpr uint64_t kPaExitNs = 100000000ull;          // wait for a CTA's own copies and MMAs before it exits

template <int HD>
struct PaShape {
    static constexpr int kPanels = HD / 64;           // 128-byte swizzled panels of a tile
    static constexpr int kTile = kPaRows * HD * 2;    // bytes of a Q, K or V tile
    static constexpr int kPanel = kPaRows * 128;
    static constexpr int kStages = HD == 128 ? 5 : 8;
    static constexpr int kMl = kPaRows * 8;           // slot 1's (m, l) for the merge of a one-tile item
    static constexpr int kSmem = 1024 + 2 * kTile + kStages * kTile + kMl + kPaBarBytes;
    static_assert(kSmem <= 227 * 1024, "shared memory");
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

// One lane of the (converged) warp: 1 in it, 0 in the others.
__device__ __forceinline__ uint32_t elect_one()
{
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r;
}

// A value that is the same in all lanes, known to the compiler as such.
__device__ __forceinline__ uint64_t uniform64(uint64_t x)
{
    const uint32_t lo = __shfl_sync(0xffffffffu, (uint32_t)x, 0), hi = __shfl_sync(0xffffffffu, (uint32_t)(x >> 32), 0);
    return ((uint64_t)hi << 32) | lo;
}

// tcgen05.mma / commit issued by the lanes with go != 0 (one of the warp).
__device__ __forceinline__ void tc_mma_if(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t go)
{
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(go)
        : "memory");
}

__device__ __forceinline__ void tc_mma_ts_if(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t go)
{
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(go)
        : "memory");
}

__device__ __forceinline__ void tc_commit_if(uint64_t* bar, uint32_t go)
{
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_addr(bar)),
        "r"(go)
        : "memory");
}

__device__ __forceinline__ void mbar_arrive_if(uint64_t* bar, uint32_t go)
{
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q mbarrier.arrive.shared::cta.b64 _, [%0];\n}\n" ::"r"(smem_addr(bar)),
                 "r"(go)
                 : "memory");
}

// Bounded wait of a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns = 2000000000ull)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, limit_ns));
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
    uint64_t* s_full = q_empty + 1;                   // [2][2] half of S of the slot is complete (and that half's P V before it)
    uint64_t* p_full = s_full + 4;                    // [2][2] half of P of the slot is written
    uint64_t* pv_done = p_full + 4;                   // [2] P V of the first half of the slot's step is complete
    uint64_t* v_dirty = pv_done + 2;                   // both issuing warps have taken the item's last V tile, which reaches past the end
    uint64_t* v_clean = v_dirty + 1;                  // it is zero there
    uint64_t* o_full = v_clean + 1;                   // [2] the slot's accumulator is complete
    uint64_t* o_empty = o_full + 2;                   // [2] it has been read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_empty + 2);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < P::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 2);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 2 + 8);
        mbar_init(v_dirty, 2);
        mbar_init(v_clean, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[2 * i], 1);
            mbar_init(&s_full[2 * i + 1], 1);
            mbar_init(&pv_done[i], 1);
            mbar_init(&p_full[2 * i], 4);
            mbar_init(&p_full[2 * i + 1], 4);
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
    // What this kernel reads is complete once it may go on; the kernel for few rows reads the same and begins behind this
    // trigger on SMs that have no tiles (left).
    pdl_wait();
    pdl_trigger();

    PaSched sched(a);
    PaSeg g{};
    bool ok = true;

    // Tiles of the segment: tokens per tile, the second tile's only where the item has more than one tile's.
    const int tokens = by_grp(a, kPaRows);
    struct Item { int row0, pos0, ntok[2]; bool dual; };
    auto item_of = [&](const PaSeg& g) {
        const int tok0 = by_grp(a, g.p0), ntok = min(g.rows - tok0, 2 * tokens);
        Item i;
        i.row0 = g.start + tok0;
        i.pos0 = g.ctx + tok0;
        i.dual = ntok > tokens;
        i.ntok[0] = min(ntok, tokens);
        i.ntok[1] = ntok - i.ntok[0];
        return i;
    };
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
            const Item im = item_of(g);
            if (lane == 0) {
                if ((long long)im.pos0 + im.ntok[0] + im.ntok[1] > sched.cap) atomicOr(a.status, kStatusPagedRange);
                const int tiles = im.dual ? 2 : 1;
                mbar_arrive_expect_tx(q_full, tiles * P::kPanels * tokens * a.grp * 128);
                for (int i = 0; i < tiles; ++i)
                    for (int p = 0; p < P::kPanels; ++p)
                        tma_load_3d(q_s + i * P::kTile + p * P::kPanel, &qmap, p * 64, g.h * a.grp, im.row0 + i * tokens,
                                    q_full);
            }
            __syncwarp();
            ++n_seg;
            const int n = g.j1 - g.j0, ahead = im.dual ? 1 : 2;
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
        if (lane == 0) pa_record(a, sched.bad, n_seg > 0, g, n_seg > 0 ? min(2 * tokens, g.rows - by_grp(a, g.p0)) * a.grp : 0, tokens * a.grp);
        // nothing of this CTA may still be landing when it exits
        for (uint32_t i = it > (uint32_t)P::kStages ? it - P::kStages : 0; i < it; ++i)
            if (!pa_wait(&full[i % P::kStages], (i / P::kStages) & 1, kPaExitNs)) ok = false;
        if (n_seg > 0 && !pa_wait(q_full, (n_seg - 1) & 1, kPaExitNs)) ok = false;
    } else if (warp == 10) {
        sched.start(blockIdx.x, gridDim.x, lane);
        // ---------------------------------------------------------------- V behind the sequence's end becomes zero
        uint32_t it = 0, n = 0;
        while (ok && sched.next(g)) {
            it += 2 * (g.j1 - g.j0);                                   // the segment's last tile is its last V
            const int valid = g.end - (g.j1 - 1) * kPaStep;
            if (valid >= kPaStep) continue;
            if (!pa_wait(v_dirty, n++ & 1)) { ok = false; break; }
            uint8_t* v = kv_s + ((it - 1) % P::kStages) * P::kTile;
            for (int i = max(valid, 0) * 8 + lane; i < kPaStep * 8; i += 32)
#pragma unroll
                for (int p = 0; p < P::kPanels; ++p)
                    *reinterpret_cast<uint4*>(v + p * P::kPanel + i * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_clean);
        }
    } else if (warp > 8) {
        sched.start(blockIdx.x, gridDim.x, lane);
        // ---------------------------------------------------------------- MMAs: warp 9 for slot 0, warp 11 for slot 1
        // Between the MMAs of a step lie waits and commits of some hundred cycles in the issuing warp; with a warp per slot
        // they pass while the other slot's MMAs run. Each whole warp runs this and one elected lane issues, so that operands
        // come from uniform registers. Both warps see every tile of the ring land and release it (the tiles of the other
        // slot at once), so neither can fall a round behind on the ring. Nor on a tile's cleaning: it begins when both have asked
        // for it, so a warp without a step in a short item is past that item's v_clean before the next item's can complete.
        constexpr uint32_t idesc_s = pa_idesc<C>(kPaStep / 2, false), idesc_o = pa_idesc<C>(HD, true);
        const int slot = warp == 11;
        const uint32_t leader = elect_one();
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint32_t s_tm = tm + slot * kPaStep, o_tm = tm + 256 + slot * HD;
        const uint64_t q_desc = uniform64(smem_desc_sw128(q_s)), k_desc = uniform64(smem_desc_sw128(kv_s)),
                       v_desc = uniform64(pa_desc_v(kv_s, P::kPanel));
        uint32_t n_seg = 0, n_clean = 0, st = 0, ring = 0, n_p = 0, n_o = 0;   // st: stage of the ring, ring: its round
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (ok && !pa_wait(bar, parity)) ok = false;
        };
        auto commit = [&](uint64_t* bar) { tc_commit_if(bar, leader & (uint32_t)ok); };
        auto take = [&]() {                                            // the stage of the ring's next tile, once it has landed
            const uint32_t i = st;
            wait(&full[i], ring & 1);
            if (++st == (uint32_t)P::kStages) {
                st = 0;
                ++ring;
            }
            return i;
        };
        auto release = [&](uint32_t i, bool mine) {
            if (mine) commit(&empty[i]);
            else if (ok && lane == 0) mbar_arrive(&empty[i]);
        };
        // S of 64 of a step's positions
        auto mma_s = [&](int tile, uint32_t stage, int half) {
            const uint64_t qd = q_desc + tile * (P::kTile >> 4), kd = k_desc + stage * (P::kTile >> 4) + half * (8192 >> 4);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                const int off = ((kk / 4) * P::kPanel + (kk % 4) * 32) >> 4;
                tc_mma_if(s_tm + half * 64, qd + off, kd + off, idesc_s, kk > 0, leader & (uint32_t)ok);
            }
            commit(&s_full[2 * slot + half]);
        };
        // P V of half of a step; `first`: the slot's first of the item
        auto mma_o = [&](uint32_t stage, int half, bool first) {
            if (first && half == 0) {
                if (n_o > 0) wait(&o_empty[slot], (n_o - 1) & 1);
                ++n_o;
            }
            wait(&p_full[2 * slot + half], n_p & 1);
            tc_fence_after();
            const uint64_t vd = v_desc + stage * (P::kTile >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                tc_mma_ts_if(o_tm, s_tm + half * 64 + kk * 8, vd + (4 * half + kk) * (2048 >> 4), idesc_o,
                             (first && half == 0 && kk == 0) ? 0u : 1u, leader & (uint32_t)ok);
            if (half == 0) commit(&pv_done[slot]);
            else ++n_p;
        };
        while (ok && sched.next(g)) {
            wait(q_full, n_seg & 1);
            ++n_seg;
            const int n = __shfl_sync(0xffffffffu, g.j1 - g.j0, 0);
            const bool dirty = __shfl_sync(0xffffffffu, g.j1 * kPaStep > g.end, 0);   // the last V tile reaches past the end
            const bool dual = __shfl_sync(0xffffffffu, item_of(g).dual, 0);
            const int ahead = dual ? 1 : 2;                            // K tiles before the first V
            for (int i = 0; i < min(n, ahead); ++i) {
                const uint32_t k = take();
                const bool mine = dual || i == slot;
                if (mine) {
                    tc_fence_after();
                    mma_s(dual ? slot : 0, k, 0);
                    mma_s(dual ? slot : 0, k, 1);
                }
                release(k, mine);
            }
            if (n <= ahead) commit(q_empty);
            for (int m = 0; m < n; ++m) {
                const bool mine = dual || (m & 1) == slot, more = m + ahead < n;
                const uint32_t v = take();
                uint32_t k = 0;
                if (more) k = take();
                if (m + 1 == n && dirty) {                             // warp 10 cleans it, once per such item
                    if (lane == 0) mbar_arrive(v_dirty);
                    wait(v_clean, n_clean++ & 1);
                }
                if (mine) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        mma_o(v, half, m < ahead);
                        if (more) mma_s(dual ? slot : 0, k, half);
                    }
                    if (!more) commit(&o_full[slot]);
                }
                release(v, mine);
                if (more) release(k, mine);
                if (m + 1 + ahead == n) commit(q_empty);
            }
        }
        // the MMAs' last reads and commits before the CTA's memory goes
        const uint32_t taken = ring * P::kStages + st;
        for (uint32_t i = taken > (uint32_t)P::kStages ? taken - P::kStages : 0; i < taken; ++i)
            if (!pa_wait(&empty[i % P::kStages], (i / P::kStages) & 1, kPaExitNs)) ok = false;
    } else {
        sched.start(blockIdx.x, gridDim.x, lane);
        // ---------------------------------------------------------------- softmax and epilogue
        const int slot = warp >> 2, quarter = warp & 3;
        const int r = quarter * 32 + lane;                             // this thread's row and TMEM lane
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_t = tmem + lanes + slot * kPaStep, o_t = tmem + lanes + 256 + slot * HD;
        const float c = a.scale_log2;
        uint32_t n_s = 0, n_o = 0;
        const uint32_t leader = elect_one();
        // A wait that gave up only clears ok: the warps stay in step with each other, since they meet at barriers.
        while (sched.next(g)) {
            const Item im = item_of(g);
            const bool dual = im.dual;
            const int tile = dual ? slot : 0;
            const int used = im.ntok[tile] * a.grp;
            const int tok = by_grp(a, r);
            const int pos = im.pos0 + tile * tokens + tok;
            const int limit = r < used ? min(pos + 1, g.end) : 0x7fffffff;    // positions this row sees; unused rows: any
            const bool idle = quarter * 32 >= used;                    // no row of this warp is used
            float m = -INFINITY, l = 0.f;
            const int n = g.j1 - g.j0;
            const int mine = dual ? n : (n + 1 - slot) / 2;
            for (int i = 0; i < mine; ++i) {
                const int step = g.j0 + (dual ? i : 2 * i + slot);
                // 64 positions at a time: while one half of S is worked on here, the tensor core does the other half's
                // P V and its S of the next step, so neither waits for the other's whole step
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    if (ok && !pa_wait(&s_full[2 * slot + half], n_s & 1)) ok = false;
                    tc_fence_after();
                    if (!idle) {
                        const uint32_t x_t = s_t + half * 64;
                        float x[64];
                        tm_ld32(x_t, x);
                        tm_ld32(x_t + 32, x + 32);
                        tc_wait_ld();
                        const int see = limit - step * kPaStep - half * 64;
                        if (__any_sync(0xffffffffu, see < 64)) {
#pragma unroll
                            for (int q = 0; q < 64; ++q) x[q] = q < see ? x[q] : -INFINITY;
                        }
                        float t0 = x[0], t1 = x[1], t2 = x[2], t3 = x[3];
#pragma unroll
                        for (int q = 4; q + 8 <= 64; q += 8) {
                            t0 = max3(t0, x[q], x[q + 1]);
                            t1 = max3(t1, x[q + 2], x[q + 3]);
                            t2 = max3(t2, x[q + 4], x[q + 5]);
                            t3 = max3(t3, x[q + 6], x[q + 7]);
                        }
                        t0 = max3(t0, x[60], x[61]);
                        t1 = max3(t1, x[62], x[63]);
                        const float top = fmaxf(max3(t0, t1, t2), t3);
                        const bool grow = (top - m) * c > kPaSlack;    // false for a row that has seen nothing yet
                        if (__any_sync(0xffffffffu, grow)) {
                            const float f = grow ? pa_weight(m, top, c) : 1.f;
                            if (grow) m = top;
                            l *= f;
                            if (i > 0 || half > 0) {
                                // the P V issued last has to be complete: the other half's S follows it, or its own commit
                                if (ok && !pa_wait(half ? &pv_done[slot] : &s_full[2 * slot + 1], n_s & 1)) ok = false;
                                tc_fence_after();
#pragma unroll 1
                                for (int q = 0; q < HD; q += 16) {
                                    float o[16];
                                    uint32_t w[16];
                                    tm_ld16(o_t + q, o);
                                    tc_wait_ld();
#pragma unroll
                                    for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * f);
                                    tc_st16(o_t + q, w);
                                }
                                tc_wait_st();
                            }
                        }
                        const float mc = m == -INFINITY ? 0.f : m * c;
                        const uint64_t c2 = f2(c, c), mc2 = f2(-mc, -mc);
                        uint64_t l01 = f2(0.f, 0.f), l23 = l01;
#pragma unroll
                        for (int part = 0; part < 2; ++part) {
                            uint32_t pk[16];
#pragma unroll
                            for (int q = 0; q < 32; q += 4) {
                                const float* y = x + part * 32 + q;
                                float e0, e1, e2, e3;
                                f2_get(f2_fma(f2(y[0], y[1]), c2, mc2), e0, e1);
                                f2_get(f2_fma(f2(y[2], y[3]), c2, mc2), e2, e3);
                                e0 = ex2(e0);
                                e1 = ex2(e1);
                                e2 = ex2(e2);
                                e3 = ex2(e3);
                                l01 = f2_add(l01, f2(e0, e1));
                                l23 = f2_add(l23, f2(e2, e3));
                                pk[q / 2] = pack2<C>(e0, e1);
                                pk[q / 2 + 1] = pack2<C>(e2, e3);
                            }
                            tc_st16(x_t + part * 16, pk);
                        }
                        float l0, l1, l2, l3;
                        f2_get(l01, l0, l1);
                        f2_get(l23, l2, l3);
                        l += (l0 + l1) + (l2 + l3);
                        tc_wait_st();
                    }
                    tc_fence_before();
                    __syncwarp();
                    mbar_arrive_if(&p_full[2 * slot + half], leader);
                }
                ++n_s;
            }
            if (mine > 0) {
                if (ok && !pa_wait(&o_full[slot], n_o & 1)) ok = false;
                ++n_o;
                tc_fence_after();
            }
            // The accumulator, 32 columns at a time. In a one-tile item slot 1's steps of the same rows join slot 0's
            // through the free Q tile, half of the columns at a time.
            float4* buf = reinterpret_cast<float4*>(q_s + P::kTile) + r;
            const bool whole = g.j0 == 0 && g.j1 == g.units;           // the whole item is this CTA's
            const int row = im.row0 + tile * tokens + tok;
            const bool live = r < used && row < a.b.rows;
            C* dst = static_cast<C*>(a.out) + ((size_t)row * a.hq + g.h * a.grp + (r - tok * a.grp)) * HD;
            uint8_t* part = pa_part<HD, kPaRows, 2>(a.parts, g.c0, blockIdx.x, tile);
            float4* pdst = reinterpret_cast<float4*>(part) + r;
            const bool joins = !dual && n > 1;                       // slot 1 had steps
            if (!dual && slot == 1) ml_s[r] = make_float2(m, l);
            float f0 = 1.f, f1 = 0.f, inv = 0.f;
#pragma unroll 1
            for (int ch = 0; ch < HD / 32; ++ch) {
                constexpr int kHalf = HD / 64;                         // chunks of a half
                const bool sends = !dual && slot == 1;
                if (!dual && slot == 0 && ch % kHalf == 0) named_bar_sync(1, 256);
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
                    tm_ld32(o_t + ch * 32, o);
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
                if (!dual && ch % kHalf == kHalf - 1) named_bar_sync(2, 256);
            }
            tc_fence_before();
            fence_proxy_async_smem();                                  // the merge buffer is a TMA destination again
            __syncwarp();
            if (lane == 0) {
                if (mine > 0) mbar_arrive(&o_empty[slot]);
                mbar_arrive(q_empty);
            }
            if (whole || (!dual && slot == 1)) continue;
            if (r < used) __stcg(reinterpret_cast<float2*>(part + PaPart<HD, kPaRows>::kMl) + r, make_float2(m, l));
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
    if (hq < 1 || hq % b->hkv || hq / b->hkv > kPaRows || (long long)b->rows * hq > 0x7fffffffll) return EXL3_E_SHAPE;
    return EXL3_OK;
}

static int attn_ctas() { return device_sm_count(); }

// Workspace: the two kernels' items, the tiles' parts, the few rows' parts.
struct AttnSpace {
    size_t few_items, tile_parts, few_parts, bytes;
};

template <int HD>
static AttnSpace attn_space()
{
    const size_t n = attn_ctas();
    AttnSpace w;
    w.few_items = n * sizeof(PaItem);
    w.tile_parts = (2 * n * sizeof(PaItem) + 255) / 256 * 256;
    w.few_parts = w.tile_parts + n * 4 * PaPart<HD, kPaRows>::kBytes;
    w.bytes = w.few_parts + n * 2 * PaPart<HD, kPaFew>::kBytes;
    return w;
}

static AttnSpace attn_space(const exl3_paged_desc& b) { return b.head_dim == 128 ? attn_space<128>() : attn_space<64>(); }

template <typename C, int HD>
static int launch_tiles(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const PaArgs& a, cudaStream_t s)
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

int pa_launch_tiles(const PaArgs& args, cudaStream_t s)
{
    PaArgs a = args;
    const int tokens = kPaRows / a.grp;
    a.span = 2 * tokens * a.grp;
    a.item = 2;
    auto encode = exl3_get_tensormap_encoder();
    if (!encode) return EXL3_E_CUDA;
    CUtensorMap qm, km, vm;
    if (!pa_map_q(encode, &qm, a.q, a.q_stride, a.b, a.hq, a.grp, tokens) || !pa_map_pages(encode, &km, a.b.k_pages, a.b) ||
        !pa_map_pages(encode, &vm, a.b.v_pages, a.b))
        return EXL3_E_CUDA;
    if (a.b.dtype == EXL3_F16)
        return a.b.head_dim == 128 ? launch_tiles<__half, 128>(qm, km, vm, a, s) : launch_tiles<__half, 64>(qm, km, vm, a, s);
    return a.b.head_dim == 128 ? launch_tiles<__nv_bfloat16, 128>(qm, km, vm, a, s)
                               : launch_tiles<__nv_bfloat16, 64>(qm, km, vm, a, s);
}

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_paged_attn_workspace(const exl3_paged_desc* batch, int hq, size_t* bytes)
{
    if (!bytes) return EXL3_E_NULL;
    if (int e = check_attn(batch, hq)) return e;
    if (int e = check_device()) return e;
    *bytes = attn_space(*batch).bytes;
    return EXL3_OK;
}

extern "C" int exl3_paged_attn(const exl3_paged_desc* batch, const void* q, long long q_stride, int hq, float scale,
                               int max_rows, void* out, void* workspace, size_t workspace_bytes, uint32_t* status, void* stream)
{
    if (int e = check_attn(batch, hq)) return e;
    if (batch->rows == 0) return EXL3_OK;
    if (!q || !out || !status || !workspace) return EXL3_E_NULL;
    if (q_stride < (long long)hq * batch->head_dim || !(scale > 0.f) || max_rows < 0) return EXL3_E_SHAPE;
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(status, 4) || !aligned(workspace, 256) || q_stride % 8)
        return EXL3_E_ALIGN;
    if (int e = check_device()) return e;
    const AttnSpace w = attn_space(*batch);
    if (workspace_bytes < w.bytes) return EXL3_E_WORKSPACE;
    PaArgs a{};
    a.b = *batch;
    a.q = q;
    a.q_stride = q_stride;
    a.out = out;
    a.status = status;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.hq = hq;
    a.grp = hq / batch->hkv;
    a.grp_magic = a.grp == 1 ? 0u : (uint32_t)(((1ull << 32) + a.grp - 1) / a.grp);
    if (!pa_list_fits(a, 8)) return EXL3_E_SHAPE;
    // Which kernel takes a sequence goes by its packed rows, which only the device knows: the host launches what they may need,
    // from their average and what it knows of the most. A 128-row tile costs the same however empty it is, and more at the
    // start, which counts while the SMs outnumber the pairs of a sequence and a kv head; 16 rows at a time read the keys and
    // values once per 16. Measured, us with sequences of up to 32 / up to 64 packed rows on the latter, each of 1 to 8 rows in
    // groups of 5 heads: 9 over 1000 positions of 8 kv heads 22.0 / 18.9, 16 26.8 / 21.9, 16 over 8000 41.4 / 44.3, 32 57.4 / 65.5, 64
    // 98.2 / 122.3, 128 127.4 / 142.4; of 4 kv heads 9 over 8000 26.8 / 23.0, 32 39.6 / 38.9, 64 61.6 / 71.6. So the limit is 64 where
    // the pairs of sequence and kv head are no more than the SMs. What also counts is the length, which the host does not know: at 128
    // pairs the rule takes the faster side over 1000 positions (by 5 us) and the slower one over 8000 (by 3). (Up to 16: 64 over
    // 8000 95.5, but 1 to 5 rows 42.7 / 39.4 at 16 / 32.) A batch with a row per sequence at most is taken for single tokens:
    // one launch, right whatever the rows are. Where both run, the kernel for few rows comes second and waits for the tiles at
    // its end only: 13 sequences of 1 to 777 rows 54.8 us, and 58.7 one after the other.
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long long packed = (long long)batch->rows * a.grp;
    const int hi = packed <= 32ll * batch->seqs && (long long)batch->seqs * batch->hkv <= attn_ctas() ? 64 : 32;
    const long long most = max_rows > 0 && max_rows < batch->rows ? (long long)max_rows * a.grp : packed;
    const bool few_only = most <= hi || (batch->rows <= batch->seqs && a.grp <= hi);
    const bool tiles_only = !few_only && (batch->seqs == 1 || a.grp > hi);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    PaArgs few = a, tiles = a;
    few.items = reinterpret_cast<PaItem*>(base + w.few_items);
    few.parts = base + w.few_parts;
    few.lo = 0;
    few.hi = few_only ? 0x7fffffff : hi;
    tiles.items = reinterpret_cast<PaItem*>(base);
    tiles.parts = base + w.tile_parts;
    tiles.lo = tiles_only ? 0 : hi;
    tiles.hi = 0x7fffffff;
    few.behind = !few_only;
    if (!few_only)
        if (int e = pa_launch_tiles(tiles, s)) return e;
    if (!tiles_only)
        if (int e = pa_launch_few(few, s)) return e;
    return pa_launch_merge(few_only ? nullptr : &tiles, tiles_only ? nullptr : &few, attn_ctas(), s);
}
