// Paged attention of few rows per sequence (a decoded token, a few drafts): up to 16 packed rows at a time, where the
// cache's bytes bound the time and a 128-row tensor-core tile would be empty. More rows are several items, the later ones
// reading the keys and values from L2.
//
// One CTA per SM, eight warps. A unit of 128 positions is a slice of 16 positions per warp: the slice's keys and
// values go to the warp's own ring of shared memory with 16-byte asynchronous copies (a warp's copies are two or four whole
// rows; small pages cost nothing, a slice never crosses one), several slices ahead and across items, so that the memory
// system always has a ring of loads in flight and no warp waits for another between items. Per slice, with positions as
// the MMA's 16-row side: S^T = K Q^T, p = exp2 in fp32 against a running maximum that is only moved when a score passes it
// by 2^8 (no cross-lane reduction on the usual path), P^T turned from accumulator to operand by movmatrix, and
// O^T += V^T P^T. At an item's end the warps' (m, l, O) are merged through shared memory in warp order.
//
// Bound by the cache's bytes where there are many: two sequences at 65,000 positions, 533 MB in 87 us (6.1 TB/s, 0.93 of a
// measured copy); 64 of 1 to 8192, 385 MB in 69 us (5.5 TB/s, 0.85); by launch and the chain of dependent loads (lengths, page,
// keys) for one short one (9.4 us at 4097 positions).
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "exl3_b200.h"
#include "exl3_common.cuh"
#include "exl3_host.h"
#include "exl3_paged.cuh"
#include "exl3_paged_sched.cuh"

namespace exl3 {

constexpr int kPfWarps = 8;
constexpr int kPfSlice = kPaStep / kPfWarps;          // 16 positions

template <int HD, int NQ>
struct PfShape {
    static constexpr int kRow = HD * 2;               // bytes of a position
    static constexpr int kSlot = 2 * kPfSlice * kRow; // a slice's K and V
    static constexpr int kDepth = HD == 128 ? 3 : 6;  // slices of a warp's ring: 192 KB in all
    static constexpr int kCols = NQ == 1 ? HD : 64;   // columns merged at a time: a quad for each of the CTA's threads
    static constexpr int kPad = kCols + 4;
    static constexpr int kMerge = kPfWarps * 8 * NQ * kPad * 4;
    static constexpr int kSmem = kPfWarps * kDepth * kSlot + kMerge;
    static_assert(kSmem + 2 * kPfWarps * 8 * NQ * 4 <= 227 * 1024, "shared memory");
};

template <typename C>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1)
{
    if constexpr (std::is_same<C, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// 16 bytes, or zeros where `bytes` is 0.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// NQ: n8 tiles of packed rows an item has (8 or 16 rows).
template <typename C, int HD, int NQ>
__global__ void __launch_bounds__(32 * kPfWarps, 1) paged_few_kernel(const __grid_constant__ PaArgs a)
{
    using S = PfShape<HD, NQ>;
    constexpr int kChunks = S::kRow / 16;             // 16-byte chunks of a position
    constexpr int kPer = 32 / kChunks;                // positions of one warp copy
    extern __shared__ __align__(128) uint8_t pf_sm[];
    __shared__ float wm[kPfWarps][8 * NQ], wl[kPfWarps][8 * NQ];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gid = lane >> 2, tig = lane & 3;
    const uint32_t ring = smem_addr(pf_sm) + warp * S::kDepth * S::kSlot;
    float* merge = reinterpret_cast<float*>(pf_sm + kPfWarps * S::kDepth * S::kSlot);
    pdl_trigger();
    if (!a.behind) pdl_wait();

    PaSched sched(a);
    sched.start(blockIdx.x, gridDim.x, lane);

    // ---- load cursor: this warp's slices of the share in order, the page of the next one looked up ahead
    PaSched ahead = sched;
    PaSeg lg{};
    int lj = 0, lpos = 0, lslot = 0;
    bool lany = true;
    const int32_t* ltab = nullptr;
    int lpage = -1;
    auto seek = [&]() {                               // the next slice that has positions, from unit lj on
        for (;;) {
            if (lj < lg.j1) {
                lpos = lj * kPaStep + warp * kPfSlice;
                if (lpos < lg.end) break;
                lj = lg.j1;
            }
            if (!ahead.next(lg)) {
                lany = false;
                return;
            }
            lj = lg.j0;
            ltab = a.b.page_table + (size_t)lg.s * a.b.table_cols;
        }
        lpage = ltab[lpos >> (31 - __clz(a.b.page_size))];             // lpos < end <= table_cols * page_size
    };
    auto load = [&]() {
        if (lany) {
            const bool has = lpage >= 0 && lpage < a.b.num_pages;
            if (!has && lane == 0) atomicOr(a.status, kStatusPagedRange);
            const size_t at = ((((size_t)(has ? lpage : 0) * a.b.hkv + lg.h) * a.b.page_size) + (lpos & (a.b.page_size - 1))) * HD +
                              lane * 8;
            const C* k = static_cast<const C*>(a.b.k_pages) + at;
            const C* v = static_cast<const C*>(a.b.v_pages) + at;
            const uint32_t dst = ring + lslot * S::kSlot;
            const int valid = has ? lg.end - lpos : 0;                 // positions behind the end are zero
#pragma unroll
            for (int i = 0; i < kPfSlice / kPer; ++i) {
                const int r = i * kPer + lane / kChunks, ch = lane % kChunks;
                const uint32_t d = dst + r * S::kRow + ((ch ^ (r & 7)) << 4);
                const int bytes = r < valid ? 16 : 0;
                cp_async16_or_zero(d, k + i * 256, bytes);
                cp_async16_or_zero(d + kPfSlice * S::kRow, v + i * 256, bytes);
            }
            lslot = lslot + 1 == S::kDepth ? 0 : lslot + 1;
            ++lj;
            seek();
        }
        cp_async_commit();
    };
    seek();
    for (int i = 0; i < S::kDepth - 1; ++i) load();

    const float c = a.scale_log2;
    PaSeg g{};
    int slot = 0;
    // ldmatrix addresses within a slot: K rows as they are, V transposed
    const int krow = lane & 15, kch = lane >> 4;
    const int vrow = (lane & 7) + ((lane >> 4) << 3), vch = (lane >> 3) & 1;
    uint32_t qb[NQ][HD / 16][2];                      // Q^T fragments of segment g
    auto load_q = [&]() {
        const int used = min(8 * NQ, g.rows * a.grp - g.p0);
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
            const int p = g.p0 + 8 * t + gid, tok = by_grp(a, p), row = g.start + tok;
            const bool live = 8 * t + gid < used && row < a.b.rows;
            const C* src = static_cast<const C*>(a.q) + row * a.q_stride + (size_t)(g.h * a.grp + (p - tok * a.grp)) * HD + 2 * tig;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                qb[t][ks][0] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * ks) : 0u;
                qb[t][ks][1] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 8) : 0u;
            }
        }
    };
    bool more = sched.next(g);
    const bool any = more;
    if (more) load_q();
    while (more) {
        const int used = min(8 * NQ, g.rows * a.grp - g.p0);
        int lim[NQ][2], least = 0x7fffffff;           // positions this lane's columns see
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int q = 8 * t + 2 * tig + e;
                lim[t][e] = q < used ? min(g.end, g.ctx + by_grp(a, g.p0 + q) + 1) : 0x7fffffff;
                least = min(least, lim[t][e]);
            }
        if (lane == 0 && warp == 0 && g.ctx + by_grp(a, g.p0 + used - 1) >= sched.cap) atomicOr(a.status, kStatusPagedRange);
        float o[HD / 16][NQ][4] = {};
        float m[NQ][2], l[NQ][2];
#pragma unroll
        for (int t = 0; t < NQ; ++t) m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f;

        for (int j = g.j0; j < g.j1; ++j) {
            const int pos = j * kPaStep + warp * kPfSlice;
            if (pos >= g.end) break;
            __syncwarp();                             // the slot about to be refilled has been read by every lane
            load();
            cp_async_wait<S::kDepth - 1>();
            __syncwarp();
            const uint32_t ks_a = ring + slot * S::kSlot, vs_a = ks_a + kPfSlice * S::kRow;
            slot = slot + 1 == S::kDepth ? 0 : slot + 1;
            float s[NQ][4] = {};
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                uint32_t k[4];
                ldsm4(ks_a + krow * S::kRow + (((2 * ks + kch) ^ (krow & 7)) << 4), k);
#pragma unroll
                for (int t = 0; t < NQ; ++t) mma_16816<C>(s[t], k[0], k[1], k[2], k[3], qb[t][ks][0], qb[t][ks][1]);
            }
            // s[.][0], [1]: position pos + gid, columns 2 tig, + 1; [2], [3]: position + 8
            if (__any_sync(0xffffffffu, pos + kPfSlice > least)) {
#pragma unroll
                for (int t = 0; t < NQ; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (pos + gid + 8 * (e >> 1) >= lim[t][e & 1]) s[t][e] = -INFINITY;
            }
            bool grow = false;
#pragma unroll
            for (int t = 0; t < NQ; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) grow |= (fmaxf(s[t][e], s[t][e + 2]) - m[t][e]) * c > kPaSlack;
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int t = 0; t < NQ; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(m[t][e], fmaxf(s[t][e], s[t][e + 2]));
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                        const float f = top == -INFINITY ? 1.f : pa_weight(m[t][e], top, c);
                        m[t][e] = top;
                        l[t][e] *= f;
#pragma unroll
                        for (int i = 0; i < HD / 16; ++i) {
                            o[i][t][e] *= f;
                            o[i][t][e + 2] *= f;
                        }
                    }
            }
            uint32_t pb[NQ][2];
#pragma unroll
            for (int t = 0; t < NQ; ++t) {
                const float b0 = m[t][0] == -INFINITY ? 0.f : m[t][0] * c, b1 = m[t][1] == -INFINITY ? 0.f : m[t][1] * c;
                const float p0 = ex2(fmaf(s[t][0], c, -b0)), p1 = ex2(fmaf(s[t][1], c, -b1));
                const float p2 = ex2(fmaf(s[t][2], c, -b0)), p3 = ex2(fmaf(s[t][3], c, -b1));
                l[t][0] += p0 + p2;
                l[t][1] += p1 + p3;
                pb[t][0] = transpose8(pack2<C>(p0, p1));
                pb[t][1] = transpose8(pack2<C>(p2, p3));
            }
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
                uint32_t v[4];
                ldsm4_t(vs_a + vrow * S::kRow + (((2 * i + vch) ^ (vrow & 7)) << 4), v);
#pragma unroll
                for (int t = 0; t < NQ; ++t) mma_16816<C>(o[i][t], v[0], v[1], v[2], v[3], pb[t][0], pb[t][1]);
            }
        }

        const PaSeg done = g;
        more = sched.next(g);
        if (more) load_q();                           // on their way while this segment is merged

        // ---- the warps' results, merged in warp order
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], x);
                if (gid == 0) {
                    wm[warp][8 * t + 2 * tig + e] = m[t][e];
                    wl[warp][8 * t + 2 * tig + e] = l[t][e];
                }
            }
        const bool whole = done.j0 == 0 && done.j1 == done.units;
        uint8_t* part = pa_part<HD, kPaFew, 1>(a.parts, done.c0, blockIdx.x, 0);
#pragma unroll
        for (int c0 = 0; c0 < HD; c0 += S::kCols) {
#pragma unroll
            for (int i = c0 / 16; i < (c0 + S::kCols) / 16; ++i)
#pragma unroll
                for (int t = 0; t < NQ; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        merge[(warp * 8 * NQ + 8 * t + 2 * tig + (e & 1)) * S::kPad + i * 16 - c0 + gid + 8 * (e >> 1)] = o[i][t][e];
            __syncthreads();
            const int r = threadIdx.x % (8 * NQ), quad = threadIdx.x / (8 * NQ);       // a thread per row and column quad
            static_assert(8 * NQ * (S::kCols / 4) <= 32 * kPfWarps, "one pass");
            if (r < used && quad < S::kCols / 4) {
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kPfWarps; ++w) top = fmaxf(top, wm[w][r]);
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kPfWarps; ++w) {
                    const float f = pa_weight(wm[w][r], top, c);
                    const float4 y = *reinterpret_cast<const float4*>(merge + (w * 8 * NQ + r) * S::kPad + quad * 4);
                    sum += wl[w][r] * f;
                    acc.x += y.x * f;
                    acc.y += y.y * f;
                    acc.z += y.z * f;
                    acc.w += y.w * f;
                }
                if (whole) {
                    const int p = done.p0 + r, tok = by_grp(a, p), row = done.start + tok;
                    if (row < a.b.rows) {
                        const float inv = 1.f / sum;
                        uint2 w = make_uint2(pack2<C>(acc.x * inv, acc.y * inv), pack2<C>(acc.z * inv, acc.w * inv));
                        if (sum == 0.f) w = make_uint2(0, 0);
                        *reinterpret_cast<uint2*>(static_cast<C*>(a.out) +
                                                  ((size_t)row * a.hq + done.h * a.grp + (p - tok * a.grp)) * HD + c0 + quad * 4) = w;
                    }
                } else {
                    __stcg(reinterpret_cast<float4*>(part) + (c0 / 4 + quad) * used + r, acc);
                    if (c0 == 0 && quad == 0) __stcg(reinterpret_cast<float2*>(part + PaPart<HD, kPaFew>::kMl) + r, make_float2(top, sum));
                }
            }
            __syncthreads();
        }
    }
    if (threadIdx.x == 0) pa_record(a, sched.bad, any, g, any ? min(8 * NQ, g.rows * a.grp - g.p0) : 0, 8 * NQ);   // g: the last segment
    cp_async_wait<0>();
    if (a.behind) pdl_wait();                         // so that the merge, which waits for this kernel, finds the tiles' parts too
}

template <typename C, int HD, int NQ>
static int launch_few(const PaArgs& args, cudaStream_t s)
{
    static bool attr_set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return EXL3_E_CUDA;
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        if (cudaFuncSetAttribute(paged_few_kernel<C, HD, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 PfShape<HD, NQ>::kSmem) != cudaSuccess)
            return EXL3_E_CUDA;
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    PaArgs a = args;
    a.span = 8 * NQ;
    a.item = 2;
    const int ctas = device_sm_count();
    return launch_pdl(paged_few_kernel<C, HD, NQ>, dim3(ctas), dim3(32 * kPfWarps), PfShape<HD, NQ>::kSmem, s, a);
}

template <typename C>
static int launch_few(const PaArgs& a, cudaStream_t s)
{
    // 8 packed rows at a time where a sequence has no more on average: half the accumulators and MMAs of 16. (24 at a time was
    // measured no faster than two passes of 16 over keys and values that the second pass finds in L2: 37.2 against 40.3 us for
    // 64 sequences of 3 rows, 39.5 against 37.1 for two of 4.)
    const bool eight = (long long)a.b.rows * a.grp <= 8ll * a.b.seqs;
    if (a.b.head_dim == 128) return eight ? launch_few<C, 128, 1>(a, s) : launch_few<C, 128, 2>(a, s);
    return eight ? launch_few<C, 64, 1>(a, s) : launch_few<C, 64, 2>(a, s);
}

int pa_launch_few(const PaArgs& a, cudaStream_t s)
{
    return a.b.dtype == EXL3_F16 ? launch_few<__half>(a, s) : launch_few<__nv_bfloat16>(a, s);
}

}  // namespace exl3
