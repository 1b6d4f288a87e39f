// Merges the partial results of paged-attention items that were cut between CTAs, in CTA order:
//   m = max m_k, out = sum_k exp2((m_k - m) c) O_k / sum_k exp2((m_k - m) c) l_k.
//
// grid (CTAs of the attention kernels, blocks of an item of few rows, then of one of tiles): block x looks at the item
// that started in CTA x's share. (One CTA, the last to finish its part, merging alone was measured first: 40 rows of 33 parts are 0.7 MB, 25 us for one
// SM.) The time is L2 latency, so a quad's parts are loaded four at a time, and by four threads where there are many.
#include <cuda_runtime.h>

#include "exl3_b200.h"
#include "exl3_common.cuh"
#include "exl3_host.h"
#include "exl3_paged.cuh"
#include "exl3_paged_sched.cuh"

namespace exl3 {

constexpr int kPmThreads = 128;
constexpr int kPmBlocks = 16;                         // of an item of tiles (8, 12 and 32 were slower: 68.3, 64.9 and 63.1 us against
                                                      // 62.7 for 512 rows over 4096 positions of 40 / 8 heads)
constexpr int kPmFewBlocks = 8;                       // of one of few rows (4: 10.7 us against 9.2 for one row over 4097)

// A column quad of an item: its tile, its row there, its place in the tile's parts.
struct PmQuad {
    int tile, row, at, quad;
};

template <int HD, int TILES>
__device__ __forceinline__ PmQuad pm_quad(const PaItem& g, int e)
{
    const int used0 = min(g.used, g.gap);
    PmQuad q;
    q.tile = TILES > 1 && e >= used0 * (HD / 4) ? 1 : 0;
    q.at = e - q.tile * used0 * (HD / 4);
    const int used = q.tile ? g.used - used0 : used0;
    q.quad = q.at / used;
    q.row = q.at - q.quad * used;
    return q;
}

// A running (m, l, O) of a column quad.
struct PmSum {
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void scale(float f)
    {
        sum *= f;
        acc.x *= f;
        acc.y *= f;
        acc.z *= f;
        acc.w *= f;
    }
    __device__ __forceinline__ void add(float l, const float4& y, float f)
    {
        sum = fmaf(l, f, sum);
        acc.x = fmaf(y.x, f, acc.x);
        acc.y = fmaf(y.y, f, acc.y);
        acc.z = fmaf(y.z, f, acc.z);
        acc.w = fmaf(y.w, f, acc.w);
    }
};

// G neighbouring threads share a quad's parts (thread k takes parts k, k + G, ...), K parts' loads in flight each.
template <typename C, int HD, int ROWS, int TILES, int G>
__device__ __forceinline__ void merge_item(const PaArgs& a, const PaItem& g, int block, int blocks)
{
    constexpr int K = 4, QW = 32 / G;                 // quads of a warp
    constexpr size_t kMl = PaPart<HD, ROWS>::kMl;
    const float c = a.scale_log2;
    const int lane = threadIdx.x & 31, part0 = lane / QW;
    const int n = g.used * (HD / 4), stride = kPmThreads / G * blocks;
    for (int e0 = (block * (kPmThreads / 32) + (threadIdx.x >> 5)) * QW; e0 < n; e0 += stride) {
        const int e = e0 + lane % QW;
        const PmQuad q = pm_quad<HD, TILES>(g, min(e, n - 1));
        PmSum p;
        for (int k0 = part0; k0 < g.parts; k0 += K * G) {
            float2 w[K];
            float4 y[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                w[k] = make_float2(-INFINITY, 0.f);
                y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k0 + k * G < g.parts) {
                    const uint8_t* pt = pa_part<HD, ROWS, TILES>(a.parts, g.c0, g.c0 + k0 + k * G, q.tile);
                    w[k] = __ldcg(reinterpret_cast<const float2*>(pt + kMl) + q.row);
                    y[k] = __ldcg(reinterpret_cast<const float4*>(pt) + q.at);
                }
            }
            float now = p.top;
#pragma unroll
            for (int k = 0; k < K; ++k) now = fmaxf(now, w[k].x);
            p.scale(pa_weight(p.top, now, c));
            p.top = now;
#pragma unroll
            for (int k = 0; k < K; ++k)
                p.add(w[k].y, y[k], pa_weight(w[k].x, now, c));
        }
#pragma unroll
        for (int o = QW; o < 32; o <<= 1) {
            const float top = __shfl_xor_sync(0xffffffffu, p.top, o), sum = __shfl_xor_sync(0xffffffffu, p.sum, o);
            float4 y;
            y.x = __shfl_xor_sync(0xffffffffu, p.acc.x, o);
            y.y = __shfl_xor_sync(0xffffffffu, p.acc.y, o);
            y.z = __shfl_xor_sync(0xffffffffu, p.acc.z, o);
            y.w = __shfl_xor_sync(0xffffffffu, p.acc.w, o);
            const float now = fmaxf(p.top, top), f0 = pa_weight(p.top, now, c), f1 = pa_weight(top, now, c);
            const bool low = !(lane & o);              // both sides add in the same order
            PmSum r;
            r.add(low ? p.sum : sum, low ? p.acc : y, low ? f0 : f1);
            r.add(low ? sum : p.sum, low ? y : p.acc, low ? f1 : f0);
            r.top = now;
            p = r;
        }
        const int pr = g.p0 + q.tile * g.gap + q.row, tok = by_grp(a, pr), row = g.start + tok;
        if (part0 > 0 || e >= n || row >= a.b.rows) continue;
        const float inv = 1.f / p.sum;
        uint2 w = make_uint2(pack2<C>(p.acc.x * inv, p.acc.y * inv), pack2<C>(p.acc.z * inv, p.acc.w * inv));
        if (p.sum == 0.f) w = make_uint2(0, 0);
        *reinterpret_cast<uint2*>(static_cast<C*>(a.out) + ((size_t)row * a.hq + g.h * a.grp + (pr - tok * a.grp)) * HD + q.quad * 4) = w;
    }
}

template <typename C, int HD, int ROWS, int TILES>
__device__ __forceinline__ void merge_item(const PaArgs& a, const PaItem& g, int block, int blocks)
{
    if (g.parts <= 4) merge_item<C, HD, ROWS, TILES, 1>(a, g, block, blocks);
    else merge_item<C, HD, ROWS, TILES, 4>(a, g, block, blocks);
}

template <typename C, int HD>
__global__ void __launch_bounds__(kPmThreads) paged_merge_kernel(const __grid_constant__ PaArgs tiles, const __grid_constant__ PaArgs few)
{
    pdl_trigger();
    pdl_wait();
    const int few_blocks = few.items ? kPmFewBlocks : 0, block = blockIdx.y;
    const bool is_few = block < few_blocks;
    const PaArgs& a = is_few ? few : tiles;
    const PaItem g = a.items[blockIdx.x];
    const int first_row = a.b.cu_rows[0], end_row = a.b.cu_rows[a.b.seqs];
    {                                                 // rows before the first sequence's and behind the last one's: zeros
        const size_t row16 = (size_t)a.hq * HD / 8, n = row16 * a.b.rows, threads = (size_t)gridDim.x * gridDim.y * kPmThreads;
        const size_t lead = g.parts < 0 ? n : row16 * first_row, gap = g.parts < 0 ? 0 : row16 * end_row - lead;
        for (size_t i = (blockIdx.y * gridDim.x + blockIdx.x) * kPmThreads + threadIdx.x; i + gap < n; i += threads)
            reinterpret_cast<uint4*>(a.out)[i < lead ? i : i + gap] = make_uint4(0, 0, 0, 0);
    }
    if (g.parts < 2) return;
    if (is_few) merge_item<C, HD, kPaFew, 1>(a, g, block, kPmFewBlocks);
    else merge_item<C, HD, kPaRows, 2>(a, g, block - few_blocks, kPmBlocks);
}

template <typename C>
static int launch_merge(const PaArgs& t, const PaArgs& f, int head_dim, dim3 grid, cudaStream_t s)
{
    return head_dim == 128 ? launch_pdl(paged_merge_kernel<C, 128>, grid, dim3(kPmThreads), 0, s, t, f)
                           : launch_pdl(paged_merge_kernel<C, 64>, grid, dim3(kPmThreads), 0, s, t, f);
}

int pa_launch_merge(const PaArgs* tiles, const PaArgs* few, int ctas, cudaStream_t s)
{
    const PaArgs none{};
    const PaArgs& a = tiles ? *tiles : *few;
    const dim3 grid(ctas, (tiles ? kPmBlocks : 0) + (few ? kPmFewBlocks : 0));
    return a.b.dtype == EXL3_F16 ? launch_merge<__half>(tiles ? *tiles : none, few ? *few : none, a.b.head_dim, grid, s)
                                 : launch_merge<__nv_bfloat16>(tiles ? *tiles : none, few ? *few : none, a.b.head_dim, grid, s);
}

}  // namespace exl3
