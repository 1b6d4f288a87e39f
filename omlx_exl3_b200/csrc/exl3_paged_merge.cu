// Merges the partial results of paged-attention items that were cut between CTAs, in CTA order:
//   m = max m_k, out = sum_k exp2((m_k - m) c) O_k / sum_k exp2((m_k - m) c) l_k.
//
// grid (CTAs of the attention kernels, blocks of an item, lists): block x looks at the item that started in CTA x's share.
// (One CTA, the last to finish its part, merging alone was measured first: 40 rows of 33 parts are 0.7 MB, 25 us for one
// SM.) The time is L2 latency: the loads of E column quads and K parts are in flight at once.
#include <cuda_runtime.h>

#include "exl3_b200.h"
#include "exl3_common.cuh"
#include "exl3_host.h"
#include "exl3_paged.cuh"
#include "exl3_paged_sched.cuh"

namespace exl3 {

constexpr int kPmThreads = 128;
constexpr int kPmBlocks = 8;                          // of an item

template <typename C, int HD, int ROWS, int TILES>
__device__ __forceinline__ void merge_item(const PaArgs& a, const PaItem& g)
{
    constexpr int E = 2, K = 4;
    constexpr size_t kMl = PaPart<HD, ROWS>::kMl;
    const float c = a.scale_log2;
    const int n = g.used * (HD / 4), stride = kPmThreads * gridDim.y;
    const int used0 = min(g.used, g.gap);
    for (int e0 = blockIdx.y * kPmThreads + threadIdx.x; e0 < n; e0 += E * stride) {
        int tile[E], at[E], row[E];                   // tile, quad index and row in the tile's part
        float top[E], sum[E];
        float4 acc[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int e = min(e0 + i * stride, n - 1);
            tile[i] = TILES > 1 && e >= used0 * (HD / 4) ? 1 : 0;
            at[i] = e - tile[i] * used0 * (HD / 4);
            row[i] = at[i] % (tile[i] ? g.used - used0 : used0);
            top[i] = -INFINITY;
            sum[i] = 0.f;
            acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        for (int k0 = 0; k0 < g.parts; k0 += K) {
            float2 w[E][K];
            float4 y[E][K];
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const uint8_t* pt = pa_part<HD, ROWS, TILES>(a.parts, g.c0, g.c0 + min(k0 + k, g.parts - 1), tile[i]);
                    w[i][k] = __ldcg(reinterpret_cast<const float2*>(pt + kMl) + row[i]);
                    y[i][k] = __ldcg(reinterpret_cast<const float4*>(pt) + at[i]);
                }
#pragma unroll
            for (int i = 0; i < E; ++i) {
                float now = top[i];
#pragma unroll
                for (int k = 0; k < K; ++k) now = fmaxf(now, w[i][k].x);      // the clamped ones are a part's own again
                const float f0 = pa_weight(top[i], now, c);
                top[i] = now;
                sum[i] *= f0;
                acc[i].x *= f0;
                acc[i].y *= f0;
                acc[i].z *= f0;
                acc[i].w *= f0;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (k0 + k >= g.parts) continue;
                    const float f = pa_weight(w[i][k].x, now, c);
                    sum[i] = fmaf(w[i][k].y, f, sum[i]);
                    acc[i].x = fmaf(y[i][k].x, f, acc[i].x);
                    acc[i].y = fmaf(y[i][k].y, f, acc[i].y);
                    acc[i].z = fmaf(y[i][k].z, f, acc[i].z);
                    acc[i].w = fmaf(y[i][k].w, f, acc[i].w);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int quad = at[i] / (tile[i] ? g.used - used0 : used0);
            const int p = g.p0 + tile[i] * g.gap + row[i], tok = p / a.grp, r = g.start + tok;
            if (e0 + i * stride >= n || r >= a.b.rows) continue;
            const float inv = 1.f / sum[i];
            uint2 w = make_uint2(pack2<C>(acc[i].x * inv, acc[i].y * inv), pack2<C>(acc[i].z * inv, acc[i].w * inv));
            if (sum[i] == 0.f) w = make_uint2(0, 0);
            *reinterpret_cast<uint2*>(static_cast<C*>(a.out) + ((size_t)r * a.hq + g.h * a.grp + (p - tok * a.grp)) * HD + quad * 4) = w;
        }
    }
}

template <typename C, int HD>
__global__ void __launch_bounds__(kPmThreads) paged_merge_kernel(const __grid_constant__ PaArgs tiles, const __grid_constant__ PaArgs few)
{
    pdl_trigger();
    pdl_wait();
    const bool is_few = blockIdx.z == 1 || !tiles.items;
    const PaArgs& a = is_few ? few : tiles;
    const PaItem g = a.items[blockIdx.x];
    if (g.parts < 2) return;
    if (is_few) merge_item<C, HD, kPaFew, 1>(a, g);
    else merge_item<C, HD, kPaRows, 2>(a, g);
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
    // an item of few rows is one pass of a block or two
    const dim3 grid(ctas, tiles ? kPmBlocks : 2, tiles && few ? 2 : 1);
    return a.b.dtype == EXL3_F16 ? launch_merge<__half>(tiles ? *tiles : none, few ? *few : none, a.b.head_dim, grid, s)
                                 : launch_merge<__nv_bfloat16>(tiles ? *tiles : none, few ? *few : none, a.b.head_dim, grid, s);
}

}  // namespace exl3
