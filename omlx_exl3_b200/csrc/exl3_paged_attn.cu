// Attention of a batch's new rows over paged keys and values.
//
//   out[r, h] = sum_j p_j V[j, h / g] / sum_j p_j,  p_j = exp(scale q[r, h] . K[j, h / g] - max),  j <= pos(r)
//
// One warp per (row, head) walks the positions one by one with a running maximum and sum in fp32.
#include <cuda_runtime.h>

#include "exl3_b200.h"
#include "exl3_common.cuh"
#include "exl3_host.h"
#include "exl3_paged.cuh"

namespace exl3 {

template <typename C, int HD>
__global__ void __launch_bounds__(128) paged_attn_kernel(const exl3_paged_desc b, const C* __restrict__ q,
                                                         long long q_stride, int hq, float scale, C* __restrict__ out,
                                                         uint32_t* status)
{
    constexpr int E = HD / 32;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int item = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int row = blockIdx.x, h = item;
    if (h >= hq) return;
    const int kvh = h / (hq / b.hkv);
    const int s = seq_of_row(b.cu_rows, b.seqs, row, lane);
    const int pos = b.lens[s] - b.cu_rows[s + 1] + row;
    float qv[E], o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        qv[i] = to_f32(q[row * q_stride + (size_t)h * HD + lane * E + i]) * scale;
        o[i] = 0.f;
    }
    const C* kp = static_cast<const C*>(b.k_pages);
    const C* vp = static_cast<const C*>(b.v_pages);
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j <= pos; ++j) {
        const int page = page_of(b, s, j);
        if (page < 0) {
            if (lane == 0) atomicOr(status, kStatusPagedRange);
            continue;
        }
        const size_t at = (((size_t)page * b.hkv + kvh) * b.page_size + (j & (b.page_size - 1))) * HD + lane * E;
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) d = fmaf(qv[i], to_f32(kp[at + i]), d);
        d = warp_sum(d);
        const float mn = fmaxf(m, d);
        if (mn == -INFINITY) continue;
        const float f = expf(m - mn), p = expf(d - mn);
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = fmaf(p, to_f32(vp[at + i]), o[i] * f);
        m = mn;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int i = 0; i < E; ++i) out[((size_t)row * hq + h) * HD + lane * E + i] = from_f32<C>(o[i] * inv);
}

template <typename C>
static int launch_attn(const exl3_paged_desc& b, const void* q, long long q_stride, int hq, float scale, void* out,
                       uint32_t* status, cudaStream_t s)
{
    const dim3 grid(b.rows, (hq + 3) / 4);
    const C* qp = static_cast<const C*>(q);
    C* op = static_cast<C*>(out);
    return b.head_dim == 128 ? launch_pdl(paged_attn_kernel<C, 128>, grid, dim3(128), 0, s, b, qp, q_stride, hq, scale, op, status)
                             : launch_pdl(paged_attn_kernel<C, 64>, grid, dim3(128), 0, s, b, qp, q_stride, hq, scale, op, status);
}

static int check_attn(const exl3_paged_desc* b, int hq)
{
    if (int e = exl3_check_paged(b)) return e;
    if (hq < 1 || hq % b->hkv || hq / b->hkv > 128) return EXL3_E_SHAPE;
    return EXL3_OK;
}

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_paged_attn_workspace(const exl3_paged_desc* batch, int hq, size_t* bytes)
{
    if (!bytes) return EXL3_E_NULL;
    if (int e = check_attn(batch, hq)) return e;
    *bytes = 0;
    return EXL3_OK;
}

extern "C" int exl3_paged_attn(const exl3_paged_desc* batch, const void* q, long long q_stride, int hq, float scale,
                               void* out, void* workspace, size_t workspace_bytes, uint32_t* status, void* stream)
{
    if (int e = check_attn(batch, hq)) return e;
    if (batch->rows == 0) return EXL3_OK;
    if (!q || !out || !status) return EXL3_E_NULL;
    if (q_stride < (long long)hq * batch->head_dim || !(scale > 0.f)) return EXL3_E_SHAPE;
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(status, 4) || q_stride % 8) return EXL3_E_ALIGN;
    if (int e = check_device()) return e;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return batch->dtype == EXL3_F16 ? launch_attn<__half>(*batch, q, q_stride, hq, scale, out, status, s)
                                    : launch_attn<__nv_bfloat16>(*batch, q, q_stride, hq, scale, out, status, s);
}
