// After the q/k/v projections of a paged batch: per-head RMSNorm of q and k, rotary embedding, k and v
// appended to the cache's pages, q in the cache's type. fp32 inside, one rounding at the end.
//
//   xn = x * rsqrt(mean(x^2) + eps) * w ;  (a, b) = (xn[c], xn[c + R]) -> (a cos - b sin, b cos + a sin), c < R
#include <cuda_runtime.h>

#include "exl3_b200.h"
#include "exl3_common.cuh"
#include "exl3_host.h"
#include "exl3_paged.cuh"

namespace exl3 {

struct PagedPostArgs {
    exl3_paged_desc b;
    const void *q, *k, *v, *qw, *kw;
    long long sq, sk, sv;
    const float *cos_t, *sin_t;
    void* q_out;
    uint32_t* status;
    float eps;
    int hq, rope_rows, rope_half, vec;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8])
{
    if (vec) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
    }
}

template <typename C>
__device__ __forceinline__ void store8(C* p, const float (&x)[8])
{
    uint4 u;
    C* e = reinterpret_cast<C*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<C>(x[i]);
    *reinterpret_cast<uint4*>(p) = u;
}

// grid (rows, parts), 4 warps: the row's heads are dealt to the row's warps. A head is HD / 8 lanes of 8
// consecutive elements, so a rotation pair sits rope_half / 8 lanes apart.
template <typename T, typename C, int HD>
__global__ void __launch_bounds__(128) paged_post_kernel(const PagedPostArgs a)
{
    constexpr int L = HD / 8;                            // lanes of one head
    constexpr int PER = 32 / L;                          // heads a warp handles at once
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x;
    const int sub = lane % L, c0 = sub * 8;
    const int R = a.rope_half;
    const exl3_paged_desc& b = a.b;
    pdl_wait();
    const int s = seq_of_row(b.cu_rows, b.seqs, row, lane);
    const int pos = b.lens[s] - b.cu_rows[s + 1] + row;
    const bool pad = pos < 0;
    const bool known = pos < a.rope_rows;
    const int page = page_of(b, s, pos);
    if (!pad && (!known || page < 0) && threadIdx.x == 0) atomicOr(a.status, kStatusPagedRange);
    const bool rotated = c0 < 2 * R;
    float co[8] = {}, si[8] = {};
    if (rotated && !pad && known) {
        const size_t at = (size_t)pos * R + (c0 < R ? c0 : c0 - R);
        *reinterpret_cast<float4*>(co) = *reinterpret_cast<const float4*>(a.cos_t + at);
        *reinterpret_cast<float4*>(co + 4) = *reinterpret_cast<const float4*>(a.cos_t + at + 4);
        *reinterpret_cast<float4*>(si) = *reinterpret_cast<const float4*>(a.sin_t + at);
        *reinterpret_cast<float4*>(si + 4) = *reinterpret_cast<const float4*>(a.sin_t + at + 4);
    }
    const int partner = c0 < R ? lane + R / 8 : lane - R / 8;
    const int heads = a.hq + 2 * b.hkv;
    const int stride = gridDim.y * 4 * PER;
    for (int h0 = (blockIdx.y * 4 + warp) * PER; h0 < heads; h0 += stride) {
        const int h = h0 + lane / L;
        const bool live = h < heads;
        const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + b.hkv;
        float x[8] = {};
        if (live) {
            const T* src = is_q ? static_cast<const T*>(a.q) + row * a.sq + (size_t)h * HD
                         : is_k ? static_cast<const T*>(a.k) + row * a.sk + (size_t)(h - a.hq) * HD
                                : static_cast<const T*>(a.v) + row * a.sv + (size_t)(h - a.hq - b.hkv) * HD;
            load8(src + c0, a.vec, x);
        }
        const T* w = static_cast<const T*>(is_q ? a.qw : a.kw);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = 1; o < L; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (live && (is_q || is_k) && w) {
            const float inv = 1.0f / sqrtf(ss / (float)HD + a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * to_f32(w[c0 + i]);
        }
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float o = __shfl_sync(0xffffffffu, x[i], rotated ? partner : lane);
            y[i] = !rotated ? x[i] : c0 < R ? x[i] * co[i] - o * si[i] : x[i] * co[i] + o * si[i];
        }
        if (!live) continue;
        if (is_q) {
            if (pad || !known)
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = 0.f;
            store8(static_cast<C*>(a.q_out) + ((size_t)row * a.hq + h) * HD + c0, y);
        } else if (!pad && known && page >= 0) {
            const int hk = h - a.hq - (is_k ? 0 : b.hkv);
            const size_t at = (((size_t)page * b.hkv + hk) * b.page_size + (pos & (b.page_size - 1))) * HD + c0;
            if (is_k) store8(static_cast<C*>(b.k_pages) + at, y);
            else store8(static_cast<C*>(b.v_pages) + at, x);
        }
    }
}

template <typename T, typename C>
static int launch_post(const PagedPostArgs& a, dim3 grid, cudaStream_t s)
{
    return a.b.head_dim == 128 ? launch_pdl(paged_post_kernel<T, C, 128>, grid, dim3(128), 0, s, a)
                               : launch_pdl(paged_post_kernel<T, C, 64>, grid, dim3(128), 0, s, a);
}

}  // namespace exl3

using namespace exl3;

int exl3_check_paged(const exl3_paged_desc* b)
{
    if (!b || !b->k_pages || !b->v_pages || !b->page_table || !b->cu_rows || !b->lens) return EXL3_E_NULL;
    if (b->seqs < 1 || b->rows < 0 || b->table_cols < 1 || b->num_pages < 1 || b->hkv < 1) return EXL3_E_SHAPE;
    if (b->page_size < 16 || (b->page_size & (b->page_size - 1))) return EXL3_E_SHAPE;
    if ((long long)b->table_cols * b->page_size > 0x7fffffffll) return EXL3_E_SHAPE;
    if (b->head_dim != 64 && b->head_dim != 128) return EXL3_E_SHAPE;
    if (b->dtype != EXL3_F16 && b->dtype != EXL3_BF16) return EXL3_E_DTYPE;
    if (!aligned(b->k_pages, 16) || !aligned(b->v_pages, 16) || !aligned(b->page_table, 4) || !aligned(b->cu_rows, 4) ||
        !aligned(b->lens, 4))
        return EXL3_E_ALIGN;
    return EXL3_OK;
}

extern "C" int exl3_paged_qkv_post(const exl3_paged_desc* batch, const void* q, const void* k, const void* v,
                                   long long q_stride, long long k_stride, long long v_stride, int in_dtype, int hq,
                                   const void* q_norm_w, const void* k_norm_w, float eps, const float* cos_table,
                                   const float* sin_table, int rope_rows, int rope_half, void* q_out, uint32_t* status,
                                   void* stream)
{
    if (int e = exl3_check_paged(batch)) return e;
    if (batch->rows == 0) return EXL3_OK;
    if (!q || !k || !v || !cos_table || !sin_table || !q_out || !status) return EXL3_E_NULL;
    if (hq < 1 || hq % batch->hkv || rope_rows < 1 || rope_half < 8 || rope_half % 8 || 2 * rope_half > batch->head_dim)
        return EXL3_E_SHAPE;
    if (q_stride < (long long)hq * batch->head_dim || k_stride < (long long)batch->hkv * batch->head_dim ||
        v_stride < (long long)batch->hkv * batch->head_dim)
        return EXL3_E_SHAPE;
    if (in_dtype != EXL3_F16 && in_dtype != EXL3_BF16) return EXL3_E_DTYPE;
    if (!aligned(q, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(q_norm_w, 2) || !aligned(k_norm_w, 2) ||
        !aligned(cos_table, 16) || !aligned(sin_table, 16) || !aligned(q_out, 16) || !aligned(status, 4))
        return EXL3_E_ALIGN;
    if (int e = check_device()) return e;
    PagedPostArgs a{};
    a.b = *batch;
    a.q = q; a.k = k; a.v = v; a.qw = q_norm_w; a.kw = k_norm_w;
    a.sq = q_stride; a.sk = k_stride; a.sv = v_stride;
    a.cos_t = cos_table; a.sin_t = sin_table;
    a.q_out = q_out; a.status = status; a.eps = eps;
    a.hq = hq; a.rope_rows = rope_rows; a.rope_half = rope_half;
    a.vec = aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && q_stride % 8 == 0 && k_stride % 8 == 0 &&
            v_stride % 8 == 0;
    const int per_cta = 4 * (32 / (batch->head_dim / 8));
    const int parts = (hq + 2 * batch->hkv + per_cta - 1) / per_cta;
    const dim3 grid(batch->rows, parts);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (in_dtype == EXL3_F16)
        return batch->dtype == EXL3_F16 ? launch_post<__half, __half>(a, grid, s)
                                        : launch_post<__half, __nv_bfloat16>(a, grid, s);
    return batch->dtype == EXL3_F16 ? launch_post<__nv_bfloat16, __half>(a, grid, s)
                                    : launch_post<__nv_bfloat16, __nv_bfloat16>(a, grid, s);
}
