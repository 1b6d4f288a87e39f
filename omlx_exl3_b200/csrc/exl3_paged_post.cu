// After the q/k/v projections of a paged batch: per-head RMSNorm of q and k, rotary embedding, k and v
// appended to the cache's pages, q in the cache's type. fp32 inside, one rounding at the end.
//
//   xn = x * rsqrt(mean(x^2) + eps) * w ;  (a, b) = (xn[c], xn[c + R]) -> (a cos - b sin, b cos + a sin), c < R
//
// Where there are many rows, bound by issue (64 % of the slots; DRAM is a quarter busy) and the rounds of loads of one wave: 3428
// rows of 40 + 2 x 8 heads of 128, 100 MB in 23.7 us, 4.2 TB/s, 0.65 of a measured copy. Where there are few, by launch and
// dependent loads (2.8 us).
#include <cuda_runtime.h>

#include <algorithm>

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
    int hq, rope_rows, rope_half;
    int per_row;                                     // warps of a row
};

// Four consecutive elements as they are stored; VEC: one 8-byte load.
template <typename T, bool VEC>
__device__ __forceinline__ uint2 load4(const T* p)
{
    if constexpr (VEC) return *reinterpret_cast<const uint2*>(p);
    const unsigned short* e = reinterpret_cast<const unsigned short*>(p);
    return make_uint2(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16);
}

template <typename T>
__device__ __forceinline__ void widen4(uint2 u, float* x)
{
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32(e[i]);
}

template <typename C>
__device__ __forceinline__ void store4(C* p, const float* x)
{
    uint2 u;
    C* e = reinterpret_cast<C*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = from_f32<C>(x[i]);
    *reinterpret_cast<uint2*>(p) = u;
}

// A warp handles one row and every per_row-th group of its heads (PER heads at once). A lane holds two runs of four elements of
// a head, the two sides of its rotation pairs (c and c + rope_half), so rotating needs no exchange; lanes past the rotated
// part hold two runs of what passes unchanged. What belongs to the row (its sequence, page, rotation) is looked up once.
// The loads are U groups deep, the first of them under way while the row is looked up (a single token 3.15 -> 2.86 us); asking for
// the next round's within a round was slower (50.6 us for the 3428 rows), and so were two or three groups at more CTAs (25.2
// to 29.5). Six CTAs an SM, since a warp that handles a whole row runs long: five took a second wave (31.9 us).
template <typename T, typename C, int HD, bool VEC>
__global__ void __launch_bounds__(128, 6) paged_post_kernel(const PagedPostArgs a)
{
    constexpr int L = HD / 8;                            // lanes of one head
    constexpr int PER = 32 / L;                          // heads a warp handles at once
    constexpr int U = 4;                                 // groups in flight
    pdl_trigger();
    const int lane = threadIdx.x & 31, sub = lane % L;
    const int item = blockIdx.x * 4 + (threadIdx.x >> 5);
    const int row = item / a.per_row, part = item - row * a.per_row;
    const exl3_paged_desc& b = a.b;
    if (row >= b.rows) return;
    const int R = a.rope_half;
    const bool rotated = sub < R / 4;
    const int c0 = rotated ? 4 * sub : R + 4 * sub;      // past the rotated part: 2 R + 4 (sub - R / 4)
    const int c1 = rotated ? c0 + R : c0 + HD / 2 - R;
    pdl_wait();
    // the heads' loads do not depend on what is looked up for the row
    const int heads = a.hq + 2 * b.hkv, stride = a.per_row * PER;
    const T* const q = static_cast<const T*>(a.q) + row * a.sq;
    const T* const k = static_cast<const T*>(a.k) + row * a.sk - (size_t)a.hq * HD;
    const T* const v = static_cast<const T*>(a.v) + row * a.sv - (size_t)(a.hq + b.hkv) * HD;
    uint2 in[U][2];
    auto fetch = [&](int u, int g) {
        const int h = min(g + lane / L, heads - 1);
        const T* src = (h < a.hq ? q : h < a.hq + b.hkv ? k : v) + (size_t)h * HD;
        in[u][0] = load4<T, VEC>(src + c0);
        in[u][1] = load4<T, VEC>(src + c1);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(u, part * PER + u * stride);
    const int s = seq_of_row(b.cu_rows, b.seqs, row, lane);
    const int start = b.cu_rows[s], end = b.cu_rows[s + 1], pos = b.lens[s] - end + row;
    const bool inside = row >= start && row < end, pad = pos < 0 || !inside, known = pos < a.rope_rows;
    const int page = page_of(b, s, pos);
    if ((pad || !known || page < 0) && lane == 0 && part == 0) {
        // a row that its sequence does not have, though it is neither the first's nor the last's: cu_rows falls there
        const bool astray = (row < start && s > 0) || (row >= end && s + 1 < b.seqs);
        if (astray || !pad) atomicOr(a.status, kStatusPagedRange);
    }
    const bool append = !pad && known && page >= 0, has_q = !pad && known;
    float co[4] = {}, si[4] = {};
    if (rotated && has_q) {
        *reinterpret_cast<float4*>(co) = *reinterpret_cast<const float4*>(a.cos_t + (size_t)pos * R + c0);
        *reinterpret_cast<float4*>(si) = *reinterpret_cast<const float4*>(a.sin_t + (size_t)pos * R + c0);
    }
    uint2 wq0{}, wq1{}, wk0{}, wk1{};
    if (a.qw) {
        wq0 = load4<T, VEC>(static_cast<const T*>(a.qw) + c0);
        wq1 = load4<T, VEC>(static_cast<const T*>(a.qw) + c1);
    }
    if (a.kw) {
        wk0 = load4<T, VEC>(static_cast<const T*>(a.kw) + c0);
        wk1 = load4<T, VEC>(static_cast<const T*>(a.kw) + c1);
    }
    C* const qo = static_cast<C*>(a.q_out) + (size_t)row * a.hq * HD;
    const size_t slot = ((size_t)max(page, 0) * b.hkv * b.page_size + (pos & (b.page_size - 1))) * HD;
    for (int g0 = part * PER; g0 < heads; g0 += U * stride) {
        if (g0 != part * PER)
#pragma unroll
            for (int u = 0; u < U; ++u) fetch(u, g0 + u * stride);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = g0 + u * stride + lane / L;
            const bool live = h < heads, is_q = h < a.hq, is_k = !is_q && h < a.hq + b.hkv;
            float x[8], y[8];
            widen4<T>(in[u][0], x);
            widen4<T>(in[u][1], x + 4);
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int o = 1; o < L; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (is_q ? a.qw != nullptr : is_k && a.kw) {
                const float inv = rsqrtf(ss / (float)HD + a.eps);
                float w[8];
                widen4<T>(make_uint2(is_q ? wq0.x : wk0.x, is_q ? wq0.y : wk0.y), w);
                widen4<T>(make_uint2(is_q ? wq1.x : wk1.x, is_q ? wq1.y : wk1.y), w + 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= inv * w[i];
            }
            if (rotated && (is_q || is_k)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[i] = x[i] * co[i] - x[i + 4] * si[i];
                    y[i + 4] = x[i + 4] * co[i] + x[i] * si[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i];
            }
            if (is_q && !has_q)
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = 0.f;
            C* dst = is_q ? qo + (size_t)h * HD
                          : static_cast<C*>(is_k ? b.k_pages : b.v_pages) + slot + (size_t)(h - a.hq - (is_k ? 0 : b.hkv)) * b.page_size * HD;
            if (live && (is_q || append)) {
                store4(dst + c0, y);
                store4(dst + c1, y + 4);
            }
        }
    }
}

// Reads and clears in one step, so that a bit set meanwhile is in this reading or the next.
__global__ void paged_status_take_kernel(uint32_t* status, uint32_t* taken) { *taken = atomicExch(status, 0u); }

template <typename T, typename C, bool VEC>
static int launch_post(const PagedPostArgs& a, dim3 grid, cudaStream_t s)
{
    return a.b.head_dim == 128 ? launch_pdl(paged_post_kernel<T, C, 128, VEC>, grid, dim3(128), 0, s, a)
                               : launch_pdl(paged_post_kernel<T, C, 64, VEC>, grid, dim3(128), 0, s, a);
}

template <typename T>
static int launch_post(const PagedPostArgs& a, bool vec, dim3 grid, cudaStream_t s)
{
    if (a.b.dtype == EXL3_F16) return vec ? launch_post<T, __half, true>(a, grid, s) : launch_post<T, __half, false>(a, grid, s);
    return vec ? launch_post<T, __nv_bfloat16, true>(a, grid, s) : launch_post<T, __nv_bfloat16, false>(a, grid, s);
}

}  // namespace exl3

using namespace exl3;

int exl3_check_paged(const exl3_paged_desc* b)
{
    if (!b || !b->k_pages || !b->v_pages || !b->page_table || !b->cu_rows || !b->lens) return EXL3_E_NULL;
    if (b->seqs < 1 || b->rows < 0 || b->table_cols < 1 || b->num_pages < 1 || b->hkv < 1) return EXL3_E_SHAPE;
    if (b->page_size < 16 || (b->page_size & (b->page_size - 1))) return EXL3_E_SHAPE;
    if ((long long)b->table_cols * b->page_size > (1ll << 30)) return EXL3_E_SHAPE;
    if (b->head_dim != 64 && b->head_dim != 128) return EXL3_E_SHAPE;
    if (b->dtype != EXL3_F16 && b->dtype != EXL3_BF16) return EXL3_E_DTYPE;
    if (!aligned(b->k_pages, 16) || !aligned(b->v_pages, 16) || !aligned(b->page_table, 4) || !aligned(b->cu_rows, 4) ||
        !aligned(b->lens, 4))
        return EXL3_E_ALIGN;
    return EXL3_OK;
}

extern "C" int exl3_paged_status_take(uint32_t* status, uint32_t* taken, void* stream)
{
    if (!status || !taken) return EXL3_E_NULL;
    if (!aligned(status, 4) || !aligned(taken, 4)) return EXL3_E_ALIGN;
    if (int e = check_device()) return e;
    paged_status_take_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(status, taken);
    return launch_status();
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
    const bool vec = aligned(q, 8) && aligned(k, 8) && aligned(v, 8) && aligned(q_norm_w, 8) && aligned(k_norm_w, 8) &&
                     q_stride % 4 == 0 && k_stride % 4 == 0 && v_stride % 4 == 0;
    // A row's warps: one for every four groups (one round of loads) while that fits the SMs' warp slots, then fewer and longer
    // ones. Measured at 56 heads of 128, us with 1 / 2 / 7 / 28 warps a row: 1 row 10.5 / 6.8 / 2.9 / 3.1, 600 rows 12.4 /
    // 11.2 / 6.8 / 15.2, 3428 rows 24.1 / 25.7 / 28.2 / 83.9.
    const int per = 32 / (batch->head_dim / 8), groups = (hq + 2 * batch->hkv + per - 1) / per;
    const int warps = 32 * device_sm_count();
    a.per_row = std::max(1, std::min((groups + 3) / 4, warps / batch->rows));
    const long long items = (long long)batch->rows * a.per_row;
    if ((items + 3) / 4 > 0x7fffffffll || items > 0x7fffffffll) return EXL3_E_SHAPE;
    const dim3 grid((unsigned)((items + 3) / 4));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return in_dtype == EXL3_F16 ? launch_post<__half>(a, vec, grid, s) : launch_post<__nv_bfloat16>(a, vec, grid, s);
}
