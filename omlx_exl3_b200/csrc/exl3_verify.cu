// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
//   a_i = min(1, p_i(x_i) / q_i(x_i)), drafts accepted while u_i < a_i, then one draw from max(0, p - q) (after
//   a rejection) or p as the first largest w(v) / noise(v).
//
// One CTA per sequence: softmax statistics of each row pair in turn, then the race over the chosen row.
#include <cuda_runtime.h>

#include "exl3_b200.h"
#include "exl3_common.cuh"
#include "exl3_host.h"

namespace exl3 {

struct VerifyArgs {
    const void *target, *draft;
    long long target_ld, draft_ld, noise_ld;
    const long long* tokens;
    const int32_t* cu_rows;
    const float *temperature, *u, *noise;
    long long* out;
    int32_t* count;
    float* prob;
    int rows, seqs, n, max_drafts;
};

constexpr int kVerifyThreads = 512;

// (max, first column of the max, sum of exp((x - max) * inv_t)) of a row, the same in every thread.
template <typename T>
__device__ void row_stats(const T* x, int n, float inv_t, float& m, int& at, float& sum)
{
    __shared__ float sm[16];
    __shared__ int sa[16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    m = -INFINITY;
    at = 0x7fffffff;
    for (int i = threadIdx.x; i < n; i += kVerifyThreads) {
        const float v = to_f32(x[i]);
        if (v > m || (v == m && i < at)) { m = v; at = i; }
    }
    for (int o = 16; o; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (om > m || (om == m && oa < at)) { m = om; at = oa; }
    }
    __syncthreads();
    if (lane == 0) { sm[warp] = m; sa[warp] = at; }
    __syncthreads();
    m = sm[0];
    at = sa[0];
    for (int w = 1; w < 16; ++w)
        if (sm[w] > m || (sm[w] == m && sa[w] < at)) { m = sm[w]; at = sa[w]; }
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f;
    for (int i = threadIdx.x; i < n; i += kVerifyThreads) s += expf((to_f32(x[i]) - base) * inv_t);
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) sm[warp] = s;
    __syncthreads();
    sum = 0.f;
    for (int w = 0; w < 16; ++w) sum += sm[w];
    m = base;
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyArgs a)
{
    __shared__ float bv[16];
    __shared__ int bi[16];
    pdl_trigger();
    pdl_wait();
    const int s = blockIdx.x, tid = threadIdx.x;
    const int lo = a.cu_rows[s], hi = a.cu_rows[s + 1];
    long long* out = a.out + (size_t)s * (a.max_drafts + 1);
    const bool sane = lo >= 0 && hi > lo && hi <= a.rows;
    const float temp = a.temperature ? a.temperature[s] : 1.f;
    const float inv_t = temp > 0.f ? 1.f / temp : 1.f;
    const int drafts = sane ? min(hi - lo - 1, a.max_drafts) : 0;
    int n_acc = 0;
    bool going = true;
    float m = 0.f, sum = 0.f, qm = 0.f, qsum = 0.f, w_inv = 0.f, q_inv = 0.f;
    int at = 0, qat;
    long long x = -1;
    bool rejected = false;
    for (int j = 0; sane && j < hi - lo; ++j) {
        const bool last = j == hi - lo - 1;
        if (last && !going) break;
        const int row = lo + j, i = row - s;
        float pm, psum;
        int pat;
        const T* tr = static_cast<const T*>(a.target) + row * a.target_ld;
        row_stats(tr, a.n, inv_t, pm, pat, psum);
        const float p_inv = psum > 0.f ? 1.f / psum : 0.f;
        if (last || (j >= a.max_drafts && going)) {
            if (going) { m = pm; at = pat; w_inv = p_inv; n_acc = j; going = false; }
            if (last) break;
        }
        if (i < 0 || i >= a.rows - a.seqs) break;
        const long long d = a.tokens[i];
        const bool in = d >= 0 && d < a.n;
        const T* dr = a.draft ? static_cast<const T*>(a.draft) + i * a.draft_ld : nullptr;
        float pd = 0.f, qd = 1.f, dm = 0.f, dsum = 0.f, d_inv = 0.f;
        if (temp > 0.f) {
            if (in) pd = expf((to_f32(tr[d]) - pm) * inv_t) * p_inv;
            if (dr) {
                row_stats(dr, a.n, inv_t, dm, qat, dsum);
                d_inv = dsum > 0.f ? 1.f / dsum : 0.f;
                qd = in ? expf((to_f32(dr[d]) - dm) * inv_t) * d_inv : 0.f;
            }
        } else {
            pd = in && d == pat && psum > 0.f ? 1.f : 0.f;
        }
        const float prob = qd > 0.f ? fminf(pd / qd, 1.f) : (pd > 0.f ? 1.f : 0.f);
        if (tid == 0) a.prob[i] = prob;
        if (!going) continue;
        if (a.u[i] < prob) {
            if (tid == 0) out[j] = d;
            continue;
        }
        going = false;
        rejected = true;
        n_acc = j;
        m = pm; at = pat; sum = psum; w_inv = p_inv; qm = dm; qsum = dsum; q_inv = d_inv;
        x = d;
    }
    (void)sum; (void)qsum; (void)drafts;
    long long next = -1;
    if (sane) {
        if (temp > 0.f) {
            const T* tr = static_cast<const T*>(a.target) + (lo + n_acc) * a.target_ld;
            const T* dr = a.draft && rejected ? static_cast<const T*>(a.draft) + (lo + n_acc - s) * a.draft_ld : nullptr;
            const float* e = a.noise + s * a.noise_ld;
            for (int pass = rejected ? 0 : 1; pass < 2 && next < 0; ++pass) {
                float best = 0.f;
                int idx = 0x7fffffff;
                for (int v = tid; v < a.n; v += kVerifyThreads) {
                    float w = expf((to_f32(tr[v]) - m) * inv_t) * w_inv;
                    if (pass == 0) w -= dr ? expf((to_f32(dr[v]) - qm) * inv_t) * q_inv : (v == x ? 1.f : 0.f);
                    const float r = w / e[v];
                    if (r > best) { best = r; idx = v; }
                }
                for (int o = 16; o; o >>= 1) {
                    const float ob = __shfl_xor_sync(0xffffffffu, best, o);
                    const int oi = __shfl_xor_sync(0xffffffffu, idx, o);
                    if (ob > best || (ob == best && oi < idx)) { best = ob; idx = oi; }
                }
                __syncthreads();
                if ((tid & 31) == 0) { bv[tid >> 5] = best; bi[tid >> 5] = idx; }
                __syncthreads();
                best = bv[0];
                idx = bi[0];
                for (int w = 1; w < 16; ++w)
                    if (bv[w] > best || (bv[w] == best && bi[w] < idx)) { best = bv[w]; idx = bi[w]; }
                if (best > 0.f) next = idx;
            }
        } else if (w_inv > 0.f) {
            next = at;
        }
    }
    if (tid == 0) {
        out[n_acc] = next;
        for (int j = n_acc + 1; j <= a.max_drafts; ++j) out[j] = -1;
        a.count[s] = sane ? n_acc + 1 : 0;
    }
}

}  // namespace exl3

using namespace exl3;

static int check_verify(int rows, int seqs, int n)
{
    return seqs < 1 || rows < seqs || n < 1 ? EXL3_E_SHAPE : EXL3_OK;
}

extern "C" int exl3_verify_workspace(int rows, int seqs, int n, size_t* bytes)
{
    if (!bytes) return EXL3_E_NULL;
    if (int e = check_verify(rows, seqs, n)) return e;
    *bytes = 0;
    return EXL3_OK;
}

extern "C" int exl3_verify_drafts(const void* target, long long target_ld, const void* draft, long long draft_ld, int dtype,
                                  int rows, int seqs, int n, const long long* draft_tokens, const int32_t* cu_rows,
                                  const float* temperature, const float* u, const float* noise, long long noise_ld,
                                  int max_drafts, long long* tokens_out, int32_t* count, float* accept_prob,
                                  void* workspace, size_t workspace_bytes, void* stream)
{
    if (int e = check_verify(rows, seqs, n)) return e;
    if (!target || !cu_rows || !noise || !tokens_out || !count) return EXL3_E_NULL;
    if (rows > seqs && (!draft_tokens || !u || !accept_prob)) return EXL3_E_NULL;
    if (target_ld < n || (draft && draft_ld < n) || noise_ld < n || max_drafts < 0) return EXL3_E_SHAPE;
    const int esz = dtype == EXL3_F32 ? 4 : 2;
    if (dtype != EXL3_F16 && dtype != EXL3_BF16 && dtype != EXL3_F32) return EXL3_E_DTYPE;
    if (!aligned(target, esz) || !aligned(draft, esz) || !aligned(noise, 4) || !aligned(u, 4) || !aligned(cu_rows, 4) ||
        !aligned(draft_tokens, 8) || !aligned(tokens_out, 8) || !aligned(count, 4) || !aligned(accept_prob, 4) ||
        !aligned(temperature, 4))
        return EXL3_E_ALIGN;
    if (int e = check_device()) return e;
    VerifyArgs a{};
    a.target = target; a.draft = draft;
    a.target_ld = target_ld; a.draft_ld = draft_ld; a.noise_ld = noise_ld;
    a.tokens = draft_tokens; a.cu_rows = cu_rows; a.temperature = temperature; a.u = u; a.noise = noise;
    a.out = tokens_out; a.count = count; a.prob = accept_prob;
    a.rows = rows; a.seqs = seqs; a.n = n; a.max_drafts = max_drafts;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const dim3 grid(seqs), block(kVerifyThreads);
    switch (dtype) {
    case EXL3_F16: return launch_pdl(verify_kernel<__half>, grid, block, 0, s, a);
    case EXL3_BF16: return launch_pdl(verify_kernel<__nv_bfloat16>, grid, block, 0, s, a);
    default: return launch_pdl(verify_kernel<float>, grid, block, 0, s, a);
    }
}
