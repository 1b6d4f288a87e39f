// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
//   p = softmax(target / T), q = softmax(draft / T); a_i = min(1, p_i(x_i) / q_i(x_i)), drafts accepted while u_i < a_i, then
//   one draw from w = max(0, p - q) (after a rejection) or w = p, as the first largest w(v) / noise(v).
//
// Two launches, both bound by reading logits (or, for a sequence or two, by latency):
//   stats    a CTA per chunk of a row keeps it in registers: maximum, sum of exp, and for T = 0 the first column of the
//            maximum. Rows do not wait for each other and every logit is read once.
//   decide   a cluster of 8 CTAs per sequence: each works out the acceptances from the statistics (the same answer in all of
//            them), then they share the columns of the one row that the next token is drawn from and reduce (value, first
//            column) through distributed shared memory.
// A draw by inverting the cumulative distribution would need a prefix sum over the vocabulary and give another token for
// another order of summation; the race depends on each w alone.
//
// 64 sequences of up to 8 rows with as many draft rows but one, 151,936 columns of bf16, 190 MB: 52 us (3.6 TB/s, 0.56 of a
// measured copy): about 31 for the statistics, near a copy's rate, the rest for a race that cannot begin before all of a
// sequence's statistics are known. One sequence of 4 rows: 13.3 us, two launches and two rounds of loads.
#include <cuda_runtime.h>

#include <cfloat>
#include <type_traits>

#include "exl3_b200.h"
#include "exl3_common.cuh"
#include "exl3_host.h"
#include "exl3_paged.cuh"
#include "exl3_paged_math.cuh"
#include "exl3_tc.cuh"

namespace exl3 {

// log2(e) / T; T far outside the range of logits counts as one at its end, so that the factor is neither 0 nor infinite.
__device__ __forceinline__ float exponent_scale(float temperature, bool greedy)
{
    return 1.4426950408889634f / (greedy ? 1.f : fminf(fmaxf(temperature, 1e-30f), 1e30f));
}
constexpr int kStatThreads = 128, kStatWarps = kStatThreads / 32;
constexpr int kStatVecs = 8;                          // 16-byte vectors a thread keeps in registers
constexpr int kDecideWarps = 16;                      // most of a CTA
constexpr int kVerifyCluster = 8;

struct VerifyArgs {
    const void *target, *draft;
    long long target_ld, draft_ld, noise_ld;
    const long long* tokens;
    const int32_t* cu_rows;
    const float *temperature, *u, *noise;
    long long* out;
    int32_t* count;
    float* prob;
    float4* stats;                                    // [target rows, then draft rows][chunks] (max, sum, first column of max)
    int rows, seqs, n, max_drafts, chunks;
};

// (value, column) of the larger value, of the first column among equals.
__device__ __forceinline__ void take_first(float& v, int& i, float ov, int oi)
{
    if (ov > v || (ov == v && oi < i)) {
        v = ov;
        i = oi;
    }
}

// ------------------------------------------------------------------------------ statistics
template <typename T> __device__ __forceinline__ uint32_t lowest_word();       // -inf in each place of a word
template <> __device__ __forceinline__ uint32_t lowest_word<__half>() { return 0xFC00FC00u; }
template <> __device__ __forceinline__ uint32_t lowest_word<__nv_bfloat16>() { return 0xFF80FF80u; }
template <> __device__ __forceinline__ uint32_t lowest_word<float>() { return 0xFF800000u; }

// Value i of a word of the row (two of a 16-bit type).
template <typename T>
__device__ __forceinline__ float word_value(uint32_t w, int i)
{
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i ? w & 0xFFFF0000u : w << 16);
    else return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w)));
}

// Larger values of two words place by place; of a number and a NaN, the number.
template <typename T>
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b)
{
    uint32_t r;
    if constexpr (sizeof(T) == 4) r = __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Small CTAs, so that some load while others reduce; a thread keeps its columns as they are stored, which leaves registers for
// 8 CTAs an SM with 128 bytes a thread in flight (6 without the few spilled bytes: 54.0 us against 52.6 for the 190 MB above;
// columns unpacked to fp32, 5 CTAs: 58.7). The row's columns from its first 16-byte boundary on go to the chunks as
// whole vectors; the few before it are chunk 0's, the last vector may be partial.
template <typename T>
__global__ void __launch_bounds__(kStatThreads, 8) verify_stats_kernel(const VerifyArgs a)
{
    constexpr int VEC = 16 / sizeof(T), PW = 4 / sizeof(T), N = kStatVecs;     // columns of a vector, of a word; vectors
    __shared__ float sv[kStatWarps];
    __shared__ int si[kStatWarps];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / a.chunks, chunk = blockIdx.x - r * a.chunks;
    const bool is_draft = r >= a.rows;
    const T* x = is_draft ? static_cast<const T*>(a.draft) + (r - a.rows) * a.draft_ld
                          : static_cast<const T*>(a.target) + r * a.target_ld;
    const int head = min(a.n, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    const int first = head + chunk * (kStatThreads * N * VEC) + tid * VEC;
    // the decision writes those of the drafts that a sequence judges; a draft that none does (a cu_rows that is no list) has 0
    if (tid == 0 && chunk == 0 && r < a.rows - a.seqs) a.prob[r] = 0.f;
    const uint32_t none = lowest_word<T>();
    uint4 w[N];
    auto fetch = [&]() {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int at = first + k * kStatThreads * VEC;
            w[k] = at + VEC <= a.n ? *reinterpret_cast<const uint4*>(x + at) : make_uint4(none, none, none, none);
        }
    };
    // a target row's logits are on their way while its temperature is looked up
    if (!is_draft) fetch();
    float temp = 1.f;
    if (a.temperature)
        temp = a.temperature[is_draft ? seq_of_row<1>(a.cu_rows, a.seqs, r - a.rows, lane) : seq_of_row(a.cu_rows, a.seqs, r, lane)];
    const bool greedy = !(temp > 0.f);
    if (is_draft) {
        if (greedy) return;                           // q is one-hot: the row is not looked at
        fetch();
    }
    if (head + (chunk + 1) * (kStatThreads * N * VEC) > a.n) {         // the row ends in this chunk: its last vector
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int at = first + k * kStatThreads * VEC;
            if (at < a.n && at + VEC > a.n) {
                uint32_t q[4] = {none, none, none, none};
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (at + i < a.n) {
                        if constexpr (PW == 1) q[i] = reinterpret_cast<const uint32_t*>(x)[at + i];
                        else q[i / 2] = __byte_perm(q[i / 2], reinterpret_cast<const unsigned short*>(x)[at + i], i & 1 ? 0x5410 : 0x3254);
                    }
                w[k] = make_uint4(q[0], q[1], q[2], q[3]);
            }
        }
    }
    const float xh = chunk == 0 && tid < head ? to_f32(x[tid]) : -INFINITY;
    uint32_t most = none;
#pragma unroll
    for (int k = 0; k < N; ++k) most = word_max<T>(most, word_max<T>(word_max<T>(w[k].x, w[k].y), word_max<T>(w[k].z, w[k].w)));
    float m = fmaxf(xh, word_value<T>(most, 0));
    if (PW == 2) m = fmaxf(m, word_value<T>(most, 1));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) sv[warp] = m;
    __syncthreads();
    m = sv[lane & (kStatWarps - 1)];
#pragma unroll
    for (int o = kStatWarps / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // relative to the largest finite number where the maximum is +inf: the sum is inf then, and NaN only where a logit is
    const float base = m == -INFINITY ? 0.f : fminf(m, FLT_MAX), c = exponent_scale(temp, greedy);
    // the maximum is taken off before scaling: the type's lowest value times 1 / T would overflow
    const uint64_t c2 = f2(c, c), zero = f2(0.f, 0.f), off = f2(-base, -base);
    uint64_t s2 = f2(ex2((xh - base) * c), 0.f);
    auto add2 = [&](float u, float v) {
        float e0, e1;
        f2_get(f2_fma(f2_add(f2(u, v), off), c2, zero), e0, e1);
        s2 = f2_add(s2, f2(ex2(e0), ex2(e1)));
    };
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t q[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
        for (int i = 0; i < 4; i += 3 - PW)
            if (PW == 2) add2(word_value<T>(q[i], 0), word_value<T>(q[i], 1));
            else add2(word_value<T>(q[i], 0), word_value<T>(q[(i + 1) & 3], 0));
    }
    float s0, s1;
    f2_get(s2, s0, s1);
    const float s = warp_sum(s0 + s1);
    int at = 0x7fffffff;
    if (greedy) {
#pragma unroll
        for (int k = N - 1; k >= 0; --k) {
            const uint32_t q[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
            for (int i = VEC - 1; i >= 0; --i)
                if (word_value<T>(q[i / PW], i % PW) == m) at = first + k * kStatThreads * VEC + i;
        }
        if (chunk == 0 && tid < head && xh == m) at = tid;
        at = __reduce_min_sync(0xffffffffu, at);
    }
    __syncthreads();
    if (lane == 0) {
        sv[warp] = s;
        si[warp] = at;
    }
    __syncthreads();
    if (tid == 0) {
        float sum = 0.f;
        int col = 0x7fffffff;
        for (int k = 0; k < kStatWarps; ++k) {
            sum += sv[k];
            col = min(col, si[k]);
        }
        // at T = 0 the sum only tells whether the row has an answer: a +inf is a maximum like any other
        a.stats[blockIdx.x] = make_float4(m, greedy && sum > 0.f ? 1.f : sum, __int_as_float(col), 0.f);
    }
}

// ------------------------------------------------------------------------------ decision
// What the race needs of a row: exp2((x - m) c) * inv is its probability.
struct RowStat {
    float m, inv;
    int first;                                        // column of the maximum
};

// Two sums of exp relative to their own maxima, relative to the larger one. A part of -inf alone has sum 0 (or NaN, which
// stays: its row has no probabilities); one whose maximum is the larger, +inf too, passes as it is.
__device__ __forceinline__ float joined(float s0, float m0, float s1, float m1, float now, float c)
{
    auto rel = [&](float s, float m) { return m == -INFINITY || m == now ? s : s * ex2((m - now) * c); };
    return rel(s0, m0) + rel(s1, m1);
}

struct PartStat {                                     // of some of a row's chunks
    float m = -INFINITY, s = 0.f;
    int first = 0x7fffffff;
    __device__ __forceinline__ void join(float om, float os, int of, float c)
    {
        s = joined(s, m, os, om, fmaxf(m, om), c);
        take_first(m, first, om, of);
    }
};

// Statistics of one or (b >= 0) two rows from their chunks', by a warp; both rows' chunks are loaded together.
__device__ __forceinline__ void row_stats(const VerifyArgs& a, long long ra, long long rb, float c, int lane, RowStat& outa, RowStat& outb)
{
    PartStat p[2];
    for (int k0 = 0; k0 < a.chunks; k0 += 64) {
        float4 w[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int k = k0 + 32 * j + lane;
                const long long row = i ? rb : ra;
                w[i][j] = row >= 0 && k < a.chunks ? __ldcg(a.stats + row * a.chunks + k)
                                                   : make_float4(-INFINITY, 0.f, __int_as_float(0x7fffffff), 0.f);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) p[i].join(w[i][j].x, w[i][j].y, __float_as_int(w[i][j].z), c);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            p[i].join(__shfl_xor_sync(0xffffffffu, p[i].m, o), __shfl_xor_sync(0xffffffffu, p[i].s, o),
                      __shfl_xor_sync(0xffffffffu, p[i].first, o), c);
        RowStat& r = i ? outb : outa;
        r.m = p[i].m == -INFINITY ? 0.f : p[i].m;
        r.inv = p[i].s > 0.f ? 1.f / p[i].s : 0.f;
        r.first = p[i].first;
    }
}

struct Verdict {                                      // of one row, by the warp that looked at it
    RowStat p, q;
    float prob;
    long long token;
    int stands;                                       // its draft was accepted
};

template <typename T>
__global__ void __launch_bounds__(32 * kDecideWarps) verify_decide_kernel(const VerifyArgs a)
{
    constexpr int VEC = 16 / sizeof(T);
    __shared__ Verdict row_s[kDecideWarps];
    __shared__ float bv[kDecideWarps];
    __shared__ int bi[kDecideWarps];
    __shared__ float2 mine[2];                        // this CTA's winner of a pass (value, column)
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthr = blockDim.x, nwarp = nthr >> 5;
    const int rank = (int)cluster_rank();
    const int s = blockIdx.x / kVerifyCluster;
    const int lo = a.cu_rows[s], hi = a.cu_rows[s + 1];
    const bool sane = lo >= s && hi > lo && hi <= a.rows && hi - s - 1 <= a.rows - a.seqs;
    const float temp = a.temperature ? a.temperature[s] : 1.f;
    const bool greedy = !(temp > 0.f);
    const float c = exponent_scale(temp, greedy);
    const int judged = sane ? hi - lo - 1 : 0;        // drafts of this sequence
    const int limit = min(judged, a.max_drafts);

    // the noise is not known to any cache yet, and its columns do not depend on the verdict
    if (sane && !greedy)
        for (int v = (rank * nthr + tid) * 32; v < a.n; v += nthr * kVerifyCluster * 32)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(a.noise + s * a.noise_ld + v));

    // rows in order, a warp each, until one does not stand (the first CTA goes on: accept_prob is every draft's)
    int n_acc = -1;
    Verdict at{};
    for (int j0 = 0; sane && j0 <= judged; j0 += nwarp) {
        const int j = j0 + warp;
        if (j <= judged) {
            const T* tr = static_cast<const T*>(a.target) + (lo + j) * a.target_ld;
            Verdict v{};
            const bool has = j < judged, two = has && a.draft && !greedy;
            const int i = lo + j - s;
            float u = 0.f, xt = 0.f, xd = 0.f;
            if (has) {
                v.token = a.tokens[i];
                u = a.u[i];
            }
            const bool in = has && v.token >= 0 && v.token < a.n;
            if (in) {
                xt = to_f32(tr[v.token]);
                if (two) xd = to_f32((static_cast<const T*>(a.draft) + i * a.draft_ld)[v.token]);
            }
            row_stats(a, lo + j, two ? (long long)a.rows + i : -1, c, lane, v.p, v.q);
            if (has) {
                float p = 0.f, q = 1.f;
                if (greedy) {
                    p = in && v.token == v.p.first && v.p.inv > 0.f ? 1.f : 0.f;
                } else {
                    if (in && v.p.inv > 0.f) p = ex2((xt - v.p.m) * c) * v.p.inv;       // a NaN logit is in a row without probabilities
                    if (two) q = in ? ex2((xd - v.q.m) * c) * v.q.inv : 0.f;
                }
                v.prob = q > 0.f ? fminf(p / q, 1.f) : (p > 0.f ? 1.f : 0.f);
                v.stands = j < limit && u < v.prob;
                if (rank == 0 && lane == 0) a.prob[i] = v.prob;
            }
            if (lane == 0) row_s[warp] = v;
        }
        __syncthreads();
        if (n_acc < 0)
            for (int k = 0; k < nwarp && j0 + k <= judged; ++k)
                if (!row_s[k].stands) {
                    n_acc = j0 + k;
                    at = row_s[k];
                    break;
                }
        __syncthreads();
        if (n_acc >= 0 && rank != 0) break;
    }
    const bool rejected = n_acc >= 0 && n_acc < limit;                // the row's own draft was turned down

    long long next = -1;
    if (sane && greedy) {
        if (at.p.inv > 0.f) next = at.p.first;
    } else if (sane) {
        const T* tr = static_cast<const T*>(a.target) + (lo + n_acc) * a.target_ld;
        const T* dr = a.draft && rejected ? static_cast<const T*>(a.draft) + (lo + n_acc - s) * a.draft_ld : nullptr;
        const float* e = a.noise + s * a.noise_ld;
        const bool vec = ((reinterpret_cast<uintptr_t>(tr) | reinterpret_cast<uintptr_t>(dr) | reinterpret_cast<uintptr_t>(e)) & 15) == 0;
        const int threads = nthr * kVerifyCluster, me = rank * nthr + tid;
        const int banned = at.token >= 0 && at.token < a.n ? (int)at.token : -1;
        // Columns of this thread in rising order; MODE 0: w = p, 1: w = p - q, 2: w = p but for the rejected token (one-hot q).
        // Threads, warps and CTAs all compare the rounded quotients w / noise, so the answer is the first column of the largest
        // however the columns are shared out. A thread asks for w >= best * noise first: a quotient that rounds to more than best is
        // more than best, so w is at least the product, rounded too; the division is for the few columns that pass.
        auto race = [&](auto mode, float& best, int& idx) {
            constexpr int MODE = decltype(mode)::value;
            auto take = [&](int v, float w, float nz) {
                const float r = w / nz;
                if (r > best) {
                    best = r;
                    idx = v;
                }
            };
            auto weight = [&](int v, float x, float d) {
                // products rounded before the difference: where q is p, w is zero
                float w = __fmul_rn(ex2((x - at.p.m) * c), at.p.inv);
                if (MODE == 1) w = __fsub_rn(w, __fmul_rn(ex2((d - at.q.m) * c), at.q.inv));
                if (MODE == 2 && v == banned) w = 0.f;
                return w;
            };
            const int whole = vec ? a.n / VEC * VEC : 0;
#pragma unroll 1
            for (int v = me * VEC; v < whole; v += threads * VEC) {
                const uint4 xr = *reinterpret_cast<const uint4*>(tr + v);
                const uint4 dx = MODE == 1 ? *reinterpret_cast<const uint4*>(dr + v) : make_uint4(0, 0, 0, 0);
                float nz[VEC], w[VEC];
#pragma unroll
                for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(nz + i) = *reinterpret_cast<const float4*>(e + v + i);
                const T* xe = reinterpret_cast<const T*>(&xr);
                const T* de = reinterpret_cast<const T*>(&dx);
                bool any = false;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    w[i] = weight(v + i, to_f32(xe[i]), to_f32(de[i]));
                    any |= w[i] >= best * nz[i];
                }
                if (any) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (w[i] >= best * nz[i]) take(v + i, w[i], nz[i]);
                }
            }
#pragma unroll 4
            for (int v = whole + me; v < a.n; v += threads) {
                const float w = weight(v, to_f32(tr[v]), MODE == 1 ? to_f32(dr[v]) : 0.f), nz = e[v];
                if (w >= best * nz) take(v, w, nz);
            }
        };
        // first the residual, then (where that is zero everywhere) p itself
        for (int pass = rejected ? 0 : 1; pass < 2; ++pass) {
            float best = 0.f;
            int idx = 0x7fffffff;
            if (pass == 1) race(std::integral_constant<int, 0>{}, best, idx);
            else if (dr) race(std::integral_constant<int, 1>{}, best, idx);
            else race(std::integral_constant<int, 2>{}, best, idx);
#pragma unroll
            for (int o = 16; o; o >>= 1) take_first(best, idx, __shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, idx, o));
            if (lane == 0) {
                bv[warp] = best;
                bi[warp] = idx;
            }
            __syncthreads();
            if (tid == 0) {
                for (int w = 1; w < nwarp; ++w) take_first(best, idx, bv[w], bi[w]);
                mine[pass] = make_float2(best, __int_as_float(idx));
            }
            cluster_sync_all();
            best = 0.f;
            idx = 0x7fffffff;
            for (int k = 0; k < kVerifyCluster; ++k) {
                float ov;
                int oi;
                const uint32_t from = cluster_addr(&mine[pass], k);
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ov) : "r"(from) : "memory");
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(oi) : "r"(from + 4) : "memory");
                take_first(best, idx, ov, oi);
            }
            if (best > 0.f) {
                next = idx;
                break;
            }
        }
        cluster_sync_all();                           // no CTA leaves while another reads its result
    }
    if (rank == 0) {
        long long* out = a.out + (size_t)s * (a.max_drafts + 1);
        for (int j = tid; j <= a.max_drafts; j += nthr)
            out[j] = j < n_acc ? a.tokens[lo + j - s] : j == n_acc ? next : -1;
        if (tid == 0) a.count[s] = n_acc + 1;
    }
}

static int verify_chunks(int n, int esz)
{
    const int columns = kStatVecs * kStatThreads * (16 / esz);
    return (n + columns - 1) / columns;
}

// Sized for the widest type, so that the query needs no dtype.
static size_t verify_bytes(int rows, int seqs, int n) { return (size_t)(2ll * rows - seqs) * verify_chunks(n, 4) * sizeof(float4); }

template <typename T>
static int launch_verify(const VerifyArgs& a, cudaStream_t s)
{
    const long long ctas = (long long)(a.rows + (a.draft ? a.rows - a.seqs : 0)) * a.chunks;
    if (ctas > 0x7fffffffll) return EXL3_E_SHAPE;
    if (int e = launch_pdl(verify_stats_kernel<T>, dim3((unsigned)ctas), dim3(kStatThreads), 0, s, a)) return e;
    // wide CTAs while every cluster has SMs of its own, then narrower ones so that all are resident at once
    const int threads = a.seqs * kVerifyCluster <= device_sm_count() ? 512 : 256;
    return launch_pdl_cluster(verify_decide_kernel<T>, dim3(a.seqs * kVerifyCluster), dim3(threads), 0, kVerifyCluster, s, a);
}

}  // namespace exl3

using namespace exl3;

static int check_verify(int rows, int seqs, int n)
{
    return seqs < 1 || seqs > (1 << 24) || rows < seqs || rows > (1 << 30) || n < 1 || n > (1 << 30) ? EXL3_E_SHAPE : EXL3_OK;
}

extern "C" int exl3_verify_workspace(int rows, int seqs, int n, size_t* bytes)
{
    if (!bytes) return EXL3_E_NULL;
    if (int e = check_verify(rows, seqs, n)) return e;
    *bytes = verify_bytes(rows, seqs, n);
    return EXL3_OK;
}

extern "C" int exl3_verify_drafts(const void* target, long long target_ld, const void* draft, long long draft_ld, int dtype,
                                  int rows, int seqs, int n, const long long* draft_tokens, const int32_t* cu_rows,
                                  const float* temperature, const float* u, const float* noise, long long noise_ld,
                                  int max_drafts, long long* tokens_out, int32_t* count, float* accept_prob,
                                  void* workspace, size_t workspace_bytes, void* stream)
{
    if (int e = check_verify(rows, seqs, n)) return e;
    if (!target || !cu_rows || !noise || !tokens_out || !count || !workspace) return EXL3_E_NULL;
    if (rows > seqs && (!draft_tokens || !u || !accept_prob)) return EXL3_E_NULL;
    if (target_ld < n || (draft && draft_ld < n) || noise_ld < n || max_drafts < 0) return EXL3_E_SHAPE;
    const int esz = dtype == EXL3_F32 ? 4 : 2;
    if (dtype != EXL3_F16 && dtype != EXL3_BF16 && dtype != EXL3_F32) return EXL3_E_DTYPE;
    if (!aligned(target, esz) || !aligned(draft, esz) || !aligned(noise, 4) || !aligned(u, 4) || !aligned(cu_rows, 4) ||
        !aligned(draft_tokens, 8) || !aligned(tokens_out, 8) || !aligned(count, 4) || !aligned(accept_prob, 4) ||
        !aligned(temperature, 4) || !aligned(workspace, 16))
        return EXL3_E_ALIGN;
    if (int e = check_device()) return e;
    if (workspace_bytes < verify_bytes(rows, seqs, n)) return EXL3_E_WORKSPACE;
    VerifyArgs a{};
    a.target = target; a.draft = draft;
    a.target_ld = target_ld; a.draft_ld = draft_ld; a.noise_ld = noise_ld;
    a.tokens = draft_tokens; a.cu_rows = cu_rows; a.temperature = temperature; a.u = u; a.noise = noise;
    a.out = tokens_out; a.count = count; a.prob = accept_prob;
    a.stats = static_cast<float4*>(workspace);
    a.rows = rows; a.seqs = seqs; a.n = n; a.max_drafts = max_drafts;
    a.chunks = verify_chunks(n, esz);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
    case EXL3_F16: return launch_verify<__half>(a, s);
    case EXL3_BF16: return launch_verify<__nv_bfloat16>(a, s);
    default: return launch_verify<float>(a, s);
    }
}
