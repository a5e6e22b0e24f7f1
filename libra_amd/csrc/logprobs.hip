// Log probabilities of given tokens, entropy and the largest alternatives of a row of logits z[V] (bf16 or fp32), and the gradient.
//   m = max z,  e_v = exp(z_v - m),  r = sum of e over every column but ONE that attains m (so r is exact to fp32 relative precision
//   also where one token is nearly certain),  log p_v = (z_v - m) - log1p(r),  H = log1p(r) - sum e_v (z_v - m) / (1 + r)
// (both terms of H are >= 0: no cancellation).  A row whose maximum is +inf (a forced token) is shared by its n infinite columns:
// log p = -log n there, -inf elsewhere, H = log n - the formulas as they stand with z_v - m := 0 where z_v = m.  A row of nothing but
// -inf answers log p = -inf, H = 0.  A row that holds a NaN answers NaN.
//   dz_v = sum_i g_i ([v = t_i] - p_v) - g_H p_v (log p_v + H),  and 1 - p_v at v = t_i as -expm1(log p_v).
// HBM-bound: V elements in (forward), V in and V out (backward) a row.
#include "hip_common.hpp"
#include "../../include/libra_hip.h"

namespace libra {

template <typename T> struct LpElem;
template <> struct LpElem<bf16_t> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float get(bf16_t v) { return bf2f(v); }
    static __device__ __forceinline__ bf16_t put(float v) { return f2bf(v); }
    static __device__ __forceinline__ void unpack(const u32x4 q, float* f) { unpack8(q, f); }
    static __device__ __forceinline__ u32x4 pack(const float* f) { return pack8(f); }
};
template <> struct LpElem<float> {
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
    static __device__ __forceinline__ void unpack(const u32x4 q, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { const unsigned u = q[i]; f[i] = __uint_as_float(u); }
    }
    static __device__ __forceinline__ u32x4 pack(const float* f) {
        u32x4 q;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = __float_as_uint(f[i]);
        return q;
    }
};
// A row is read in 16-byte pieces at 16-byte addresses: piece c holds the columns [c VEC - off, (c + 1) VEC - off), off = how many
// elements the row begins behind an aligned address (any V and any row stride).  Columns outside the row come as `fill`.
template <typename T>
__device__ __forceinline__ int lp_off(const T* row) { return (int)(((uintptr_t)row & 15) / sizeof(T)); }
template <typename T>
__device__ __forceinline__ void lp_load(const T* row, int off, int V, int c, float fill, float* f) {
    constexpr int VEC = LpElem<T>::VEC;
    const int v0 = c * VEC - off;
    if (v0 >= 0 && v0 + VEC <= V) {
        LpElem<T>::unpack(*(const u32x4*)(row + v0), f);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = (v0 + e >= 0 && v0 + e < V) ? LpElem<T>::get(row[v0 + e]) : fill;
    }
}
// order of the alternatives: larger value first, then smaller column; NaN behind everything
__device__ __forceinline__ unsigned long long lp_key(float z, int v) {
    unsigned u = __float_as_uint(z);
    u = z != z ? 0u : (u == 0x80000000u ? 0x80000000u : (u & 0x80000000u ? ~u : u | 0x80000000u));    // (-0 = +0)
    return ((unsigned long long)u << 32) | (unsigned)~v;
}
__device__ __forceinline__ float lp_diff(float z, float m) { return z == m ? 0.f : z - m; }

constexpr int LP_THREADS = 256;
template <typename F>
__device__ __forceinline__ float lp_block(float x, F op, float* red) {
    for (int o = 32; o > 0; o >>= 1) x = op(x, __shfl_xor(x, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    return op(op(red[0], red[1]), op(red[2], red[3]));
}

struct LogprobArgs {
    const void* z; long ldz; int V; long rows;
    const long long* targets; int T; long long tsub;
    float* logprobs;                                  // [T, rows]
    float* stats;                                     // [3, rows]: max, log1p(r), entropy
    int top; long long* top_ids; float* top_lp;       // [rows, top]
};

template <typename T>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(const LogprobArgs p) {
    constexpr int VEC = LpElem<T>::VEC;
    __shared__ float red[4];
    __shared__ unsigned long long redk[4];
    const long row = blockIdx.x;
    const T* z = (const T*)p.z + row * p.ldz;
    const int off = lp_off(z), nc = (p.V + off + VEC - 1) / VEC;
    const int tid = threadIdx.x;
    auto maxf = [](float a, float b) { return fmaxf(a, b); };
    auto addf = [](float a, float b) { return a + b; };
    float m = -INFINITY;
    bool nan = false;
    for (int c = tid; c < nc; c += LP_THREADS) {
        float f[VEC];
        lp_load(z, off, p.V, c, -INFINITY, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { nan |= f[e] != f[e]; m = fmaxf(m, f[e]); }
    }
    m = lp_block(m, maxf, red);
    nan = __syncthreads_or(nan);
    // which column is the one left out of r: the first that attains m
    int first = 0x7fffffff;
    float s = 0.f, t = 0.f;
    for (int c = tid; c < nc; c += LP_THREADS) {
        float f[VEC];
        lp_load(z, off, p.V, c, -INFINITY, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int v = c * VEC - off + e;
            if (v < 0 || v >= p.V) continue;
            const float d = lp_diff(f[e], m);
            if (d == 0.f) { if (v < first) first = v; }
            const float ex = __expf(d);
            s += d == 0.f ? 0.f : ex;
            t += ex > 0.f ? ex * d : 0.f;
        }
    }
    int equal = 0;                                     // columns that attain m beyond the first
    for (int c = tid; c < nc; c += LP_THREADS) {
        float f[VEC];
        lp_load(z, off, p.V, c, -INFINITY, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { const int v = c * VEC - off + e; equal += (v >= 0 && v < p.V && f[e] == m) ? 1 : 0; }
    }
    s = lp_block(s, addf, red);
    t = lp_block(t, addf, red);
    const float n_eq = lp_block((float)equal, addf, red);
    const bool empty = m == -INFINITY;
    const float r = s + (n_eq - 1.f);
    const float lsum = empty ? 0.f : log1pf(r);
    const float ent = empty ? 0.f : lsum - t / (1.f + r);
    const float qnan = __uint_as_float(0x7fc00000u);
    if (tid == 0) {
        p.stats[row] = nan ? qnan : m;
        p.stats[p.rows + row] = nan ? qnan : lsum;
        p.stats[2 * p.rows + row] = nan ? qnan : ent;
    }
    auto logp = [&](float zv) { return nan ? qnan : empty ? -INFINITY : lp_diff(zv, m) - lsum; };
    for (int i = tid; i < p.T; i += LP_THREADS) {
        const long long tg = p.targets[i * p.rows + row], v = tg - p.tsub;
        p.logprobs[i * p.rows + row] = tg < 0 ? 0.f : (v >= 0 && v < p.V) ? logp(LpElem<T>::get(z[v])) : nan ? qnan : -INFINITY;
    }
    unsigned long long last = ~0ull;                   // alternatives one by one: the largest key below the previous one
    for (int k = 0; k < p.top; ++k) {
        unsigned long long best = 0;
        for (int c = tid; c < nc; c += LP_THREADS) {
            float f[VEC];
            lp_load(z, off, p.V, c, -INFINITY, f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int v = c * VEC - off + e;
                if (v < 0 || v >= p.V) continue;
                const unsigned long long key = lp_key(f[e], v);
                if (key < last && key > best) best = key;
            }
        }
        for (int o = 32; o > 0; o >>= 1) { const unsigned long long x = __shfl_xor(best, o, 64); best = x > best ? x : best; }
        __syncthreads();
        if ((tid & 63) == 0) redk[tid >> 6] = best;
        __syncthreads();
        for (int i = 0; i < 4; ++i) best = redk[i] > best ? redk[i] : best;
        last = best;
        if (tid == 0) {
            const int v = (int)~(unsigned)best;
            p.top_ids[row * p.top + k] = v + p.tsub;
            p.top_lp[row * p.top + k] = logp(LpElem<T>::get(z[v]));
        }
    }
}

struct LogprobBwdArgs {
    const void* z; long ldz; int V; long rows;
    const long long* targets; int T; long long tsub;
    const float* stats; const float* g_lp; const float* g_ent;      // [3, rows]; [T, rows] or null; [rows] or null
    void* dz; long lddz;
};

template <typename T>
__global__ __launch_bounds__(LP_THREADS) void logprobs_bwd_kernel(const LogprobBwdArgs p) {
    constexpr int VEC = LpElem<T>::VEC;
    const long row = blockIdx.x;
    const T* z = (const T*)p.z + row * p.ldz;
    T* dz = (T*)p.dz + row * p.lddz;
    const int off = lp_off(z), nc = (p.V + off + VEC - 1) / VEC;
    const bool same = lp_off(dz) == off;
    const float m = p.stats[row], lsum = p.stats[p.rows + row], ent = p.stats[2 * p.rows + row];
    const bool flat = m == INFINITY || m == -INFINITY;              // a forced row, or one with nothing left: no gradient
    const float gh = p.g_ent ? p.g_ent[row] : 0.f;
    float g = 0.f;
    for (int i = 0; i < p.T; ++i) if (p.g_lp && p.targets[i * p.rows + row] >= 0) g += p.g_lp[i * p.rows + row];
    for (int c = threadIdx.x; c < nc; c += LP_THREADS) {
        float f[VEC];
        lp_load(z, off, p.V, c, -INFINITY, f);
        const int v0 = c * VEC - off;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float lp = f[e] - m - lsum, pr = __expf(lp);
            f[e] = flat ? 0.f : -pr * g - (pr > 0.f ? pr * (lp + ent) * gh : 0.f);
        }
        for (int i = 0; i < p.T; ++i) {
            if (!p.g_lp) break;
            const long long tg = p.targets[i * p.rows + row], v = tg - p.tsub;
            if (tg < 0 || v < v0 || v >= v0 + VEC || v < 0 || v >= p.V || flat) continue;
            // a given token's column anew, with its share as -expm1(log p): 1 - p taken as a difference would lose a sure token's gradient
            const float lp = LpElem<T>::get(z[v]) - m - lsum, pr = __expf(lp), one = -expm1f(lp);
            float sum = -(pr > 0.f ? pr * (lp + ent) * gh : 0.f);
            for (int k = 0; k < p.T; ++k) {
                const long long tk = p.targets[k * p.rows + row];
                if (tk >= 0) sum += p.g_lp[k * p.rows + row] * (tk == tg ? one : -pr);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = (v0 + e == v) ? sum : f[e];
        }
        if (same && v0 >= 0 && v0 + VEC <= p.V) {
            *(u32x4*)(dz + v0) = LpElem<T>::pack(f);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) if (v0 + e >= 0 && v0 + e < p.V) dz[v0 + e] = LpElem<T>::put(f[e]);
        }
    }
}

}  // namespace libra

using namespace libra;

static int lp_check(const void* z, int64_t ldz, int64_t rows, int64_t V, int f32, const int64_t* targets, int64_t n_targets) {
    if (rows < 0 || rows > 0x7fffffffL || V <= 0 || V > 0x7ffffff0L || ldz < V || n_targets < 0 || n_targets > 64) return LIBRA_ERR_SHAPE;
    if (!z || ((uintptr_t)z % (f32 ? 4 : 2))) return LIBRA_ERR_ALIGN;
    if (n_targets && !targets) return LIBRA_ERR_ALIGN;
    return LIBRA_OK;
}

extern "C" int libra_token_logprobs(const void* logits, int64_t ldz, int64_t rows, int64_t V, int f32, const int64_t* targets,
                                    int64_t n_targets, int64_t target_sub, float* logprobs, float* stats, int64_t top, int64_t* top_ids,
                                    float* top_logprobs, void* stream) {
    if (rows == 0) return LIBRA_OK;
    const int rc = lp_check(logits, ldz, rows, V, f32, targets, n_targets);
    if (rc != LIBRA_OK) return rc;
    if (top < 0 || top > 64 || top > V) return LIBRA_ERR_SHAPE;
    if (!stats || (n_targets && !logprobs) || (top && (!top_ids || !top_logprobs))) return LIBRA_ERR_ALIGN;
    LogprobArgs a{logits, (long)ldz, (int)V, (long)rows, (const long long*)targets, (int)n_targets, (long long)target_sub, logprobs, stats,
                  (int)top, (long long*)top_ids, top_logprobs};
    if (f32) hipLaunchKernelGGL(logprobs_kernel<float>, dim3((unsigned)rows), dim3(LP_THREADS), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(logprobs_kernel<bf16_t>, dim3((unsigned)rows), dim3(LP_THREADS), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? LIBRA_OK : LIBRA_ERR_LAUNCH;
}

extern "C" int libra_token_logprobs_bwd(const void* logits, int64_t ldz, int64_t rows, int64_t V, int f32, const int64_t* targets,
                                        int64_t n_targets, int64_t target_sub, const float* stats, const float* g_logprobs,
                                        const float* g_entropy, void* dlogits, int64_t lddz, void* stream) {
    if (rows == 0) return LIBRA_OK;
    const int rc = lp_check(logits, ldz, rows, V, f32, targets, n_targets);
    if (rc != LIBRA_OK) return rc;
    if (lddz < V) return LIBRA_ERR_SHAPE;
    if (!stats || !dlogits || ((uintptr_t)dlogits % (f32 ? 4 : 2)) || (g_logprobs && !targets)) return LIBRA_ERR_ALIGN;
    LogprobBwdArgs a{logits, (long)ldz, (int)V, (long)rows, (const long long*)targets, (int)n_targets, (long long)target_sub, stats,
                     g_logprobs, g_entropy, dlogits, (long)lddz};
    if (f32) hipLaunchKernelGGL(logprobs_bwd_kernel<float>, dim3((unsigned)rows), dim3(LP_THREADS), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(logprobs_bwd_kernel<bf16_t>, dim3((unsigned)rows), dim3(LP_THREADS), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? LIBRA_OK : LIBRA_ERR_LAUNCH;
}
