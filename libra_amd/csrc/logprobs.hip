// Log probabilities of given tokens, entropy and the largest alternatives of a row of logits z[V] (bf16 or fp32), and the gradient.
//   m = max z,  e_v = exp(z_v - m),  r = sum of e over every column but ONE that attains m (so r has fp32's relative precision also
//   where one token is nearly certain),  log p_v = (z_v - m) - log1p(r),  H = log1p(r) - sum e_v (z_v - m) / (1 + r)
// (both terms of H are >= 0: no cancellation).  A row whose maximum is +inf (a forced token) is shared by its n infinite columns:
// log p = -log n there, -inf elsewhere, H = log n - the formulas as they stand with z_v - m := 0 where z_v = m.  A row of nothing but
// -inf answers log p = -inf, H = 0.  A row that holds a NaN answers NaN.
//   dz_v = sum_i g_i ([v = t_i] - p_v) - g_H p_v (log p_v + H),  and 1 - p_v at v = t_i as -expm1(log p_v).
// HBM-bound where there are many large rows: V elements in (forward), V in and V out (backward) a row.  Measured, bf16: 8188 x 32000 in
// 126 us (4.2 TB/s, VALU 64 % busy) and 189 us (5.5 TB/s); 16 x 32514 with 20 alternatives in 10 us (latency of one row's phases, 5
// without alternatives: threshold, listing and ranking wait for each other).  Short rows are bound by issue, not memory: 9248 x 514 in 8.1 +
// 8.6 us for 9.5 and 19 MB.  A wave a row: 280 VALU instructions, of which the 9 columns a lane take some 95 (10.4 a column in long rows) -
// the rest, two wave-wide reductions, log1p, statistics and targets, is paid by 64 lanes for one row - and 9248 waves are more than
// the chip holds at a time (8192, 8 a SIMD), so a second, nearly empty generation follows.
#include <algorithm>
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
    static __device__ __forceinline__ u32x4 pack_all(float v) { const unsigned w = pack2bf(v, v); return u32x4{w, w, w, w}; }
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
    static __device__ __forceinline__ u32x4 pack_all(float v) { const unsigned w = __float_as_uint(v); return u32x4{w, w, w, w}; }
};
// A row is read in 16-byte pieces, piece c = the columns [c VEC, (c + 1) VEC), wherever the row begins (any V, any row stride: the
// hardware loads 16 bytes at any address of the element's alignment); the fewer than VEC columns behind the last whole piece are
// taken one a thread.  Nothing outside the row is read.
template <typename T>
__device__ __forceinline__ u32x4 lp_whole(const T* at) {
    u32x4 q;
    __builtin_memcpy(&q, at, 16);
    return q;
}
template <typename T>
__device__ __forceinline__ void lp_load(const T* row, int V, int c, float* f) {
    constexpr int VEC = LpElem<T>::VEC;
    if ((c + 1) * VEC <= V) {
        LpElem<T>::unpack(lp_whole(row + c * VEC), f);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = c * VEC + e < V ? LpElem<T>::get(row[c * VEC + e]) : -INFINITY;
    }
}
// order of the alternatives: larger value first, then smaller column; NaN behind everything
__device__ __forceinline__ unsigned long long lp_key(float z, int v) {
    unsigned u = __float_as_uint(z);
    u = z != z ? 0u : (u == 0x80000000u ? 0x80000000u : (u & 0x80000000u ? ~u : u | 0x80000000u));    // (-0 = +0)
    return ((unsigned long long)u << 32) | (unsigned)~v;
}
__device__ __forceinline__ float lp_diff(float z, float m) { return z == m ? 0.f : z - m; }

// the value part of lp_key
__device__ __forceinline__ unsigned lp_sort(float z) { return (unsigned)(lp_key(z, 0) >> 32); }

template <int N>
__device__ __forceinline__ float row_ror_fmax(float x) {
    const unsigned r = (unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x120 + N, 0xf, 0xf, false);
    return fmaxf(x, __uint_as_float(r));
}
// wave-wide maximum / sum: four DPP row rotations and two lane swaps, no trip through LDS
__device__ __forceinline__ float lp_wave_max(float x) {
    x = row_ror_fmax<1>(row_ror_fmax<2>(row_ror_fmax<4>(row_ror_fmax<8>(x))));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return half_swap_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float lp_wave_sum(float x) {
    x = row_ror_add<1>(row_ror_add<2>(row_ror_add<4>(row_ror_add<8>(x))));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return half_swap_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

struct LogprobArgs {
    const void* z; long ldz; int V; long rows, row0;  // this launch's rows begin at row0
    const long long* targets; int T; long long tsub;
    float* logprobs;                                  // [T, rows]
    float* stats;                                     // [3, rows]: max, log1p(r), entropy
    int top; long long* top_ids; float* top_lp;       // [rows, top]
};

// A row held in registers: NT threads x NCH pieces of 16 bytes (piece i of thread t = row piece i NT + t), one workgroup a row - the
// row is read ONCE, its maximum, its sums and its alternatives all come from registers.  (8 x 512 threads for a row of 32 k columns:
// 126 us at 8188 rows against 143 us with 4 x 1024 and 129 us with 16 x 256.)
// Alternatives (top <= 64): tau = the largest threshold that at least `top` of the threads' maxima reach (binary search over the bits
// by one wave, ended early once no more than max(top, 24) do), so at least `top` columns reach it, and only those few threads' columns
// can: they lay their pieces into LDS, what reaches tau is listed and ranked by counting.  Where the search ends with more threads at
// tau (rows with masked columns, constant rows: ties), the listed ones are those above tau (of fewer than `top` threads) and the rest
// are the first columns that equal it, found by a prefix count in column order.
template <typename T, int NT, int NCH, bool TOP, int ROWS>
__global__ __launch_bounds__(NT * ROWS, NCH <= 4 && !TOP ? 8 : 4) void logprobs_row_kernel(const LogprobArgs p) {
    static_assert(ROWS == 1 || (NT == 64 && !TOP), "several rows a workgroup: a wave each, nothing shared");
    typedef LpElem<T> E;
    constexpr int VEC = E::VEC, NW = NT / 64, NV = NCH * VEC, NEAR = TOP ? 64 : 1, LIST = NEAR * (NV + 1);
    constexpr int LOW = sizeof(T) == 2 ? 16 : 0;                     // lowest bit of the keys that tells two values apart
    __shared__ float red_m[NW], red_s[NW], red_t[NW], red_e[NW];
    __shared__ unsigned keymax[TOP ? NT : 1];
    __shared__ u32x4 near_z[TOP ? NEAR * NCH : 1];                   // [NEAR][NCH] pieces of the threads that reach tau, and who they are
    __shared__ int near_tid[NEAR];
    __shared__ float near_one[NEAR];
    __shared__ unsigned long long list[TOP ? LIST : 1];
    __shared__ unsigned nnear, nlist, tau_s, many_s, wtot[NW];
    const long row = p.row0 + (long)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x >> 6 : 0);
    if (ROWS > 1 && row >= p.rows) return;
    const T* z = (const T*)p.z + row * p.ldz;
    const int tid = ROWS > 1 ? threadIdx.x & 63 : threadIdx.x, wave = tid >> 6, lane = tid & 63;
    u32x4 raw[NCH];
    const int whole = p.V / VEC, rest = whole * VEC;                 // whole pieces; thread t also holds column rest + t, if there is one
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        raw[i] = E::pack_all(-INFINITY);
        if (i * NT + tid < whole) raw[i] = lp_whole(z + (i * NT + tid) * VEC);
    }
    const float one = rest + tid < p.V ? E::get(z[rest + tid]) : -INFINITY;
    // the given tokens' logits: requested before the row's own reductions
    float zt = 0.f;
    long long tg = -1, tcol = -1;
    if (tid < p.T) {
        tg = p.targets[tid * p.rows + row];
        tcol = tg - p.tsub;
        if (tg >= 0 && tcol >= 0 && tcol < p.V) zt = E::get(z[tcol]);
    }
    if (TOP && tid == 0) nnear = nlist = 0;
    float mine = fmaxf(one, -INFINITY);                              // (a NaN does not count)
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        float f[VEC];
        E::unpack(raw[i], f);
#pragma unroll
        for (int e = 0; e < VEC; e += 2) mine = max3f(mine, f[e], f[e + 1]);
        __builtin_amdgcn_sched_barrier(0);
    }
    if (TOP) keymax[tid] = lp_sort(mine);
    const float mw = lp_wave_max(mine);
    float m = mw;
    if (ROWS == 1) {
        if (lane == 0) red_m[wave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, red_m[w]);
    }
    // (the floats are derived from the packed pieces anew in every phase: kept, they are twice the registers and half the waves)
    // s = sum of 2^x, t = sum of 2^x x over the columns BELOW m, eq = how many attain it; x = z log2 e - c, c = m log2 e as rounded: one fused
    // operation a column.  What c's rounding and log2 e's are off by is a factor common to all columns; it goes out with em = 2^xm, xm =
    // x at z = m.  (c's rounding stays below 2^-9 for |m| < 16384; beyond that, and for infinite m, x = (z - m) log2 e, xm = 0.)
    // Only the wave that holds m has columns to leave out: the others take the short loop.
    constexpr float L2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
    const float c = m * L2E;
    const bool close = fabsf(m) < 16384.f;
    float s, t, eq;
    auto add = [&](float zv) {
        const float x = close ? fmaf(zv, L2E, -c) : lp_diff(zv, m) * L2E, ex = zv == m ? 0.f : __builtin_amdgcn_exp2f(x);
        eq += zv == m ? 1.f : 0.f;
        s += ex;                                                     // (NaN iff the row has one)
        t = fmaf(ex, fmaxf(x, -1e4f), t);                            // (2^x is 0 by then: keeps 0 * -inf out)
    };
    s = t = eq = 0.f;
    add(one);
    if (close && mw < m) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            float f[VEC];
            pin(raw[i]);
            E::unpack(raw[i], f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float x = fmaf(f[e], L2E, -c), ex = __builtin_amdgcn_exp2f(x);
                s += ex;
                t = fmaf(ex, fmaxf(x, -1e4f), t);
            }
            __builtin_amdgcn_sched_barrier(0);                       // (one piece at a time: 64 exponentials in flight double the registers)
        }
    } else if (close) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            float f[VEC];
            pin(raw[i]);
            E::unpack(raw[i], f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float x = fmaf(f[e], L2E, -c), ex = f[e] == m ? 0.f : __builtin_amdgcn_exp2f(x);
                eq += f[e] == m ? 1.f : 0.f;
                s += ex;
                t = fmaf(ex, fmaxf(x, -1e4f), t);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        eq = lp_wave_sum(eq);
    } else {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            float f[VEC];
            pin(raw[i]);
            E::unpack(raw[i], f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) add(f[e]);
            __builtin_amdgcn_sched_barrier(0);
        }
        eq = lp_wave_sum(eq);
    }
    s = lp_wave_sum(s);
    t = lp_wave_sum(t);
    if (ROWS == 1 && lane == 0) { red_s[wave] = s; red_t[wave] = t; red_e[wave] = mw < m ? 0.f : eq; }
    if (TOP && wave == 0) {                                          // tau, by wave 0
        unsigned key[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) key[w] = keymax[w * 64 + lane];
        unsigned tau = 0;
        int have = NT;
        const int enough = min(max(p.top, 24), NEAR - 1);            // (fewer to rank, for a few more steps)
        for (int bit = 31; bit >= LOW && have > enough; --bit) {
            const unsigned trial = tau | (1u << bit);
            int n = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) n += __popcll(__ballot(key[w] >= trial));
            if (n >= p.top) { tau = trial; have = n; }
        }
        // (the keys of negative bf16 values have ones below LOW, that of NaN, 0, has none: tau becomes the whole key where it is compared
        //  for equality)
        if (LOW && have > enough && tau && !(tau & 0x80000000u)) tau |= (1u << LOW) - 1;
        if (lane == 0) { tau_s = tau; many_s = have > enough; }
    }
    if (ROWS == 1) {
        __syncthreads();
        s = t = eq = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) { s += red_s[w]; t += red_t[w]; eq += red_e[w]; }
    }
    if (!TOP && wave > 0) return;                                    // (what is left is a few numbers a row)
    const bool nan = s != s, empty = m == -INFINITY;
    const float xm = close ? fmaf(m, L2E, -c) : 0.f, iem = __builtin_amdgcn_exp2f(-xm);
    const float r = (eq - 1.f) + s * iem;                            // sum of exp(z - m) beside one column that attains m
    const float qnan = __uint_as_float(0x7fc00000u);
    const float lsum = empty ? 0.f : r < 0.125f ? log1pf(r) : __builtin_amdgcn_logf(1.f + r) * LN2;
    // H = log1p(r) - sum p (z - m); the columns at m have no part in the second sum
    const float ent = empty ? 0.f : lsum - LN2 * (t - xm * s) * iem * __builtin_amdgcn_rcpf(1.f + r);
    auto logp = [&](float zv) { return nan ? qnan : empty ? -INFINITY : lp_diff(zv, m) - lsum; };
    if (tid == 0) {
        p.stats[row] = nan ? qnan : m;
        p.stats[p.rows + row] = nan ? qnan : lsum;
        p.stats[2 * p.rows + row] = nan ? qnan : ent;
    }
    if (tid < p.T) p.logprobs[tid * p.rows + row] = tg < 0 ? 0.f : (tcol >= 0 && tcol < p.V) ? logp(zt) : nan ? qnan : -INFINITY;
    if constexpr (TOP) {
        const unsigned tau = tau_s, my = lp_sort(mine);
        const bool many = many_s != 0;
        if (many ? my > tau : my >= tau) {                           // <= 64 threads: the `have` of them, or fewer than `top`
            const unsigned at = atomicAdd(&nnear, 1u);
            if (at < NEAR) {
                near_tid[at] = tid;
                near_one[at] = one;
#pragma unroll
                for (int i = 0; i < NCH; ++i) near_z[at * NCH + i] = raw[i];
            }
        }
        __syncthreads();
        const int nn = min((int)nnear, NEAR) * NV;
        for (int x = tid; x < nn; x += NT) {
            const int i = x / VEC % NCH, e = x % VEC, at = x / NV;
            const int v = (i * NT + near_tid[at]) * VEC + e;
            const unsigned long long key = lp_key(E::get(((const T*)near_z)[x]), v);
            const unsigned u = (unsigned)(key >> 32);
            if (v < rest && (many ? u > tau : u >= tau)) list[atomicAdd(&nlist, 1u)] = key;
        }
        for (int x = tid; x < nn / NV; x += NT) {
            const int v = rest + near_tid[x];
            const unsigned long long key = lp_key(near_one[x], v);
            const unsigned u = (unsigned)(key >> 32);
            if (v < p.V && (many ? u > tau : u >= tau)) list[atomicAdd(&nlist, 1u)] = key;
        }
        __syncthreads();
        int n = (int)nlist;
        int need = p.top - n;                                        // > 0 only where many: the first columns that equal tau fill up
        // (a thread without columns, or with NaNs only, counted as -inf above: where that made tau -inf, NaNs fill what is still missing)
        for (int k = 0; k < 2 * (NCH + 1) && need > 0; ++k) {        // (uniform; one pass nearly always, the others' pieces come from the cache)
            const int i = k <= NCH ? k : k - (NCH + 1);
            const unsigned want = k <= NCH ? tau : 0u;
            float f[VEC];
            int v0 = (i * NT + tid) * VEC, end = rest;
            if (i == 0) E::unpack(raw[0], f);
            else if (i < NCH) lp_load(z, p.V, i * NT + tid, f);
            else { v0 = rest + tid; end = min(v0 + 1, p.V); f[0] = one; }            // the columns behind the last whole piece
            unsigned mask = 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) mask |= (v0 + e < end && lp_sort(f[e]) == want) ? 1u << e : 0u;
            int incl = __popc(mask);
            for (int o = 1; o < 64; o <<= 1) { const int up = __shfl_up(incl, o, 64); incl += lane >= o ? up : 0; }
            if (lane == 63) wtot[wave] = (unsigned)incl;
            __syncthreads();
            int before = incl - __popc(mask), total = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) { before += w < wave ? (int)wtot[w] : 0; total += (int)wtot[w]; }
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (mask >> e & 1) {
                    if (before < need) list[n + before] = lp_key(f[e], v0 + e);
                    ++before;
                }
            const int got = total < need ? total : need;
            n += got;
            need -= got;
            __syncthreads();
        }
        for (int i = tid; i < n; i += NT) {                          // rank = how many listed keys are larger (they are all different)
            const unsigned long long key = list[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += list[j] > key ? 1 : 0;
            if (rank < p.top) {
                const unsigned u = (unsigned)(key >> 32);
                const float zv = __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);              // the key's value (a row with a NaN answers NaN)
                p.top_ids[row * p.top + rank] = (int)~(unsigned)key + p.tsub;
                p.top_lp[row * p.top + rank] = logp(zv);
            }
        }
    }
}

constexpr int LP_THREADS = 256;
template <typename F>
__device__ __forceinline__ float lp_block(float x, F op, float* red) {
    for (int o = 32; o > 0; o >>= 1) x = op(x, __shfl_xor(x, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    return op(op(red[0], red[1]), op(red[2], red[3]));
}

// Rows that no register variant holds (V > ~65 500): the row is read again for each quantity.
template <typename T>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(const LogprobArgs p) {
    constexpr int VEC = LpElem<T>::VEC;
    __shared__ float red[4];
    __shared__ unsigned long long redk[4];
    const long row = p.row0 + blockIdx.x;
    const T* z = (const T*)p.z + row * p.ldz;
    const int nc = (p.V + VEC - 1) / VEC, tid = threadIdx.x;
    auto maxf = [](float a, float b) { return fmaxf(a, b); };
    auto addf = [](float a, float b) { return a + b; };
    float m = -INFINITY;
    bool nan = false;
    for (int c = tid; c < nc; c += LP_THREADS) {
        float f[VEC];
        lp_load(z, p.V, c, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { nan |= f[e] != f[e]; m = fmaxf(m, f[e]); }
    }
    m = lp_block(m, maxf, red);
    nan = __syncthreads_or(nan);
    float s = 0.f, t = 0.f;
    for (int c = tid; c < nc; c += LP_THREADS) {
        float f[VEC];
        lp_load(z, p.V, c, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int v = c * VEC + e;
            if (v >= p.V) continue;
            const float d = lp_diff(f[e], m);
            const float ex = __expf(d);
            s += d == 0.f ? 0.f : ex;
            t += ex > 0.f ? ex * d : 0.f;
        }
    }
    int equal = 0;                                     // columns that attain m: all but one of them belong to r
    for (int c = tid; c < nc; c += LP_THREADS) {
        float f[VEC];
        lp_load(z, p.V, c, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { const int v = c * VEC + e; equal += (v < p.V && f[e] == m) ? 1 : 0; }
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
            lp_load(z, p.V, c, f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int v = c * VEC + e;
                if (v >= p.V) continue;
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
    const void* z; long ldz; int V; long rows, row0;
    const long long* targets; int T; long long tsub;
    const float* stats; const float* g_lp; const float* g_ent;      // [3, rows]; [T, rows] or null; [rows] or null
    void* dz; long lddz;
};

// NT threads a row (ROWS rows a workgroup), every column by itself: x = (z - m - log_sum) log2 e, dz = -2^x (g + g_H (log p + H)).
// The pieces of a thread that hold a given token (a bit a piece, found first) get that column anew in a rare branch.
template <typename T, int NT, int ROWS>
__global__ __launch_bounds__(NT * ROWS) void logprobs_bwd_kernel(const LogprobBwdArgs p) {
    constexpr int VEC = LpElem<T>::VEC, U = NT > 64 ? 4 : 1;          // pieces whose loads are in flight together (short rows: more waves instead)
    constexpr float L2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
    const long row = p.row0 + (long)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / NT : 0);
    if (ROWS > 1 && row >= p.rows) return;
    const int tid = ROWS > 1 ? threadIdx.x % NT : threadIdx.x;
    const T* z = (const T*)p.z + row * p.ldz;
    T* dz = (T*)p.dz + row * p.lddz;
    const int whole = p.V / VEC;                                     // piece `whole` may be partial
    const float m = p.stats[row], lsum = p.stats[p.rows + row], ent = p.stats[2 * p.rows + row];
    const bool flat = m == INFINITY || m == -INFINITY;              // a forced row, or one with nothing left: no gradient
    const float gh = p.g_ent ? p.g_ent[row] : 0.f;
    float g = 0.f;
    unsigned long long hits = 0;                                     // bit j: piece tid + j NT holds a given token (63: and all behind it may)
    if (p.g_lp) {
        for (int i = 0; i < p.T; ++i) {
            const long long tg = p.targets[i * p.rows + row], v = tg - p.tsub;
            if (tg < 0) continue;
            g += p.g_lp[i * p.rows + row];
            if (v < 0 || v >= p.V) continue;                         // (in no column: only its -p, by g)
            const int c = (int)v / VEC, j = c / NT;
            if (c % NT == tid) hits |= 1ull << (j < 63 ? j : 63);
        }
    }
    const float ls2 = lsum * L2E, a0 = flat ? 0.f : g + gh * ent, a1 = flat ? 0.f : gh * LN2;
    // a given token's column: its share as -expm1(log p) - 1 - p taken as a difference would lose a sure token's gradient
    auto given = [&](float zv, long long tg) {
        const float lp = zv - m - lsum, pr = __expf(lp), one = -expm1f(lp);
        float sum = -(pr > 0.f ? pr * (lp + ent) * gh : 0.f);
        for (int k = 0; k < p.T; ++k) {
            const long long tk = p.targets[k * p.rows + row];
            if (tk >= 0) sum += p.g_lp[k * p.rows + row] * (tk == tg ? one : -pr);
        }
        return sum;
    };
    auto piece = [&](int c, int j, float* f) {
        const int v0 = c * VEC;
        float zk[VEC];
        const bool hit = (hits >> (j < 63 ? j : 63) & 1) && !flat;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            zk[e] = f[e];
            const float x = fmaxf(fmaf(f[e] - m, L2E, -ls2), -1e4f);  // (2^x is 0 by then: keeps 0 * -inf out; a NaN row's a0 is NaN)
            f[e] = -__builtin_amdgcn_exp2f(x) * fmaf(a1, x, a0);
        }
        if (hit) {
            for (int i = 0; i < p.T; ++i) {
                const long long tg = p.targets[i * p.rows + row], v = tg - p.tsub;
                if (tg < 0 || v < v0 || v >= v0 + VEC || v < 0 || v >= p.V) continue;
                float zv = 0.f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) zv = v0 + e == v ? zk[e] : zv;
                const float sum = given(zv, tg);
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] = (v0 + e == v) ? sum : f[e];
            }
        }
        if (flat) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = 0.f;
        }
    };
    int c = tid, j = 0;
    for (; c + (U - 1) * NT < whole; c += U * NT, j += U) {          // U pieces' loads in flight together
        u32x4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = lp_whole(z + (c + u * NT) * VEC);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[VEC];
            LpElem<T>::unpack(q[u], f);
            piece(c + u * NT, j + u, f);
            const u32x4 o = LpElem<T>::pack(f);
            __builtin_memcpy(dz + (c + u * NT) * VEC, &o, 16);
        }
    }
    for (; c < whole; c += NT, ++j) {
        float f[VEC];
        LpElem<T>::unpack(lp_whole(z + c * VEC), f);
        piece(c, j, f);
        const u32x4 o = LpElem<T>::pack(f);
        __builtin_memcpy(dz + c * VEC, &o, 16);
    }
    const int v = whole * VEC + tid;                                 // a column behind the last whole piece
    if (v < p.V) {
        const float zv = LpElem<T>::get(z[v]), x = fmaxf(fmaf(zv - m, L2E, -ls2), -1e4f);
        float d = -__builtin_amdgcn_exp2f(x) * fmaf(a1, x, a0);
        if (p.g_lp)
            for (int i = 0; i < p.T; ++i)
                if (p.targets[i * p.rows + row] >= 0 && p.targets[i * p.rows + row] - p.tsub == v) { d = given(zv, p.targets[i * p.rows + row]); break; }
        dz[v] = LpElem<T>::put(flat ? 0.f : d);
    }
}
}  // namespace libra

using namespace libra;

constexpr long LP_CHUNK = 1L << 21;                                 // rows of a launch: the threads of a grid are counted in 32 bits

// the smallest workgroup whose registers hold a row
template <typename T, bool TOP>
static void lp_launch(const LogprobArgs& a, hipStream_t st) {
    constexpr int W = 8 / LpElem<T>::VEC;                            // pieces are half as wide in fp32
    constexpr int R = TOP ? 1 : 4;                                   // short rows: four waves, four rows a workgroup
    const long rows = std::min(a.rows - a.row0, LP_CHUNK);
    const dim3 g((unsigned)rows);
    const int P = a.V / LpElem<T>::VEC;                              // whole pieces
    const dim3 g4((unsigned)((rows + R - 1) / R)), t4(64 * R);
    if (P <= 64 * W) hipLaunchKernelGGL((logprobs_row_kernel<T, 64, W, TOP, R>), g4, t4, 0, st, a);
    else if (P <= 128 * W) hipLaunchKernelGGL((logprobs_row_kernel<T, 64, 2 * W, TOP, R>), g4, t4, 0, st, a);
    else if (P <= 1024 * W) hipLaunchKernelGGL((logprobs_row_kernel<T, 256, 4 * W, TOP, 1>), g, dim3(256), 0, st, a);
    else if (P <= 4096 * W) hipLaunchKernelGGL((logprobs_row_kernel<T, 512, 8 * W, TOP, 1>), g, dim3(512), 0, st, a);
    else if (P <= 8192 * W) hipLaunchKernelGGL((logprobs_row_kernel<T, 1024, 8 * W, TOP, 1>), g, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL(logprobs_kernel<T>, g, dim3(LP_THREADS), 0, st, a);
}

template <typename T>
static void lp_launch_bwd(const LogprobBwdArgs& a, hipStream_t st) {
    const long rows = std::min(a.rows - a.row0, LP_CHUNK);
    if (a.V <= 2048) hipLaunchKernelGGL((logprobs_bwd_kernel<T, 64, 4>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((logprobs_bwd_kernel<T, 256, 1>), dim3((unsigned)rows), dim3(256), 0, st, a);
}

static int lp_check(const void* z, int64_t ldz, int64_t rows, int64_t V, int f32, const int64_t* targets, int64_t n_targets) {
    if (rows < 0 || rows > (1L << 40) || V <= 0 || V > 0x7fff0000L || ldz < V || n_targets < 0 || n_targets > 64) return LIBRA_ERR_SHAPE;
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
    LogprobArgs a{logits, (long)ldz, (int)V, (long)rows, 0, (const long long*)targets, (int)n_targets, (long long)target_sub, logprobs, stats,
                  (int)top, (long long*)top_ids, top_logprobs};
    const hipStream_t st = (hipStream_t)stream;
    for (; a.row0 < a.rows; a.row0 += LP_CHUNK) {
        if (f32) { if (top) lp_launch<float, true>(a, st); else lp_launch<float, false>(a, st); }
        else if (top) lp_launch<bf16_t, true>(a, st);
        else lp_launch<bf16_t, false>(a, st);
        if (hipGetLastError() != hipSuccess) return LIBRA_ERR_LAUNCH;
    }
    return LIBRA_OK;
}

extern "C" int libra_token_logprobs_bwd(const void* logits, int64_t ldz, int64_t rows, int64_t V, int f32, const int64_t* targets,
                                        int64_t n_targets, int64_t target_sub, const float* stats, const float* g_logprobs,
                                        const float* g_entropy, void* dlogits, int64_t lddz, void* stream) {
    if (rows == 0) return LIBRA_OK;
    const int rc = lp_check(logits, ldz, rows, V, f32, targets, n_targets);
    if (rc != LIBRA_OK) return rc;
    if (lddz < V) return LIBRA_ERR_SHAPE;
    if (!stats || !dlogits || ((uintptr_t)dlogits % (f32 ? 4 : 2)) || (g_logprobs && !targets)) return LIBRA_ERR_ALIGN;
    LogprobBwdArgs a{logits, (long)ldz, (int)V, (long)rows, 0, (const long long*)targets, (int)n_targets, (long long)target_sub, stats,
                     g_logprobs, g_entropy, dlogits, (long)lddz};
    for (; a.row0 < a.rows; a.row0 += LP_CHUNK) {
        if (f32) lp_launch_bwd<float>(a, (hipStream_t)stream);
        else lp_launch_bwd<bf16_t>(a, (hipStream_t)stream);
        if (hipGetLastError() != hipSuccess) return LIBRA_ERR_LAUNCH;
    }
    return LIBRA_OK;
}
