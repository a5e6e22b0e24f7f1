// Routed-bridge attention of ONE new query token per sequence over the 8-bit cache (format: kv8.hpp): the same selection as
// bridge_attn_decode,  s_j = q . K[m_q != m_j][j] / sqrt(128),  o = sum_j softmax(s)_j V[m_q != m_j][j],  start <= j < len,
// with K, V = code * 2^(scale - 127).  A key's K scale multiplies its finished score and its V scale its probability: one
// multiplication a key instead of 128, and exact (powers of two).
// HBM-bound: 256 bytes a key and head; 48 ragged sequences up to 2048 x 32 heads (560 MB) in 101 us = 5.5 TB/s with the VALU 43 % busy,
// 8 x 1024 in 14 us.  (No matrix instruction: one query row a head would fill 1 of its 16 rows.)  A wave takes 64 keys at a time, at multiples of 64:
//   * lane (g, u) = lane >> 3, lane & 7 reads the modality and, routed by it, the two scale bytes of key 8 u + g: one load each for 64
//     keys; the routing comes back to everyone as a ballot, the scales by a lane permutation when they are needed;
//   * 8 lanes own a key (16 codes = 16 bytes a lane): piece u of K and of V is one instruction of 8 keys = 1 KB contiguous, and the 16
//     of them (16 KB) are in flight together - one round trip to memory for the modality, one for all the rest;
//   * an 8-lane group keeps its own running maximum, sum and output (no traffic between lanes but the 3 steps of a dot product); groups
//     are merged once at the end, waves through LDS, key splits by a second kernel.
#include <algorithm>
#include "kv8.hpp"
#include "../../include/libra_hip.h"

namespace libra {

struct Decode8Args {
    const bf16_t* q; long ldq;                       // [B, H*128] roped query of the new token
    const unsigned char* codes; const unsigned char* scales;
    const unsigned char* kflag; long fstride;        // [B, >= capacity] modality of every cached token
    const unsigned char* qflag;                      // [B]
    const int* lens; const int* starts;              // [B] end of the valid tokens; first valid token or null
    bf16_t* out; long ldo;
    int B, H, cap, lg; float sl2;                    // scale * log2(e)
    float* part; int nsplit;                         // nsplit > 1: states [B*H][nsplit][D8_PART] instead of `out`
};
constexpr int D8_WAVES = 8;
constexpr int D8_KEYS = 64 * D8_WAVES;               // keys of a workgroup's iteration
constexpr int D8_MAX_SPLIT = 64;
constexpr int D8_PART = 132;                         // floats per partial state: 128 outputs, max, sum, 2 pad (rows 16-byte aligned)

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
    return x + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, false));
}
// sum over the 8 lanes of a group: within quads, then the other quad (whose lanes all hold the same by then)
__device__ __forceinline__ float group8_sum(float x) { return dpp_add<0x141>(dpp_add<0x4e>(dpp_add<0xb1>(x))); }
// over the 8 groups of a wave (lanes xor 8, 16, 32)
__device__ __forceinline__ float groups_max(float x) {
    x = fmaxf(x, __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x128, 0xf, 0xf, false)));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return half_swap_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float groups_sum(float x) {
    x = row_ror_add<8>(x);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return half_swap_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
// the share of split z of the keys [start, end): whole iterations of a workgroup; splits that get nothing have first >= end
struct D8Range { int start, end, first, last; };
__device__ __forceinline__ D8Range d8_range(const int* lens, const int* starts, int b, int cap, int nsplit, int z) {
    D8Range r;
    r.end = min(lens[b], cap);
    r.start = starts ? max(starts[b], 0) : 0;
    const int base = r.start & ~63;
    const int iters = r.end > r.start ? (r.end - base + D8_KEYS - 1) / D8_KEYS : 0;
    const int per = (iters + nsplit - 1) / nsplit;
    r.first = base + z * per * D8_KEYS;
    r.last = min(r.first + per * D8_KEYS, r.end);
    return r;
}

__global__ __launch_bounds__(D8_WAVES * 64, 4) void bridge_attn_decode8_kernel(const Decode8Args p) {
    __shared__ float red_m[D8_WAVES], red_l[D8_WAVES];
    __shared__ __attribute__((aligned(16))) float red_o[D8_WAVES][128];
    const int h = blockIdx.x, b = blockIdx.y, z = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 3, sub = lane & 7;                         // 16 channels [16 sub, 16 sub + 16) of keys 8 u + g
    const D8Range rg = d8_range(p.lens, p.starts, b, p.cap, p.nsplit, z);
    if (rg.first >= rg.last && z > 0) return;                        // (the merge knows; split 0 answers for a sequence without keys)
    const bool vis = p.qflag[b] != 0;
    float qf[16];
    unpack8(*(const u32x4*)(p.q + (long)b * p.ldq + h * 128 + sub * 16), qf);
    unpack8(*(const u32x4*)(p.q + (long)b * p.ldq + h * 128 + sub * 16 + 8), qf + 8);
#pragma unroll
    for (int e = 0; e < 16; ++e) qf[e] *= p.sl2;                     // scores in log2 units
    const unsigned char* fl = p.kflag + (long)b * p.fstride;
    const long plane = (long)p.B * p.H * p.cap, splane = plane >> p.lg;              // one of the four buffers, in tokens / scales
    const long head = ((long)b * p.H + h) * p.cap, shead = head >> p.lg;
    const unsigned char* kb = p.codes + head * 128 + sub * 16;
    const unsigned char* sb = p.scales + shead;
    float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = 0.f;
    for (int j0 = rg.first + wave * 64; j0 < rg.last; j0 += D8_KEYS) {
        // key 8 sub + g of the 64: clamped into the valid ones, so that nothing outside them is ever read
        const int mine = min(max(j0 + 8 * sub + g, rg.start), rg.end - 1);
        const bool cross = (fl[mine] != 0) != vis;
        const long so = (mine >> p.lg) + (cross ? splane : 0);
        const unsigned sc = ((unsigned)sb[so] << 8) | sb[so + 2 * splane];
        const unsigned long long ball = __ballot(cross);
        const unsigned routed = (unsigned)(ball >> (lane & 56)) & 0xffu;             // bit u: key 8 u + g takes the cross buffers
        const bool whole = j0 >= rg.start && j0 + 64 <= rg.end;
        u32x4 kq[8], vq[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int j = whole ? j0 + 8 * u + g : min(max(j0 + 8 * u + g, rg.start), rg.end - 1);
            const unsigned char* at = kb + ((long)j + ((routed >> u & 1) ? plane : 0)) * 128;
            kq[u] = *(const u32x4*)at;
            vq[u] = *(const u32x4*)(at + 2 * plane * 128);
        }
        float s[8], vs[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            float a = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float f[4];
                const unsigned w = kq[u][i];
                kv8_decode4(w, f);
#pragma unroll
                for (int e = 0; e < 4; ++e) a = fmaf(qf[4 * i + e], f[e], a);
            }
            const unsigned w = (unsigned)__shfl((int)sc, (lane & 56) | u, 64);
            s[u] = group8_sum(a) * kv8_scale(w >> 8);
            vs[u] = kv8_scale(w & 0xff);
            if (!whole) { const int j = j0 + 8 * u + g; s[u] = (j >= rg.start && j < rg.end) ? s[u] : -INFINITY; }
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < 8; ++u) mn = fmaxf(mn, s[u]);
        const float base = mn == -INFINITY ? 0.f : mn;               // a group that has seen no key yet: every weight 0, no NaN
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] *= alpha;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float pr = __builtin_amdgcn_exp2f(s[u] - base);
            l += pr;
            const float pv = pr * vs[u];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float f[4];
                const unsigned w = vq[u][i];
                kv8_decode4(w, f);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[4 * i + e] = fmaf(pv, f[e], o[4 * i + e]);
            }
        }
    }
    // groups of the wave, then the waves
    const float mw = groups_max(m);
    const float wt = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mw);
    l = groups_sum(l * wt);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = groups_sum(o[e] * wt);
    if (lane == 0) { red_m[wave] = mw; red_l[wave] = l; }
    if (g == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *(f32x4*)(&red_o[wave][sub * 16 + 4 * i]) = f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]};
    }
    __syncthreads();
    if (threadIdx.x < 128) {
        float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < D8_WAVES; ++w) M = fmaxf(M, red_m[w]);
#pragma unroll
        for (int w = 0; w < D8_WAVES; ++w) {
            const float f = red_m[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(red_m[w] - M);
            L = fmaf(red_l[w], f, L);
            acc = fmaf(red_o[w][threadIdx.x], f, acc);
        }
        if (p.nsplit > 1) {
            float* pt = p.part + (((long)b * p.H + h) * p.nsplit + z) * D8_PART;
            pt[threadIdx.x] = acc;
            if (threadIdx.x == 0) { pt[128] = M; pt[129] = L; }
        } else {
            p.out[(long)b * p.ldo + h * 128 + threadIdx.x] = f2bf(L == 0.f ? 0.f : acc / L);
        }
    }
}

// fold the key splits of one (sequence, head): four waves take every fourth split, two channels a lane (the order is fixed)
__global__ __launch_bounds__(256) void bridge_attn_decode8_merge_kernel(const Decode8Args p) {
    __shared__ float acc_s[4][128];
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float* pt = p.part + ((long)b * p.H + h) * p.nsplit * D8_PART;
    const D8Range rg = d8_range(p.lens, p.starts, b, p.cap, p.nsplit, 0);
    const int per = max(rg.last - rg.first, 1);                      // keys of a full split: split z has some iff first + z per < end
    const int n = rg.end > rg.start ? min(p.nsplit, (rg.end - rg.first + per - 1) / per) : 1;
    float mz = -INFINITY, lz = 0.f;
    if (lane < n) { mz = pt[lane * D8_PART + 128]; lz = pt[lane * D8_PART + 129]; }
    float M = mz;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) M = fmaxf(M, __shfl_xor(M, s, 64));
    const float w = mz == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mz - M);
    float L = lz * w;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) L += __shfl_xor(L, s, 64);
    float a0 = 0.f, a1 = 0.f;
#pragma unroll 8
    for (int z = wave; z < n; z += 4) {
        const float wz = __shfl(w, z, 64);
        a0 = fmaf(pt[z * D8_PART + lane * 2], wz, a0);
        a1 = fmaf(pt[z * D8_PART + lane * 2 + 1], wz, a1);
    }
    acc_s[wave][lane * 2] = a0;
    acc_s[wave][lane * 2 + 1] = a1;
    __syncthreads();
    if (threadIdx.x < 128) {
        const int c = threadIdx.x;
        const float a = (acc_s[0][c] + acc_s[1][c]) + (acc_s[2][c] + acc_s[3][c]);
        p.out[(long)b * p.ldo + h * 128 + c] = f2bf(L == 0.f ? 0.f : a / L);          // (no key: zeros)
    }
}

// Key splits of a (sequence, head): 1 - no second kernel - where the pairs alone give every CU a workgroup; below that, as many as that
// takes, at most one for two iterations of the CAPACITY (the lengths are device words: a captured step must not depend on them).
// Workgroups of 8 waves, two a CU, measured against 4 and 16 waves with 1 ... 32 splits at 17 sizes of 32 heads.  us (waves x splits),
// the rule's first, in brackets the bytes at the rate of a large copy (5.2 TB/s: what to expect, no bound - reads alone go faster):
//   1 x 8191 [12.9]: 19.8 (8x8) 23.7 (8x4) 59.9 (8x1) 19.6 (4x16) 19.7 (16x8)    2 x 4000 [12.6]: 19.1 (8x4) 34.0 (8x1) 20.9 (8x8) 19.1 (16x4)
//   4 x 2048 [12.9]: 18.8 (8x2) 20.7 (8x1) 19.5 (8x4) 18.7 (16x1)     8 x 1024 [12.9]: 15.8 (8x1) 20.9 (8x2) 15.3 (16x1) 19.1 (4x4)
//   16 x 2048 [51.6]: 50.1 (8x1) 53.0 (8x2) 53.3 (16x1) 50.6 (4x1)    64 x 2048 [206]: 181 (8x1) 195 (8x2) 189 (16x1) 189 (4x1)
//   32 x 600 [30.2]: 31.1 (8x1) 39.3 (8x2) 40.9 (16x1) 31.7 (4x1)
// Within 4 % of the best at the sizes from 8 sequences on and at long contexts.  It is NOT the best where a small batch's contexts
// are short of a capacity that splits (two splits share what one or two iterations hold, and the merge costs its launch), 2048 slots:
//   1 x 300: 8.0 (8x2) 5.8 (8x1)    1 x 1024: 9.7 (8x2) 9.5 (8x1) 8.4 (4x4)    2 x 1024: 10.3 (8x2) 9.6 (8x1) 9.3 (4x4)
//   4 x 1024: 13.8 (8x2) 13.7 (8x1) 12.2 (16x1)
// The split decides the order of the fp32 sums: the same bits for the same (B H, capacity), and at any batch up to 1024 slots.
static int d8_splits(int64_t B, int64_t H, int64_t capacity) {
    const int64_t want = (256 + B * H - 1) / (B * H), most = (capacity + 2 * D8_KEYS - 1) / (2 * D8_KEYS);
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, most), D8_MAX_SPLIT));
}

}  // namespace libra

using namespace libra;

extern "C" int libra_kv8_geometry_(const void* codes, const void* scales, int64_t B, int64_t H, int64_t capacity, int64_t block);

extern "C" size_t libra_bridge_attn_decode8_workspace_bytes(int64_t B, int64_t H, int64_t capacity) {
    const int n = (B <= 0 || H <= 0 || capacity <= 0) ? 1 : d8_splits(B, H, capacity);
    return n == 1 ? 0 : (size_t)B * (size_t)H * n * D8_PART * sizeof(float);
}

extern "C" int libra_bridge_attn_decode8(const void* q, int64_t ldq, const uint8_t* codes, const uint8_t* scales, const uint8_t* key_flag,
                                         int64_t flag_stride, const uint8_t* query_flag, const int32_t* kv_len, const int32_t* kv_start,
                                         void* out, int64_t ldo, int64_t B, int64_t H, int64_t capacity, int64_t block, float scale,
                                         float* workspace, size_t workspace_bytes, void* stream) {
    if (B == 0) return LIBRA_OK;
    const int lg = libra_kv8_geometry_(codes, scales, B, H, capacity, block);
    if (lg < 0) return lg;
    if (ldq < H * 128 || ldo < H * 128 || flag_stride < capacity) return LIBRA_ERR_SHAPE;
    if (!q || !key_flag || !query_flag || !kv_len || !out) return LIBRA_ERR_ALIGN;
    if ((ldq % 8) || ((uintptr_t)q & 15) || ((uintptr_t)out & 1)) return LIBRA_ERR_ALIGN;
    const size_t need = libra_bridge_attn_decode8_workspace_bytes(B, H, capacity);
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return LIBRA_ERR_ALIGN;
    Decode8Args a;
    a.q = (const bf16_t*)q; a.ldq = ldq; a.codes = codes; a.scales = scales; a.kflag = key_flag; a.fstride = flag_stride;
    a.qflag = query_flag; a.lens = kv_len; a.starts = kv_start; a.out = (bf16_t*)out; a.ldo = ldo;
    a.B = (int)B; a.H = (int)H; a.cap = (int)capacity; a.lg = lg; a.sl2 = scale * 1.4426950408889634f;
    a.part = workspace; a.nsplit = d8_splits(B, H, capacity);
    const dim3 grid((unsigned)H, (unsigned)B, (unsigned)a.nsplit), grid2((unsigned)H, (unsigned)B);
    const hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(bridge_attn_decode8_kernel, grid, dim3(D8_WAVES * 64), 0, st, a);
    if (hipGetLastError() != hipSuccess) return LIBRA_ERR_LAUNCH;
    if (a.nsplit > 1) hipLaunchKernelGGL(bridge_attn_decode8_merge_kernel, grid2, dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? LIBRA_OK : LIBRA_ERR_LAUNCH;
}
