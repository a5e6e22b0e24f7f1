// Routed-bridge attention of ONE new query token per sequence over the 8-bit cache (format: kv8.hpp): the same selection as
// bridge_attn_decode,  s_j = q . K[m_q != m_j][j] / sqrt(128),  o = sum_j softmax(s)_j V[m_q != m_j][j],  start <= j < len,
// with K, V = code * 2^(scale - 127).  A key's K scale multiplies its finished score and its V scale its probability: one
// multiplication a key instead of 128, and exact (powers of two).
// 8 lanes own a key (16 codes = 16 bytes a lane): a wave reads 8 keys = 1 KB contiguous per instruction.
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
    float* part; int nsplit;
};
constexpr int D8_SPLIT = 8;                          // key splits a workspace has room for
constexpr int D8_PART = 132;                         // floats per partial state: 128 outputs, max, sum, 2 pad
constexpr int D8_WAVES = 4;

__global__ __launch_bounds__(D8_WAVES * 64) void bridge_attn_decode8_kernel(const Decode8Args p) {
    __shared__ float red_m[D8_WAVES * 8], red_l[D8_WAVES * 8];
    __shared__ __attribute__((aligned(16))) float red_o[D8_WAVES * 8][128];
    const int h = blockIdx.x, b = blockIdx.y, z = blockIdx.z;
    const int grp = threadIdx.x >> 3, sub = threadIdx.x & 7;         // 16 channels [16 sub, 16 sub + 16)
    const int end_all = min(p.lens[b], p.cap);
    const int start_all = p.starts ? max(p.starts[b], 0) : 0;
    constexpr int KEYS = D8_WAVES * 8;
    int per = (end_all - start_all + p.nsplit - 1) / p.nsplit;
    per = (per + KEYS - 1) / KEYS * KEYS;
    const int j0 = start_all + z * per, j1 = min(j0 + per, end_all);
    const int mq = p.qflag[b] != 0;
    float qf[16];
    unpack8(*(const u32x4*)(p.q + (long)b * p.ldq + h * 128 + sub * 16), qf);
    unpack8(*(const u32x4*)(p.q + (long)b * p.ldq + h * 128 + sub * 16 + 8), qf + 8);
    const unsigned char* fl = p.kflag + (long)b * p.fstride;
    const long plane = (long)p.B * p.H;
    const long head = (long)b * p.H + h;
    float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = 0.f;
    for (int j = j0 + grp; j < j1; j += KEYS) {
        const long hk = ((fl[j] != 0) != (mq != 0) ? plane : 0) + head, hv = hk + 2 * plane;
        const u32x4 kq = *(const u32x4*)(p.codes + (hk * p.cap + j) * 128 + sub * 16);
        const u32x4 vq = *(const u32x4*)(p.codes + (hv * p.cap + j) * 128 + sub * 16);
        const float ks = kv8_scale(p.scales[hk * (p.cap >> p.lg) + (j >> p.lg)]);
        const float vs = kv8_scale(p.scales[hv * (p.cap >> p.lg) + (j >> p.lg)]);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float f[4];
            const unsigned w = kq[i];
            kv8_decode4(w, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fmaf(qf[4 * i + e], f[e], s);
        }
        s += __shfl_xor(s, 1, 64);
        s += __shfl_xor(s, 2, 64);
        s += __shfl_xor(s, 4, 64);
        s *= ks * p.sl2;
        const float mn = fmaxf(m, s);
        const float alpha = __builtin_amdgcn_exp2f(m - mn);           // first key: exp2(-inf) = 0
        const float pr = __builtin_amdgcn_exp2f(s - mn);
        l = l * alpha + pr;
        const float pv = pr * vs;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float f[4];
            const unsigned w = vq[i];
            kv8_decode4(w, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * i + e] = fmaf(pv, f[e], o[4 * i + e] * alpha);
        }
        m = mn;
    }
    if (sub == 0) { red_m[grp] = m; red_l[grp] = l; }
#pragma unroll
    for (int i = 0; i < 4; ++i) *(f32x4*)(&red_o[grp][sub * 16 + 4 * i]) = f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]};
    __syncthreads();
    if (threadIdx.x < 128) {
        float M = -INFINITY;
        for (int g = 0; g < KEYS; ++g) M = fmaxf(M, red_m[g]);
        float L = 0.f, acc = 0.f;
        for (int g = 0; g < KEYS; ++g) {
            const float w = red_m[g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(red_m[g] - M);   // groups that saw no key
            L = fmaf(red_l[g], w, L);
            acc = fmaf(red_o[g][threadIdx.x], w, acc);
        }
        if (p.nsplit > 1) {
            float* pt = p.part + (head * p.nsplit + z) * D8_PART;
            pt[threadIdx.x] = acc;
            if (threadIdx.x == 0) { pt[128] = M; pt[129] = L; }
        } else {
            p.out[(long)b * p.ldo + h * 128 + threadIdx.x] = f2bf(L > 0.f ? acc / L : 0.f);
        }
    }
}

// fold the key splits of one (sequence, head) in split order
__global__ __launch_bounds__(128) void bridge_attn_decode8_merge_kernel(const float* __restrict__ part, int nsplit, bf16_t* __restrict__ out,
                                                                        long ldo, int H) {
    const int h = blockIdx.x, b = blockIdx.y;
    const float* pt = part + ((long)b * H + h) * nsplit * D8_PART;
    float M = -INFINITY;
    for (int z = 0; z < nsplit; ++z) M = fmaxf(M, pt[z * D8_PART + 128]);
    float L = 0.f, acc = 0.f;
    for (int z = 0; z < nsplit; ++z) {
        const float mz = pt[z * D8_PART + 128];
        const float w = mz == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mz - M);
        L = fmaf(pt[z * D8_PART + 129], w, L);
        acc = fmaf(pt[z * D8_PART + threadIdx.x], w, acc);
    }
    out[(long)b * ldo + h * 128 + threadIdx.x] = f2bf(L > 0.f ? acc / L : 0.f);
}

}  // namespace libra

using namespace libra;

extern "C" int libra_kv8_geometry_(const void* codes, const void* scales, int64_t B, int64_t H, int64_t capacity, int64_t block);

extern "C" size_t libra_bridge_attn_decode8_workspace_bytes(int64_t B, int64_t H) {
    return (B <= 0 || H <= 0) ? 0 : (size_t)B * (size_t)H * D8_SPLIT * D8_PART * sizeof(float);
}

extern "C" int libra_bridge_attn_decode8(const void* q, int64_t ldq, const uint8_t* codes, const uint8_t* scales, const uint8_t* key_flag,
                                         int64_t flag_stride, const uint8_t* query_flag, const int32_t* kv_len, const int32_t* kv_start,
                                         void* out, int64_t ldo, int64_t B, int64_t H, int64_t capacity, int64_t block, float scale,
                                         float* workspace, size_t workspace_bytes, void* stream) {
    if (B == 0) return LIBRA_OK;
    const int lg = libra_kv8_geometry_(codes, scales, B, H, capacity, block);
    if (lg < 0) return lg;
    if (ldq < H * 128 || ldo < H * 128 || flag_stride < capacity) return LIBRA_ERR_SHAPE;
    if (!q || !key_flag || !query_flag || !kv_len || !out || !workspace) return LIBRA_ERR_ALIGN;
    if ((ldq % 8) || ((uintptr_t)q & 15) || ((uintptr_t)workspace & 15) || ((uintptr_t)out & 1)) return LIBRA_ERR_ALIGN;
    if (workspace_bytes < libra_bridge_attn_decode8_workspace_bytes(B, H)) return LIBRA_ERR_ALIGN;
    Decode8Args a;
    a.q = (const bf16_t*)q; a.ldq = ldq; a.codes = codes; a.scales = scales; a.kflag = key_flag; a.fstride = flag_stride;
    a.qflag = query_flag; a.lens = kv_len; a.starts = kv_start; a.out = (bf16_t*)out; a.ldo = ldo;
    a.B = (int)B; a.H = (int)H; a.cap = (int)capacity; a.lg = lg; a.sl2 = scale * 1.4426950408889634f;
    a.part = workspace; a.nsplit = D8_SPLIT;
    hipLaunchKernelGGL(bridge_attn_decode8_kernel, dim3((unsigned)H, (unsigned)B, (unsigned)a.nsplit), dim3(D8_WAVES * 64), 0,
                       (hipStream_t)stream, a);
    if (hipGetLastError() != hipSuccess) return LIBRA_ERR_LAUNCH;
    hipLaunchKernelGGL(bridge_attn_decode8_merge_kernel, dim3((unsigned)H, (unsigned)B), dim3(128), 0, (hipStream_t)stream,
                       (const float*)workspace, a.nsplit, (bf16_t*)out, (long)ldo, (int)H);
    return hipGetLastError() == hipSuccess ? LIBRA_OK : LIBRA_ERR_LAUNCH;
}
