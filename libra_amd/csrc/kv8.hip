// Writers and reader of the 8-bit K / V cache (format: kv8.hpp), all HBM-bound: 2 bytes in and 1 out a value (fill, append), or the reverse.
// A 16-lane group owns one row of one head (8 channels a lane): the block maximum is four DPP row steps, no LDS, no atomics.
#include "kv8.hpp"
#include "../../include/libra_hip.h"

namespace libra {

struct Kv8FillArgs {
    const bf16_t* src[4]; long ld[4];                 // [B*S, H*128] rows
    unsigned char* codes; unsigned char* scales;
    const int* start;                                 // [B] first valid token of each sequence, or null
    int B, S, H, lg, cap;
};

// One wave = 64 tokens of one head, each of its 16-lane groups 16 of them, all 16 rows of a group in flight together (read once, kept
// packed in registers).  The maximum of a block of up to 16 tokens stays within the group; larger blocks join 2 or 4 groups.
// Tokens before `start` are stored as zeros and do not count for the scale (what a padded position holds must not coarsen, or poison,
// its neighbours).  Bound by HBM: 3 bytes a value.  One pass instead of two reads of the block: 213 -> 152 us at 8 x 2048 x
// 32 heads (806 MB, 5.3 TB/s).
template <int LG>
__global__ __launch_bounds__(256) void kv8_fill_kernel(const Kv8FillArgs p) {
    const int h = (int)blockIdx.y * 4 + (threadIdx.x >> 6);
    if (h >= p.H) return;
    const int w = blockIdx.z & 3, b = blockIdx.z >> 2;
    const int sub = threadIdx.x & 15;
    const int t0 = (int)blockIdx.x * 64 + (threadIdx.x >> 4 & 3) * 16;               // first of the group's tokens
    const int first = p.start ? max(p.start[b], 0) : 0;
    const bf16_t* src = w == 0 ? p.src[0] : w == 1 ? p.src[1] : w == 2 ? p.src[2] : p.src[3];
    const long ld = w == 0 ? p.ld[0] : w == 1 ? p.ld[1] : w == 2 ? p.ld[2] : p.ld[3];
    const bf16_t* s = src + ((long)b * p.S + t0) * ld + h * 128 + sub * 8;
    u32x4 raw[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        raw[i] = u32x4{0u, 0u, 0u, 0u};
        if (t0 + i >= first && t0 + i < p.S) raw[i] = *(const u32x4*)(s + i * ld);
    }
    unsigned mx[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        mx[i] = 0;
        float f[8];
        unpack8(raw[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) { const unsigned a = kv8_abs_bits(f[e]); mx[i] = a > mx[i] ? a : mx[i]; }
    }
    constexpr int IN = LG < 4 ? LG : 4, NB = 16 >> IN;               // blocks of a group
    int byte[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        unsigned x = 0;
#pragma unroll
        for (int i = 0; i < (1 << IN); ++i) { const unsigned a = mx[(k << IN) + i]; x = a > x ? a : x; }
        x = row16_max(x);
        if (LG >= 5) { const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false); x = max((unsigned)r[0], (unsigned)r[1]); }
        if (LG >= 6) { const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false); x = max((unsigned)r[0], (unsigned)r[1]); }
        byte[k] = kv8_byte(x);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) pin(raw[i]);                        // (the floats are derived again below: kept, they double the registers)
    const long head = ((long)w * p.B + b) * p.H + h;
    unsigned char* sc = p.scales + head * (p.cap >> LG);
    unsigned char* dst = p.codes + (head * p.cap + t0) * 128 + sub * 8;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        const int t = t0 + (k << IN);
        if (sub == 0 && t < p.S && (t & ((1 << LG) - 1)) == 0) sc[t >> LG] = (unsigned char)byte[k];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float inv = kv8_inverse(byte[i >> IN]);
        float f[8];
        unpack8(raw[i], f);
        u32x2 c;
        c[0] = kv8_encode4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
        c[1] = kv8_encode4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
        if (t0 + i < p.S) *(u32x2*)(dst + i * 128) = c;
    }
}

struct Kv8AppendArgs {
    const bf16_t* src[4]; long ld[4];                 // [B, H*128] rows
    unsigned char* codes; unsigned char* scales;
    const long long* slot;                            // device word: the step stays capturable
    int B, H, lg, cap;
};

// One 16-lane group = one row of one head.  The first token of a block sets its scale; a later one that needs a larger scale
// re-expresses the block's earlier codes (the group owns the whole block of its head: no other wave touches it).  Bound by launch and one
// round trip to memory (two where a block grows): 2.8 us for 1 sequence x 32 heads, 4.0 us for 64.
__global__ __launch_bounds__(256) void kv8_append_kernel(const Kv8AppendArgs p) {
    const int w = blockIdx.y, b = blockIdx.z;
    const int h = (int)blockIdx.x * 16 + (threadIdx.x >> 4), sub = threadIdx.x & 15;
    const long long slot = p.slot[0];
    if (h >= p.H || slot < 0 || slot >= p.cap) return;                // outside the cache: nothing is stored (as kv_cache_append)
    const bf16_t* src = w == 0 ? p.src[0] : w == 1 ? p.src[1] : w == 2 ? p.src[2] : p.src[3];
    const long ld = w == 0 ? p.ld[0] : w == 1 ? p.ld[1] : w == 2 ? p.ld[2] : p.ld[3];
    const long head = ((long)w * p.B + b) * p.H + h;
    unsigned char* sc = p.scales + head * (p.cap >> p.lg) + (slot >> p.lg);
    const int old = sc[0];                                            // (in flight together with the row)
    float f[8];
    unpack8(*(const u32x4*)(src + b * ld + h * 128 + sub * 8), f);
    unsigned mx = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) { const unsigned a = kv8_abs_bits(f[e]); mx = a > mx ? a : mx; }
    int byte = kv8_byte(row16_max(mx));
    unsigned char* dst = p.codes + head * p.cap * 128 + sub * 8;
    const int in_block = (int)slot & ((1 << p.lg) - 1);
    byte = kv8_grow(dst - sub * 8 + (slot - in_block) * 128, in_block, byte, old, sub);
    const float inv = kv8_inverse(byte);
    u32x2 c;
    c[0] = kv8_encode4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
    c[1] = kv8_encode4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
    *(u32x2*)(dst + slot * 128) = c;
    if (sub == 0) sc[0] = (unsigned char)byte;
}

struct Kv8ReadArgs {
    const unsigned char* codes; const unsigned char* scales;
    bf16_t* out; long ldo, buf_stride;                // [4][B*n] rows of H*128
    int B, H, lg, cap, first, n;
};
// One thread = 8 channels of one row (8 bytes in, 16 out).  e4m3 times a power of two is exact in bf16 (bf16 has the wider exponent
// and 4 more mantissa bits; below 2^-126 the nearest bf16).  Bound by HBM: 8 x 1024 tokens x 32 heads (404 MB) in 77 us, 5.2 TB/s.
__global__ __launch_bounds__(256) void kv8_read_kernel(const Kv8ReadArgs p) {
    const int w = blockIdx.z, b = blockIdx.y, t = p.first + (int)blockIdx.x;
    const long row = (long)b * p.n + blockIdx.x;
    for (int c = threadIdx.x; c < p.H * 16; c += 256) {
        const int h = c >> 4, sub = c & 15;
        const long head = ((long)w * p.B + b) * p.H + h;
        const float s = kv8_scale(p.scales[head * (p.cap >> p.lg) + (t >> p.lg)]);
        const u32x2 q = *(const u32x2*)(p.codes + (head * p.cap + t) * 128 + sub * 8);
        float f[8];
        kv8_decode4(q[0], f);
        kv8_decode4(q[1], f + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= s;
        *(u32x4*)(p.out + w * p.buf_stride + row * p.ldo + c * 8) = pack8(f);
    }
}

static inline bool al16(const void* p) { return (((uintptr_t)p) & 15) == 0; }
static inline int launched() { return hipGetLastError() == hipSuccess ? LIBRA_OK : LIBRA_ERR_LAUNCH; }

}  // namespace libra

using namespace libra;

// shared argument checks: geometry of the cache; returns log2(block) or a negative error code
extern "C" int libra_kv8_geometry_(const void* codes, const void* scales, int64_t B, int64_t H, int64_t capacity, int64_t block) {
    if (B <= 0 || B > 16383 || H <= 0 || H > 4096 || capacity <= 0 || capacity > 0x3fffffffL) return LIBRA_ERR_SHAPE;
    if (block <= 0 || block > KV8_MAX_BLOCK || (block & (block - 1)) || capacity % block) return LIBRA_ERR_SHAPE;
    if (!codes || !scales || !al16(codes)) return LIBRA_ERR_ALIGN;
    int lg = 0;
    while ((1 << lg) < block) ++lg;
    return lg;
}

extern "C" int libra_kv8_fill(const void* k_same, int64_t ld_ks, const void* k_cross, int64_t ld_kc, const void* v_same, int64_t ld_vs,
                              const void* v_cross, int64_t ld_vc, uint8_t* codes, uint8_t* scales, int64_t B, int64_t S, int64_t H,
                              int64_t capacity, int64_t block, const int32_t* kv_start, void* stream) {
    if (B == 0 || S == 0) return LIBRA_OK;
    const int lg = libra_kv8_geometry_(codes, scales, B, H, capacity, block);
    if (lg < 0) return lg;
    if (S < 0 || S > capacity) return LIBRA_ERR_SHAPE;
    Kv8FillArgs a;
    const void* src[4] = {k_same, k_cross, v_same, v_cross};
    const int64_t ld[4] = {ld_ks, ld_kc, ld_vs, ld_vc};
    for (int i = 0; i < 4; ++i) {
        if (ld[i] < H * 128) return LIBRA_ERR_SHAPE;
        if (!src[i] || !al16(src[i]) || ld[i] % 8) return LIBRA_ERR_ALIGN;
        a.src[i] = (const bf16_t*)src[i]; a.ld[i] = ld[i];
    }
    a.codes = codes; a.scales = scales; a.start = kv_start; a.B = (int)B; a.S = (int)S; a.H = (int)H; a.lg = lg; a.cap = (int)capacity;
    const dim3 g((unsigned)((S + 63) / 64), (unsigned)((H + 3) / 4), (unsigned)(4 * B)), t(256);
    const hipStream_t st = (hipStream_t)stream;
    switch (lg) {
        case 0: hipLaunchKernelGGL(kv8_fill_kernel<0>, g, t, 0, st, a); break;
        case 1: hipLaunchKernelGGL(kv8_fill_kernel<1>, g, t, 0, st, a); break;
        case 2: hipLaunchKernelGGL(kv8_fill_kernel<2>, g, t, 0, st, a); break;
        case 3: hipLaunchKernelGGL(kv8_fill_kernel<3>, g, t, 0, st, a); break;
        case 4: hipLaunchKernelGGL(kv8_fill_kernel<4>, g, t, 0, st, a); break;
        case 5: hipLaunchKernelGGL(kv8_fill_kernel<5>, g, t, 0, st, a); break;
        default: hipLaunchKernelGGL(kv8_fill_kernel<6>, g, t, 0, st, a);
    }
    return launched();
}

extern "C" int libra_kv8_append(const void* k_same, int64_t ld_ks, const void* k_cross, int64_t ld_kc, const void* v_same, int64_t ld_vs,
                                const void* v_cross, int64_t ld_vc, uint8_t* codes, uint8_t* scales, int64_t B, int64_t H,
                                int64_t capacity, int64_t block, const int64_t* slot, void* stream) {
    if (B == 0) return LIBRA_OK;
    const int lg = libra_kv8_geometry_(codes, scales, B, H, capacity, block);
    if (lg < 0) return lg;
    if (!slot) return LIBRA_ERR_ALIGN;
    Kv8AppendArgs a;
    const void* src[4] = {k_same, k_cross, v_same, v_cross};
    const int64_t ld[4] = {ld_ks, ld_kc, ld_vs, ld_vc};
    for (int i = 0; i < 4; ++i) {
        if (ld[i] < H * 128) return LIBRA_ERR_SHAPE;
        if (!src[i] || !al16(src[i]) || ld[i] % 8) return LIBRA_ERR_ALIGN;
        a.src[i] = (const bf16_t*)src[i]; a.ld[i] = ld[i];
    }
    a.codes = codes; a.scales = scales; a.slot = (const long long*)slot; a.B = (int)B; a.H = (int)H; a.lg = lg; a.cap = (int)capacity;
    hipLaunchKernelGGL(kv8_append_kernel, dim3((unsigned)((H + 15) / 16), 4, (unsigned)B), dim3(256), 0, (hipStream_t)stream, a);
    return launched();
}

extern "C" int libra_kv8_read(const uint8_t* codes, const uint8_t* scales, void* out, int64_t ldo, int64_t buffer_stride, int64_t B,
                              int64_t H, int64_t capacity, int64_t block, int64_t first, int64_t n, void* stream) {
    if (B == 0 || n == 0) return LIBRA_OK;
    const int lg = libra_kv8_geometry_(codes, scales, B, H, capacity, block);
    if (lg < 0) return lg;
    if (n < 0 || first < 0 || first + n > capacity || ldo < H * 128 || buffer_stride < 0 || n > 0xffffffL) return LIBRA_ERR_SHAPE;
    if (!out || !al16(out) || ldo % 8 || buffer_stride % 8) return LIBRA_ERR_ALIGN;
    Kv8ReadArgs a{codes, scales, (bf16_t*)out, (long)ldo, (long)buffer_stride, (int)B, (int)H, lg, (int)capacity, (int)first, (int)n};
    hipLaunchKernelGGL(kv8_read_kernel, dim3((unsigned)n, (unsigned)B, 4), dim3(256), 0, (hipStream_t)stream, a);
    return launched();
}
