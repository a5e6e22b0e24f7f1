// The 8-bit K / V cache: number format and the per-lane steps that its writers and readers share.
//
// codes  uint8 [4][B][H][capacity][128]     (K_same, K_cross, V_same, V_cross; e4m3 values; a head's tokens lie together, so the 128
//                                            bytes of consecutive keys are one contiguous stream per (sequence, head))
// scales uint8 [4][B][H][capacity / block]  one power of two, 2^(byte - 127), for each block of `block` tokens (2^lg, 1..64) and head
//
// a = the largest finite |x| of the block = 2^n (1 + f); the scale is the smallest power of two with a <= 448 * 2^s (448 = the largest
// e4m3 number): s = n - 8 + [f > 3/4], not below -126.  Multiplying by a power of two is exact, so the ONLY rounding is the one to
// e4m3's 3 mantissa bits (round to nearest even): |x^ - x| <= max(2^-4 |x|, 2^-10 2^s).  Infinities saturate to +-448 2^s, NaN stays NaN.
#pragma once
#include "hip_common.hpp"

namespace libra {

constexpr int KV8_MAX_BLOCK = 64;

// bit pattern of |x| for the block maximum; infinities and NaN do not count
__device__ __forceinline__ unsigned kv8_abs_bits(float x) {
    const unsigned u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
// maximum over the 16 lanes of a DPP row (order-free: integer maximum of the bit patterns of non-negative floats)
template <int N>
__device__ __forceinline__ unsigned row_ror_max(unsigned x) {
    const unsigned r = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + N, 0xf, 0xf, false);
    return x > r ? x : r;
}
__device__ __forceinline__ unsigned row16_max(unsigned x) { return row_ror_max<1>(row_ror_max<2>(row_ror_max<4>(row_ror_max<8>(x)))); }
// scale byte of a block maximum's bit pattern (0x600000: mantissa of 1.75)
__device__ __forceinline__ int kv8_byte(unsigned amax_bits) {
    const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b > 1 ? b : 1;
}
__device__ __forceinline__ float kv8_scale(int byte) { return __uint_as_float((unsigned)byte << 23); }             // 2^(byte - 127)
__device__ __forceinline__ float kv8_inverse(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }   // 2^(127 - byte)

__device__ __forceinline__ float kv8_clamp(float y) { return y != y ? y : fminf(fmaxf(y, -448.f), 448.f); }
// 4 floats (already multiplied by the block's inverse scale) -> 4 codes
__device__ __forceinline__ unsigned kv8_encode4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(kv8_clamp(a), kv8_clamp(b), 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(kv8_clamp(c), kv8_clamp(d), w, true);
}
__device__ __forceinline__ void kv8_decode4(unsigned w, float* f) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = lo[0]; f[1] = lo[1]; f[2] = hi[0]; f[3] = hi[1];
}
// 4 codes of a block whose scale grows by the factor 1 / down (down = 2^(old - new) < 1): exact but for values that leave the normal range
__device__ __forceinline__ unsigned kv8_rescale4(unsigned w, float down) {
    float f[4];
    kv8_decode4(w, f);
    return kv8_encode4(f[0] * down, f[1] * down, f[2] * down, f[3] * down);
}
// The scale of a block that gets one more token (its `in_block`-th, 0 = the first; `need` = the byte that the token asks for, `old` = the
// byte that was there): -> the byte to use; where it grows, the codes of the earlier tokens - `in_block` * 128 contiguous bytes at `codes` -
// are re-expressed.  A 16-lane group does it (lane = 0..15), 16 tokens at a time with all their loads in flight: one round trip to
// memory instead of one a token.
__device__ __forceinline__ int kv8_grow(unsigned char* codes, int in_block, int need, int old, int lane) {
    if (in_block == 0) return need;
    old = min(old, 254);
    if (need <= old) return old;
    const float down = kv8_scale(max(127 + old - need, 0));
    const int bytes = in_block * 128;
    for (int at = lane * 16; at < bytes; at += 2048) {
        u32x4 w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) if (at + k * 256 < bytes) w[k] = *(const u32x4*)(codes + at + k * 256);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (at + k * 256 >= bytes) continue;
            u32x4 o;
#pragma unroll
            for (int i = 0; i < 4; ++i) { const unsigned x = w[k][i]; o[i] = kv8_rescale4(x, down); }
            *(u32x4*)(codes + at + k * 256) = o;
        }
    }
    return need;
}

}  // namespace libra
