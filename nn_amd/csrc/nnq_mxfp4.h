// Device helpers shared by the kernels over MXFP4 rows: e2m1 codes (two to a byte, the even column in the low
// half) with an E8M0 scale for every 32 columns of a row.
#pragma once

#include "nnq_device.h"
#include "nnq_int4.h"
#include "nnq_internal.h"

namespace nnq {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// (the host pass has no such builtins and would drop the kernels' launch stubs)
// codes 2i and 2i + 1 of byte SEL of w times 2^(s - 127), s the exponent field of `scale`, as packed bf16.  Exact:
// at most two significant bits, and bf16 reaches from 2^-133 (subnormal) to 6 * 2^125.
template <int SEL>
__device__ __forceinline__ uint32_t mx_pair_bf16(uint32_t w, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
#else
    return 0;
#endif
}
__device__ __forceinline__ u32x4 mx_codes_bf16(uint32_t w, float scale) {  // eight codes, in column order
    return u32x4{mx_pair_bf16<0>(w, scale), mx_pair_bf16<1>(w, scale), mx_pair_bf16<2>(w, scale), mx_pair_bf16<3>(w, scale)};
}
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }  // (0: read as 2^-127)

// 16x16x128: lane 16p + r supplies block p (32 columns) of A's row r and of B's column r with their scales; lane l
// receives D[4 (l / 16) + i][l % 16].  32x32x64: lane 32h + r block h of row r; D[8 (i / 4) + 4h + i % 4][l % 32].
template <int BYTE>  // of the words of scales
__device__ __forceinline__ floatx4 mfma_mx16(u32x4 a, uint32_t sa, u32x4 b, uint32_t sb, floatx4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, BYTE, (int)sa, BYTE, (int)sb);
#else
    return c;
#endif
}

// ---- quantization of 32 values ------------------------------------------------------
// The scale byte of a block whose largest magnitude has the bits `mx`: ceil: the smallest 2^s with mx <= 6 * 2^s;
// floor: 2^(floor(log2 mx) - 2), where more than 6 * 2^s saturates.  From 0 to 252 (2^-127 .. 2^125), so that every
// value a code stands for is finite; 255 (NaN) where the block holds NaN or an infinity.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t mx, int floor_rule) {
    const int e = (int)((mx + (floor_rule ? 0u : 0x3FFFFFu)) >> 23) - 2;
    return mx >= 0x7F800000u ? 255u : (uint32_t)min(max(e, 0), 252);
}
// four pairs -> eight codes, to the nearest, halves to even, above 6 saturating
__device__ __forceinline__ uint32_t mx_codes_f32(const float (&v)[8], float scale) {
    uint32_t r = 0;
#if defined(__HIP_DEVICE_COMPILE__)
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
#endif
    return r;
}
__device__ __forceinline__ uint32_t mx_codes_bf16x8(u32x4 x, float scale) {
    uint32_t r = 0;
#if defined(__HIP_DEVICE_COMPILE__)
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)x[0]), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)x[1]), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)x[2]), scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)x[3]), scale, 3);
#endif
    return r;
}
// the bits of the largest magnitude of 16 bytes (NaN above infinity above every number), as f32
template <bool BF16>
__device__ __forceinline__ uint32_t mx_largest(u32x4 x, uint32_t mx) {
    if constexpr (BF16) {
#pragma unroll
        for (int e = 0; e < 4; e++) mx = pk_max_u16(mx, x[e] & 0x7FFF7FFFu);  // (two maxima, high and low half)
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) mx = max(mx, x[e] & 0x7FFFFFFFu);
    }
    return mx;
}
template <bool BF16>
__device__ __forceinline__ uint32_t mx_largest_bits(uint32_t mx) {
    return BF16 ? max(mx & 0xFFFFu, mx >> 16) << 16 : mx;
}
// a whole block in one lane: 4 (bf16) or 8 (f32) loads of 16 bytes -> 16 bytes of codes and the scale byte
template <bool BF16>
__device__ __forceinline__ u32x4 mx_quantize_block(const u32x4 (&x)[BF16 ? 4 : 8], int floor_rule, uint32_t &byte) {
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < (BF16 ? 4 : 8); i++) mx = mx_largest<BF16>(x[i], mx);
    byte = mx_scale_byte(mx_largest_bits<BF16>(mx), floor_rule);
    const float s = mx_scale(byte);
    u32x4 q;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (BF16) {
            q[i] = mx_codes_bf16x8(x[i], s);
        } else {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __uint_as_float(x[2 * i + e / 4][e % 4]);
            q[i] = mx_codes_f32(v, s);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) q[i] = byte == 255u ? 0u : q[i];
    return q;
}

}  // namespace nnq
