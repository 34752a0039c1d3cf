// Device helpers shared by the kernels over 4-bit codes with group scales: a unit's scales and zero
// points, the exact f16 form of the codes, and the f16 parts of activations.
#pragma once

#include "nnq_device.h"
#include "nnq_internal.h"

namespace nnq {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// A buffer: a lane's offset in a vector register, the uniform one in a scalar one.  (An offset of the
// lane past its end reads zeros.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)min(bytes, (int64_t)0x7FFFFFF0), 0x00020000);
}
// 16 bytes a lane from a buffer straight into LDS: the wave's 64 pieces land one after another at `lds`.
// (The host pass has no such builtin and would drop the kernels' launch stubs.)
__device__ __forceinline__ void copy16_lds(__amdgpu_buffer_rsrc_t t, uint8_t *lds, int voff, int soff) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(t, (__attribute__((address_space(3))) void *)lds, 16, voff, soff, 0, 0);
#endif
}
// a row's GS scales (16 bits each) at ls and zero points (8 bits each) at lz of the unit record at `at`;
// AUX: the cache policy (2: non-temporal).  WORD: the zero points' whole aligned word (widening a byte of
// it would wait for it in the next round of a loop that loads ahead).
template <int GS, bool Z, int AUX, bool WORD>
__device__ __forceinline__ void load_scales(__amdgpu_buffer_rsrc_t t, int ls, int lz, int at, uint32_t (&s)[(GS + 1) / 2],
                                            uint32_t &z) {
    if constexpr (GS == 1) {
        s[0] = __builtin_amdgcn_raw_buffer_load_b16(t, ls, at, AUX);
        if constexpr (Z && !WORD) z = __builtin_amdgcn_raw_buffer_load_b8(t, lz, at, AUX);
    } else if constexpr (GS == 2) {
        s[0] = __builtin_amdgcn_raw_buffer_load_b32(t, ls, at, AUX);
        if constexpr (Z && !WORD) z = __builtin_amdgcn_raw_buffer_load_b16(t, lz, at, AUX);
    } else {
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(t, ls, at, AUX));
        s[0] = v[0];
        s[1] = v[1];
        if constexpr (Z && !WORD) z = __builtin_amdgcn_raw_buffer_load_b32(t, lz, at, AUX);
    }
    if constexpr (Z && WORD) z = __builtin_amdgcn_raw_buffer_load_b32(t, lz & ~3, at, AUX);
}

// all ones where scales are bf16, zero where they are f16, in a vector register: selecting by a scalar
// condition would become branches between the MFMAs
__device__ __forceinline__ uint32_t scale_mask(int bf16) {
    uint32_t m = bf16 ? 0xFFFFFFFFu : 0u;
    asm("" : "+v"(m));
    return m;
}
template <int N>
__device__ __forceinline__ float group_scale(const uint32_t (&s)[N], int g, uint32_t mask) {
    const uint32_t h = s[g >> 1] >> (16 * (g & 1));
    const uint32_t b = (g & 1) ? s[g >> 1] & 0xFFFF0000u : h << 16, f = __float_as_uint(f16_to_f32(h & 0xFFFFu));
    return __uint_as_float((b & mask) | (f & ~mask));
}

__device__ __forceinline__ uint32_t pk_add(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, a) + __builtin_bit_cast(half2v, b));
}

// -(1024 + z) and -(64 + z) as packed f16 (z = 8 without zero points), for byte g of zs: byte 0xE4 over
// the zero point is the first, and adding 960 to it the second, exactly.  `sel` selects byte 0.
constexpr uint32_t kZeroSel = 0x04000400u;
template <bool Z>
__device__ __forceinline__ void zero_consts(uint32_t zs, int g, uint32_t &c1, uint32_t &c2, uint32_t sel = kZeroSel) {
    if constexpr (Z) {
        c1 = __builtin_amdgcn_perm(0xE4E4E4E4u, zs, sel + 0x00010001u * (uint32_t)g);
        c2 = pk_add(c1, 0x63806380u);
    } else {
        c1 = 0xE408E408u;
        c2 = 0xD480D480u;
    }
}

// The masks and exponents of the codes' f16 form: held in registers (one scalar source per
// instruction, and no literals in three-operand ones), an AND and an OR are one instruction.
struct CodeMasks {
    uint32_t lo, hi, e1, e2;
    __device__ __forceinline__ CodeMasks() {
        asm("s_mov_b32 %0, 0x000f000f" : "=s"(lo));
        asm("s_mov_b32 %0, 0x00f000f0" : "=s"(hi));
        asm("v_mov_b32 %0, 0x64006400" : "=v"(e1));
        asm("v_mov_b32 %0, 0x54005400" : "=v"(e2));
    }
};

// codes 2i and 2i + 1 of a word -> q - z as f16; all eight in column order
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i, uint32_t c1, uint32_t c2, const CodeMasks &k) {
    const uint32_t v = i < 2 ? w : w >> 8;
    return i & 1 ? pk_add((v & k.hi) | k.e2, c2) : pk_add((v & k.lo) | k.e1, c1);
}
__device__ __forceinline__ u32x4 codes_f16(uint32_t w, uint32_t c1, uint32_t c2, const CodeMasks &k) {
    return u32x4{code_pair(w, 0, c1, c2, k), code_pair(w, 1, c1, c2, k), code_pair(w, 2, c1, c2, k),
                 code_pair(w, 3, c1, c2, k)};
}

typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max_u16(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, a), __builtin_bit_cast(ushort2v, b)));
}
// bf16 pairs as f16 under a power of two, in integers: a bf16 of exponent field e becomes an f16 of field
// e - E0 with the same 7 mantissa bits, where E0 = max(E - 29, 0) brings the row's largest magnitude
// (field E) into [2^14, 2^15).  Exact but for values below 2^-29 of that magnitude, which keep an error
// of at most that; subnormals convert exactly where they count (E0 = 0).  A row with a NaN or infinity
// (field 255) becomes NaN throughout.
struct Bf16Scale {
    uint32_t sub, nan;
    float back;  // 2^(E0 - 112): f16 value times back = bf16 value
    __device__ __forceinline__ explicit Bf16Scale(uint32_t largest) {  // bits of the largest magnitude
        const int e = (int)(largest >> 7), e0 = max(e - 29, 0);
        sub = (uint32_t)e0 * 0x00800080u;
        nan = e == 255 ? 0x7E007E00u : 0u;
        back = __uint_as_float((uint32_t)(e0 + 15) << 23);
    }
    __device__ __forceinline__ uint32_t f16(uint32_t x) const {
        const ushort2v d = __builtin_elementwise_sub_sat(__builtin_bit_cast(ushort2v, x & 0x7FFF7FFFu),
                                                         __builtin_bit_cast(ushort2v, sub));
        const ushort2v h = d << (unsigned short)3;
        return (x & 0x80008000u) | __builtin_bit_cast(uint32_t, h) | nan;
    }
    Bf16Scale() = default;
};

// v * s (s a power of two that brings it into f16's range) as f16, and with LO what that leaves, as f16
template <bool LO>
__device__ __forceinline__ void split8(const float (&v)[8], float s, u32x4 &hi, u32x4 &lo) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float p = v[2 * e] * s, q = v[2 * e + 1] * s;
        const _Float16 hp = (_Float16)p, hq = (_Float16)q;
        hi[e] = __builtin_bit_cast(uint32_t, half2v{hp, hq});
        if constexpr (LO) lo[e] = __builtin_bit_cast(uint32_t, half2v{(_Float16)(p - (float)hp), (_Float16)(q - (float)hq)});
    }
}

// let `kernel` take `bytes` of dynamic LDS on the current device
inline hipError_t allow_lds(const void *kernel, size_t bytes) {
    return bytes <= 65536 ? hipSuccess : hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

}  // namespace nnq
