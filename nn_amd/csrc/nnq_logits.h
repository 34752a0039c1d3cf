// Device helpers of the kernels that read rows of logits, 2048 of a row in a wave's registers: orders, sums over a wave,
// the exponential, and the candidates of a segment's largest.
#pragma once

#include "nnq_device.h"
#include "nnq_internal.h"

namespace nnq {

constexpr int kSeg = 2048;          // logits of a wave
constexpr int kPer = kSeg / 64;     // logits of a lane
constexpr float kNegInf = -__builtin_huge_valf();
constexpr uint32_t kOrdNegInf = 0x007FFFFFu;

__device__ __forceinline__ uint32_t ord(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 and +0 are equal logits
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unord(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o); }
// larger logits first, then lower indices; 0 is no candidate (ord(-inf) > 0)
__device__ __forceinline__ uint64_t cand_key(float v, uint32_t i) { return ((uint64_t)ord(v) << 32) | (0xFFFFFFFFu - i); }

template <class T>
__device__ __forceinline__ float widen(T h);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
struct Bf16 {
    uint16_t h;
};
struct F16 {
    uint16_t h;
};
template <>
__device__ __forceinline__ float widen<Bf16>(Bf16 v) { return bf16_to_f32(v.h); }
template <>
__device__ __forceinline__ float widen<F16>(F16 v) { return f16_to_f32(v.h); }

template <class T>
__device__ __forceinline__ void widen16(u32x4 r, float *x) {  // the elements of 16 bytes
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = __uint_as_float(r[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[2 * e] = widen<T>(T{(uint16_t)(r[e] & 0xFFFFu)});
            x[2 * e + 1] = widen<T>(T{(uint16_t)(r[e] >> 16)});
        }
    }
}

// Sum and maximum over the wave's 64 lanes, the same in every lane, without LDS: DPP within the rows
// of 16, lane swaps between them.  Every lane must be active.
template <int CTRL>
__device__ __forceinline__ uint32_t lane_of(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <class F>
__device__ __forceinline__ uint32_t across(uint32_t v, F &&f) {
    v = f(v, lane_of<0xB1>(v));   // lane ^ 1
    v = f(v, lane_of<0x4E>(v));   // lane ^ 2
    v = f(v, lane_of<0x141>(v));  // the other quad of 8
    v = f(v, lane_of<0x140>(v));  // the other half of 16
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(p[0], p[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(q[0], q[1]);
}
__device__ __forceinline__ float sum64(float v) {
    return __uint_as_float(across(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
__device__ __forceinline__ float max64(float v) {
    return __uint_as_float(across(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ uint32_t sum64u(uint32_t v) {
    return across(v, [](uint32_t a, uint32_t b) { return a + b; });
}

// e^d for d from -1e30 to 0, to a relative 2^-22 (below d = -87.3, where it would be subnormal, it may be 0).
// 2^p alone, with p = d log2(e) rounded, would be off by up to 2^-18 at d = -80: half a step of p, and the
// constant's own rounding, which moves every term the same way.  The factor that is missing is e^(d - p log(2)),
// 1 + a number below 2^-17; three FMAs beside the product and the exponential (301 rows with rank and
// alternatives: 41.3 -> 41.5 us the whole call, 512 without 55.5 -> 56.5).
__device__ __forceinline__ float exp_of(float d) {
    const float p = d * 1.44269504088896340736f, e = __builtin_amdgcn_exp2f(p);
    // log(2) in two parts: 0x1.62e43p-1 and what is left of it
    return fmaf(e, fmaf(p, 1.9046542e-9f, fmaf(p, -0x1.62e43p-1f, d)), e);
}

// The largest t with at least `want` lanes' or elements' keys >= t, count(t) counting them
// (non-increasing in t; count(0) >= want).
// BITS: only the leading ones are settled (a smaller t).
template <int BITS, class F>
__device__ __forceinline__ uint32_t largest_with(int want, F &&count) {
    uint32_t t = 0;
    for (uint32_t bit = 0x80000000u; bit >> (BITS == 32 ? 0 : 32 - BITS); bit >>= 1)
        if (count(t | bit) >= want) t |= bit;
    return t;
}

// The candidates of the `want` largest of a segment, as keys, at cand[0 .. slots) (0: none).  Element e of a lane is
// logit base + (e / V) * 64 V + e % V; lm: the lane's largest, -inf where there is no logit; list: 64 keys of LDS of the
// wave's own.  BITS: how many leading bits of the bound are settled; bf16 has 16.
template <int V, int BITS = 24>
__device__ __forceinline__ void segment_candidates(const float (&x)[kPer], float lm, int64_t base, int want, int slots, int lane,
                                                   uint64_t *list, uint64_t *cand) {
    const uint32_t mine = lm == lm ? ord(lm) : 0;  // (no number in the lane)
    // (its leading 24 bits do: a bound 2^-15 of its size below lets hardly more candidates in, also for
    // logits far from 0; with 16 bits 301 x 151936 logits around 300 took 114 us, 43 with 24)
    const uint32_t lanes = largest_with<BITS>(want, [&](uint32_t k) { return __popcll(__ballot(mine >= k)); });
    float t = unord(max(lanes, kOrdNegInf + 1));  // (-inf is no candidate)
    // the lane's candidates as bits, element 0 the highest
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < kPer; e++) bits = bits + bits + (x[e] >= t);
    const int total = (int)sum64u(__popc(bits));
    if (total > 64) {  // uniform
        // The exact N-th largest: the lanes' bound in all its bits where fewer logits lie above it (many
        // logits equal to it), else searched over the 2048.
        auto above = [&]() {
            int c = 0;
#pragma unroll
            for (int e = 0; e < kPer; e++) c += __popcll(__ballot(x[e] > t));
            return c;
        };
        t = unord(max(largest_with<32>(want, [&](uint32_t k) { return __popcll(__ballot(mine >= k)); }), kOrdNegInf + 1));
        int more = above();
        if (more >= want) {
            t = unord(largest_with<32>(want, [&](uint32_t k) {
                const float f = unord(k);
                int c = 0;
#pragma unroll
                for (int e = 0; e < kPer; e++) c += __popcll(__ballot(x[e] >= f));
                return c;
            }));
            more = above();
        }
        // of the logits equal to it the first want - more in index order
        uint32_t before = more;
        bits = 0;
#pragma unroll
        for (int v = 0; v < kPer / V; v++) {
            uint32_t at_lane = before;
#pragma unroll
            for (int e = 0; e < V; e++) {
                const uint64_t b = __ballot(x[v * V + e] == t);
                at_lane = __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, at_lane));
                before += __popcll(b);
            }
#pragma unroll
            for (int e = 0; e < V; e++) {
                const bool eq = x[v * V + e] == t;
                bits = bits + bits + (x[v * V + e] > t || (eq && at_lane < (uint32_t)want));
                at_lane += eq;
            }
        }
    }
    // a round takes one candidate of every lane that has any
    int listed = 0;
    while (__ballot(bits != 0)) {
        const uint64_t b = __ballot(bits != 0);
        const int e = bits ? __clz(bits) : 0;
        float v = x[0];
#pragma unroll
        for (int i = 1; i < kPer; i++) v = i == e ? x[i] : v;
        if (bits) {
            const int slot = listed + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
            if (slot < 64) list[slot] = cand_key(v, (uint32_t)(base + (e / V) * 64 * V + e % V));
        }
        listed += __popcll(b);
        bits &= ~(0x80000000u >> e);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const uint64_t key = lane < listed ? list[lane] : 0ull;
    int place = lane;
    if (listed > slots) {  // uniform: the largest `slots` of up to 64
        place = 0;
        for (int j = 0; j < listed; j++) place += list[j] > key;
        if (lane >= listed) place = slots;
    }
    if (place < slots) cand[place] = key;
}

}  // namespace nnq
