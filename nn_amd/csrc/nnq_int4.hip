// Linear over 4-bit codes with group scales on gfx950, one to sixteen token rows per launch:
//   y[t][r] = sum_g s[r][g] * sum_{k in g} (q[r][k] - z[r][g]) * x[t][k]  (+ bias[r]),
// g the groups of 32, 64 or 128 columns of row r, z = 8 where no zero points are stored.
//
// Bound: the weight stream from HBM (n * k / 2 bytes of codes, 2 or 3 bytes per group), so the
// weight is read once for all token rows and everything else is kept small beside it:
//  * A workgroup of up to 16 waves owns blocks of R 16-row tiles; wave w takes units w,
//    w + waves, ... of 128 k.  One 16-byte load per lane is a unit of a tile, and exactly the
//    B operands of four 16x16x32 f16 MFMAs.  The next step's loads are in flight while the
//    current one is computed.
//  * x of a unit is scaled by a power of two per token row (its largest magnitude into
//    [2^14, 2^15)) to f16 (bf16 x; exact but for values below 2^-29 of that magnitude) or to an
//    f16 hi + lo pair (f32 x, ~22 bits), and passes through a wave-private LDS buffer into A
//    operands.  With K in one pass they stay in registers for all the workgroup's tiles.
//  * A code becomes an exact f16 integer: (w & 0x000F000F) | 0x6400.. is 1024 + q, and
//    (w & 0x00F000F0) | 0x5400.. is 64 + q in place, without a shift; one packed add takes off
//    1024 + z (64 + z), exactly.  Nine instructions make eight operands.  The integers are kept
//    normal: as f16 subnormals they would cost the matrix core's aligned sums low bits.
//  * Every product is exact in f32; a group's sum is scaled in f32 (one rounding for the scale,
//    one per addition).  The waves' sums meet in LDS, one barrier per block of tiles.
//  * Five rows and more of a long K split it over workgroups (int4_rows_split), and from some size on
//    the GEMM's two launches are shorter (int4_takes_rows).
// Measured (MI355X, in a graph, over copies of the weight that together pass the 256 MB Infinity Cache; in
// parentheses one weight again and again): 1 x 4096 -> 4096 5.6 us (5.5; 8.7 MB, an empty launch is 1.8), ->
// 24576 12.5 us (11.1), 4.2 TB/s, -> 151936 52 us (326 MB, 6.2 TB/s; the streaming read's rate is 7.0); 5
// f32 rows of 2880 -> 5751 9.6 us (9.2); 12 bf16 rows of 12288 -> 4096 16.5 us (16.1) with the sum: reading
// and converting x in every workgroup (25 MB from L2) before its first tile, and the second launch.
#include <algorithm>
#include <type_traits>

#include "nnq_device.h"
#include "nnq_int4.h"
#include "nnq_internal.h"

namespace nnq {

namespace {

// The raw bytes of one unit of a tile in the lane that holds row lane % 16.
template <int GS, bool Z>
struct Unit {
    u32x4 q;
    uint32_t s[(GS + 1) / 2];  // GS scales (16 bits each)
    uint32_t z;                // GS zero points (8 bits each)
};

// (the weight stream non-temporal; lq = 16 lane, and the offsets of the row's scales and zero points)
template <int GS, bool Z>
__device__ __forceinline__ void load_unit(__amdgpu_buffer_rsrc_t t, int lq, int ls, int lz, int at, Unit<GS, Z> &u) {
    u.q = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(t, lq, at, 2));
    load_scales<GS, Z, 2, false>(t, ls, lz, at, u.s, u.z);
}

__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int CTRL>
__device__ __forceinline__ uint32_t umax_row(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
    return v > o ? v : o;
}

template <int CTRL>
__device__ __forceinline__ float add_row(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}

// token rows and A operand planes: bf16 x, 16 rows; f32 x, 8 tokens as row pairs (hi, lo); f32 x, 16
// tokens as two planes (lo, hi)
enum { XBF16 = 0, XPAIR = 1, XPLANES = 2 };
constexpr int planes(int xf) { return xf == XPLANES ? 2 : 1; }

// x of one pass as loaded: lane 16i + c holds columns 8c .. 8c + 7 of rows i, 4 + i, .. (IT of them) of
// each of the wave's units.
template <int XF, int IT, int UPW>
struct XRaw {
    static constexpr int XR = XF == XBF16 ? 1 : 2;  // 16-byte loads of 8 columns
    u32x4 r[IT][UPW][XR];
};
// (units u0, u0 + waves, ..; rows past m and columns from kend on are zeros.  K is a multiple of 32, so a
// lane's 8 columns are all in or all out.)
template <int XF, int IT, int UPW>
__device__ __forceinline__ void load_x(const Int4Args &a, __amdgpu_buffer_rsrc_t rx, int u0, int waves, int kend, int lane,
                                       XRaw<XF, IT, UPW> &x) {
    constexpr int XR = XRaw<XF, IT, UPW>::XR;
    const int c = lane & 15, i4 = lane >> 4, m = (int)a.m;
#pragma unroll
    for (int it = 0; it < IT; it++) {
        const int t = 4 * it + i4;
#pragma unroll
        for (int j = 0; j < UPW; j++) {
            const int k0 = (u0 + j * waves) * kInt4Unit + 8 * c;
            const int at = t < m && k0 < kend ? (t * (int)a.k + k0) * 2 * XR : 0x7FFFFFF0;
#pragma unroll
            for (int e = 0; e < XR; e++)
                x.r[it][j][e] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rx, at, 16 * e, 0));
        }
    }
}

// x of one pass -> A operands of its units' MFMAs (per plane) and the rows' power of two back (one for
// all the units); `buf` (4 KB) and `bk` (16 floats) are the wave's own.  No branches: rows past the
// tokens are zeros (a branch per row group would spill the operands).
template <int XF, int IT, int UPW>
__device__ __forceinline__ void stage_units(int lane, uint16_t *buf, float *bk, XRaw<XF, IT, UPW> &x,
                                            u32x4 (&A)[UPW][planes(XF)][4], float (&back)[4]) {
    constexpr int XR = XRaw<XF, IT, UPW>::XR;
    const int c = lane & 15, i4 = lane >> 4;
    u32x4(&raw)[IT][UPW][XR] = x.r;
    struct Scale {
        float s, back;
    };
    typename std::conditional<XF == XBF16, Bf16Scale, Scale>::type sc[IT];
#pragma unroll
    for (int it = 0; it < IT; it++) {
        // largest |x| of the row's columns as bits (NaN above infinity above every number)
        uint32_t mx = 0;
#pragma unroll
        for (int j = 0; j < UPW; j++)
#pragma unroll
            for (int e = 0; e < 4 * XR; e++) {
                if constexpr (XF == XBF16)
                    mx = pk_max_u16(mx, raw[it][j][0][e] & 0x7FFF7FFFu);
                else
                    mx = max(mx, raw[it][j][e / 4][e % 4] & 0x7FFFFFFFu);
            }
        if constexpr (XF == XBF16) mx = max(mx & 0xFFFFu, mx >> 16);
        mx = umax_row<0xB1>(mx);
        mx = umax_row<0x4E>(mx);
        mx = umax_row<0x141>(mx);
        mx = umax_row<0x140>(mx);
        if constexpr (XF == XBF16)
            sc[it] = Bf16Scale(mx);
        else
            f16_prescale(__uint_as_float(mx), sc[it].s, sc[it].back);
        const int t = 4 * it + i4;  // (the 16 lanes of a row store the same value)
        if constexpr (XF == XPAIR)
            *reinterpret_cast<float2 *>(bk + 2 * t) = float2{sc[it].back, sc[it].back};
        else
            bk[t] = sc[it].back;
    }
    // (the compiler would keep every row's masked values from above instead of masking them again)
#pragma unroll
    for (int it = 0; it < IT; it++)
#pragma unroll
        for (int j = 0; j < UPW; j++)
#pragma unroll
            for (int e = 0; e < XR; e++) asm volatile("" : "+v"(raw[it][j][e]));
    // unit by unit, plane by plane through the buffer: operand (j, p) of row r at 16-byte slot
    // (4j + p) * 16 + r, with c = 4j + p
    u32x4 *slot = reinterpret_cast<u32x4 *>(buf) + c * 16;
#pragma unroll
    for (int j = 0; j < UPW; j++)
#pragma unroll
        for (int pl = 0; pl < planes(XF); pl++) {
#pragma unroll
            for (int it = 0; it < IT; it++) {
                const int t = 4 * it + i4;
                u32x4 hi, lo;
                if constexpr (XF == XBF16) {
#pragma unroll
                    for (int e = 0; e < 4; e++) hi[e] = sc[it].f16(raw[it][j][0][e]);
                } else {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = __uint_as_float(raw[it][j][e / 4][e % 4]);
                    split8<true>(v, sc[it].s, hi, lo);
                }
                if constexpr (XF == XPAIR) {
                    slot[2 * t] = hi;
                    slot[2 * t + 1] = lo;
                } else {
                    slot[t] = XF == XPLANES && pl == 0 ? lo : hi;
                }
            }
            wave_fence();
            // rows past 4 IT read what the buffer holds: MFMA rows are independent, theirs are not stored
#pragma unroll
            for (int q = 0; q < 4; q++) A[j][pl][q] = reinterpret_cast<const u32x4 *>(buf)[(4 * q + i4) * 16 + c];
            wave_fence();
        }
    const floatx4 b4 = *reinterpret_cast<const floatx4 *>(bk + 4 * i4);
#pragma unroll
    for (int e = 0; e < 4; e++) back[e] = b4[e];
    wave_fence();
}

__device__ __forceinline__ uint64_t int4_argmax_key(float v, uint32_t idx) {
    if (v != v) return ~0ull;
    const uint32_t b = __float_as_uint(v);
    return ((uint64_t)((b & 0x80000000u) ? ~b : (b | 0x80000000u)) << 32) | (0xFFFFFFFFu - idx);
}

// Part kp = blockIdx.x % ks of K, in passes of waves * UPW units, over blocks blockIdx.x / ks, + gridDim.x
// / ks, ... of R tiles, for up to 4 IT token rows.
template <int XF, int IT, int GS, bool Z, int R, int UPW>
__global__ __launch_bounds__(1024) void int4_rows_kernel(Int4Args a) {
    constexpr int P = planes(XF), TOK = 4 * IT;  // tokens
    constexpr int UB = int4_unit_bytes(kInt4Unit / GS, Z);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)(blockDim.x >> 6);
    // LDS: per wave a 4 KB staging buffer and 16 floats, then two reduction buffers
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    uint16_t *buf = reinterpret_cast<uint16_t *>(lds + wv * 4096);
    float *bk = reinterpret_cast<float *>(lds + waves * 4096 + wv * 64);
    float *red = reinterpret_cast<float *>(lds + waves * (4096 + 64));
    const int m = (int)a.m, units = (int)a.units;
    const int ks = a.ks, kp = (int)blockIdx.x % ks, step = (int)gridDim.x / ks;
    const int ub = (int)((int64_t)units * kp / ks), ue = (int)((int64_t)units * (kp + 1) / ks);  // this part's units
    const int kend = (int)min(a.k, (int64_t)ue * kInt4Unit);
    const int npass = (ue - ub + waves * UPW - 1) / (waves * UPW);
    const int nblock = (int)((a.ntile + R - 1) / R);
    const int c = lane & 15, p4 = lane >> 4;

    const CodeMasks km;
    const uint32_t sm = scale_mask(a.scale_bf16);
    const __amdgpu_buffer_rsrc_t rx = rsrc(a.x, a.m * a.k * (XF == XBF16 ? 2 : 4));
    u32x4 A[UPW][P][4];
    float back[4];
    Unit<GS, Z> W[R][UPW];
    const int lq = 16 * lane, ls = 1024 + 2 * GS * c, lz = 1024 + 32 * GS + GS * c;
    // a unit that does not exist is read at the last that does (its A operands are zeros), a tile that does
    // not exist as a buffer of no bytes
    auto tile_buffer = [&](int b, int r) {
        const int64_t tile = (int64_t)b * R + r;
        return rsrc(a.w + (size_t)min(tile, a.ntile - 1) * units * UB, tile < a.ntile ? (int64_t)units * UB : 0);
    };
    auto load = [&](__amdgpu_buffer_rsrc_t t, int pass, int r, int j) {
        load_unit<GS, Z>(t, lq, ls, lz, min(ub + (pass * UPW + j) * waves + wv, ue - 1) * UB, W[r][j]);
    };
    uint64_t key = 0;
    int b = (int)blockIdx.x / ks, par = 0;
    auto x_of = [&](int pass, XRaw<XF, IT, UPW> &x) {
        load_x<XF, IT, UPW>(a, rx, ub + pass * UPW * waves + wv, waves, kend, lane, x);
    };
    // x before the weights: loads return in order, and x comes from L2
    XRaw<XF, IT, UPW> x;
    x_of(0, x);
#pragma unroll
    for (int r = 0; r < R; r++) {
        const __amdgpu_buffer_rsrc_t t = tile_buffer(b, r);
#pragma unroll
        for (int j = 0; j < UPW; j++) load(t, 0, r, j);
    }
    stage_units<XF, IT, UPW>(lane, buf, bk, x, A, back);
    if (IT == 1 && npass > 1) x_of(1, x);
    for (; b < nblock; b += step) {
        float sum[R][4];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) sum[r][i] = 0.f;
        for (int pass = 0; pass < npass; pass++) {
            // the next step: the next pass, or the next block's first; a unit's registers are loaded for it
            // as soon as they have been used
            const bool last = pass + 1 == npass;
            const int nb = last ? b + step : b, np = last ? 0 : pass + 1;
#pragma unroll
            for (int r = 0; r < R; r++) {
                const __amdgpu_buffer_rsrc_t t = tile_buffer(nb, r);
                float tot[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < UPW; j++) {
#pragma unroll
                    for (int g = 0; g < GS; g++) {
                        uint32_t c1, c2;
                        zero_consts<Z>(W[r][j].z, g, c1, c2);
                        u32x4 B[4 / GS];
#pragma unroll
                        for (int h = 0; h < 4 / GS; h++) B[h] = codes_f16(W[r][j].q[g * (4 / GS) + h], c1, c2, km);
                        floatx4 acc = {0.f, 0.f, 0.f, 0.f};
                        // (the lo plane first: added to a finished hi sum its low bits would be cut off)
#pragma unroll
                        for (int pl = 0; pl < P; pl++)
#pragma unroll
                            for (int h = 0; h < 4 / GS; h++)
                                acc = mfma16x16x32_f16(A[j][pl][g * (4 / GS) + h], B[h], acc);
                        const float s = group_scale(W[r][j].s, g, sm);
#pragma unroll
                        for (int i = 0; i < 4; i++) tot[i] = fmaf(s, acc[i], tot[i]);
                        // here: moved on, the sums would keep every group's `acc`
#pragma unroll
                        for (int i = 0; i < 4; i++) asm volatile("" : "+v"(tot[i]));
                    }
                    load(t, np, r, j);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) sum[r][i] = fmaf(back[i], tot[i], sum[r][i]);
            }
            // with K in one pass A stays.  With one row group the x of the pass after next is on its way
            // while the next is computed; more have no registers for that
            if (npass > 1 && nb < nblock) {
                if constexpr (IT > 1) {
                    XRaw<XF, IT, UPW> xn;
                    x_of(np, xn);
                    stage_units<XF, IT, UPW>(lane, buf, bk, xn, A, back);
                } else {
                    stage_units<XF, IT, UPW>(lane, buf, bk, x, A, back);
                    x_of(np + 1 < npass ? np + 1 : 0, x);
                }
            }
        }
        // lane 16p + c: rows 4p .. 4p + 3 of output column c, for each tile -> [tile][token][column][17 waves]
        float *rb = red + par * R * TOK * 272;
#pragma unroll
        for (int r = 0; r < R; r++) {
            float *o = rb + (r * TOK * 16 + c) * 17 + wv;
            if constexpr (XF == XPAIR) {
                if (2 * p4 < m) o[(2 * p4) * 272] = sum[r][0] + sum[r][1];
                if (2 * p4 + 1 < m) o[(2 * p4 + 1) * 272] = sum[r][2] + sum[r][3];
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (4 * p4 + i < m) o[(4 * p4 + i) * 272] = sum[r][i];
            }
        }
        __syncthreads();  // also: every wave is past its reads of the other buffer
        // a wave takes four outputs at a time, a wave's part of each to a lane of 16
        for (int i = wv; i < R * m * 4; i += waves) {
            int r = 0, t = i >> 2;
#pragma unroll
            for (int q = 1; q < R; q++)
                if (t >= m) r++, t -= m;
            const int col = 4 * (i & 3) + p4;
            float v = c < waves ? rb[((r * TOK + t) * 16 + col) * 17 + c] : 0.f;
            v = add_row<0xB1>(v);
            v = add_row<0x4E>(v);
            v = add_row<0x141>(v);
            v = add_row<0x140>(v);
            const int64_t row = ((int64_t)b * R + r) * kTile + col;
            if (c == 0 && row < a.n) {
                if (ks > 1) {
                    a.slabs[((int64_t)kp * m + t) * a.n + row] = v;
                    continue;
                }
                if (a.bias) v += a.bias[row];
                if (a.y_bf16)
                    reinterpret_cast<uint16_t *>(a.y)[t * a.n + row] = (uint16_t)f32_to_bf16_bits(v);
                else
                    reinterpret_cast<float *>(a.y)[t * a.n + row] = v;
                if (a.argmax_partial) key = max(key, int4_argmax_key(v, (uint32_t)row));
            }
        }
        par ^= 1;
    }
    if (a.argmax_partial) {
        // m = 1: lanes that stored outputs hold keys (0 elsewhere); one key per workgroup
        __syncthreads();
        unsigned long long *kr = reinterpret_cast<unsigned long long *>(red);
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)key, o, 64);
            key = other > key ? other : key;
        }
        if (lane == 0) kr[wv] = key;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < waves; w++) key = max(key, (uint64_t)kr[w]);
            a.argmax_partial[blockIdx.x] = key;
        }
    }
}

int cus() {
    static int n[64] = {0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (n[dev] == 0) {
        int c = 0;
        if (hipDeviceGetAttribute(&c, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || c <= 0) c = 256;
        n[dev] = c;  // concurrent first calls store the same value
    }
    return n[dev];
}

// a wave for every unit of a part of K, 4 to 16
int rows_waves(const Int4Args &a) {
    const int64_t part = (a.units + a.ks - 1) / a.ks;
    int waves = 16;
    while (waves > 4 && waves / 2 >= part) waves /= 2;
    return waves;
}

template <int XF, int IT, int GS, bool Z, int R, int UPW>
int launch_rows_t(const Int4Args &a, void *stream) {
    const int waves = rows_waves(a);  // the chip holds 16 / waves workgroups per CU
    const int64_t blocks = (a.ntile + R - 1) / R;
    const int64_t grid = std::min<int64_t>(blocks, std::max<int64_t>(1, (int64_t)cus() * (16 / waves) / a.ks)) * a.ks;
    const size_t lds = (size_t)waves * (4096 + 64) + 2 * R * 4 * IT * 272 * 4;
    if (a.argmax_count) *a.argmax_count = grid;
    auto *kernel = int4_rows_kernel<XF, IT, GS, Z, R, UPW>;
    hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), lds);
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(waves * 64), lds, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

template <int XF, int IT, int GS, bool Z>
int launch_rows_r(const Int4Args &a, void *stream) {
    if constexpr (XF == XPLANES) {
        return launch_rows_t<XF, IT, GS, Z, 1, 1>(a, stream);
    } else {
        // Two tiles at a time where every workgroup has more than two; up to 16 units a wave has one, not a
        // second that does not exist (us, R = 2: 1 x 2048 -> 151936 34 with one unit a wave, 56 with two,
        // 1024 -> 151936 20 and 30; R = 1: 2048 -> 4096 4.6 and 5.1; 8 x 2048 -> 12288 9.1 and 12.0).
        const bool two = a.ntile > 2 * (int64_t)cus() * (16 / rows_waves(a));
        if ((a.units + a.ks - 1) / a.ks <= 16)
            return two ? launch_rows_t<XF, IT, GS, Z, 2, 1>(a, stream) : launch_rows_t<XF, IT, GS, Z, 1, 1>(a, stream);
        return two ? launch_rows_t<XF, IT, GS, Z, 2, 2>(a, stream) : launch_rows_t<XF, IT, GS, Z, 1, 2>(a, stream);
    }
}

template <int XF, int IT>
int launch_rows_x(const Int4Args &a, void *stream) {
    if (a.zeros) {
        if (a.group == 128) return launch_rows_r<XF, IT, 1, true>(a, stream);
        if (a.group == 64) return launch_rows_r<XF, IT, 2, true>(a, stream);
        return launch_rows_r<XF, IT, 4, true>(a, stream);
    }
    if (a.group == 128) return launch_rows_r<XF, IT, 1, false>(a, stream);
    if (a.group == 64) return launch_rows_r<XF, IT, 2, false>(a, stream);
    return launch_rows_r<XF, IT, 4, false>(a, stream);
}

// Bit-exact decode: (q - z) has at most 5 bits and the scale 11, so the product is exact in f32.
// One wave per (tile, unit).
__global__ __launch_bounds__(256) void dequant_int4_kernel(const uint8_t *w, int64_t n, int64_t k, int64_t units,
                                                           int64_t jobs, int group, int zeros, int scale_bf16,
                                                           float *out) {
    const int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (job >= jobs) return;
    const int lane = threadIdx.x & 63, r = lane & 15, p = lane >> 4;
    const int gs = kInt4Unit / group;
    const uint8_t *rec = w + (size_t)job * int4_unit_bytes(group, zeros);
    const int64_t row = job / units * kTile + r;
    if (row >= n) return;
    const u32x4 q = ldg128(rec + 16 * lane);
    for (int j = 0; j < 4; j++) {
        const int64_t k0 = job % units * kInt4Unit + 32 * j + 8 * p;
        if (k0 >= k) break;
        const int g = 32 * j / group;
        const uint32_t h = reinterpret_cast<const uint16_t *>(rec + 1024)[r * gs + g];
        const float s = scale_bf16 ? bf16_to_f32(h) : f16_to_f32(h);
        const int z = zeros ? rec[1024 + 32 * gs + r * gs + g] : 8;
        for (int e = 0; e < 8; e++) {
            const int code = (int)((q[j] >> (4 * (e / 2) + 16 * (e & 1))) & 0xFu);
            out[row * k + k0 + e] = (float)(code - z) * s;
        }
    }
}

// The image of codes, scales and zero points that are on the device already; one wave per (tile, unit),
// lane 16p + r the 16 bytes of row r (rows and columns past the end: zeros).  bad[0], bad[1] and bad[2] (start:
// all ones): the lowest index of a scale that is not finite, of a zero point above 16 and of a bf16 scale that
// is too large.  Bound by HBM: it reads and writes the weight once (151936 x 4096: under 0.34 ms, the whole call).
__global__ __launch_bounds__(256) void int4_repack_kernel(const uint8_t *codes, const uint16_t *scales,
                                                          const uint8_t *zeros, int64_t n, int64_t k, int64_t units,
                                                          int64_t jobs, int group, int scale_bf16, uint8_t *w,
                                                          unsigned long long *bad) {
    const int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (job >= jobs) return;
    const int lane = threadIdx.x & 63, r = lane & 15, p = lane >> 4, gs = kInt4Unit / group;
    const int64_t row0 = job / units * kTile, u = job % units, row = row0 + r;
    uint8_t *rec = w + (size_t)job * int4_unit_bytes(group, zeros != nullptr);
    u32x4 q = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int64_t k0 = u * kInt4Unit + 32 * j + 8 * p;
        if (row >= n || k0 >= k) continue;
        const uint32_t c = *reinterpret_cast<const uint32_t *>(codes + row * (k / 2) + k0 / 2);  // column e at bits 4e
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) v |= ((c >> (8 * i)) & 0xFu) << (4 * i) | ((c >> (8 * i + 4)) & 0xFu) << (16 + 4 * i);
        q[j] = v;
    }
    *reinterpret_cast<u32x4 *>(rec + 16 * lane) = q;
    if (lane < kTile * gs) {
        const int64_t srow = row0 + lane / gs, g = u * gs + lane % gs, ngroup = k / group, at = srow * ngroup + g;
        const bool in = srow < n && g < ngroup;
        const uint32_t s = in ? scales[at] : 0u, ex = scale_bf16 ? 0x7F80u : 0x7C00u;
        if ((s & ex) == ex) atomicMin(bad, (unsigned long long)at);
        else if (scale_bf16 && (s & ex) >= kInt4ScaleLimit) atomicMin(bad + 2, (unsigned long long)at);
        reinterpret_cast<uint16_t *>(rec + 1024)[lane] = (uint16_t)s;
        if (zeros) {
            const uint32_t z = in ? zeros[at] : 0u;
            if (z > 16) atomicMin(bad + 1, (unsigned long long)at);
            rec[1024 + 32 * gs + lane] = (uint8_t)z;
        }
    }
}

}  // namespace

int launch_int4_repack(const Layout &L, const uint8_t *codes, const uint16_t *scales, const uint8_t *zeros, uint8_t *w,
                       unsigned long long *bad, void *stream) {
    const int64_t jobs = L.ntile * L.nblk;
    if ((jobs + 3) / 4 > INT32_MAX) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(int4_repack_kernel, dim3((unsigned)((jobs + 3) / 4)), dim3(256), 0, (hipStream_t)stream, codes,
                       scales, zeros, L.n, L.k, L.nblk, jobs, L.group, L.scale_bf16, w, bad);
    return (int)hipGetLastError();
}

int launch_int4_rows(const Int4Args &g, void *scratch, void *stream) {
    Int4Args a = g;
    a.ks = scratch ? int4_rows_split(a.m, a.n, a.k, a.x_bf16) : 1;
    a.slabs = reinterpret_cast<float *>(scratch);
    if (a.m < 1 || a.m > kInt4Rows || a.units < 1 || a.ntile < 1 || (a.argmax_partial && (a.m != 1 || a.ks != 1)))
        return (int)hipErrorInvalidValue;
    int e;
    if (a.x_bf16)
        e = a.m <= 4   ? launch_rows_x<XBF16, 1>(a, stream)
            : a.m <= 8 ? launch_rows_x<XBF16, 2>(a, stream) : launch_rows_x<XBF16, 4>(a, stream);
    else if (a.m <= 8)
        e = a.m <= 4 ? launch_rows_x<XPAIR, 1>(a, stream) : launch_rows_x<XPAIR, 2>(a, stream);
    else
        e = launch_rows_x<XPLANES, 4>(a, stream);
    if (e || a.ks == 1) return e;
    return launch_int4_sum(a.slabs, a.ks, a.m, a.n, a.bias, a.y, a.y_bf16, stream);
}

int launch_int4_dequant(const Layout &L, const uint8_t *w, float *out, void *stream) {
    const int64_t jobs = L.ntile * L.nblk;
    hipLaunchKernelGGL(dequant_int4_kernel, dim3((unsigned)((jobs + 3) / 4)), dim3(256), 0, (hipStream_t)stream, w, L.n,
                       L.k, L.nblk, jobs, L.group, L.zeros, L.scale_bf16, out);
    return (int)hipGetLastError();
}

}  // namespace nnq
