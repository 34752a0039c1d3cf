// MXFP4 rows on gfx950: x = c * 2^(s - 127) with an e2m1 code c (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) for
// every column and an E8M0 byte s for every 32 columns of a row.  Quantization and its inverse, the device image of
// weights, and the linears of one to sixteen token rows:
//   y[t][r] = sum_k W[r][k] x[t][k] (+ bias[r]),  x as it is (bf16 products) or quantized to MXFP4 too.
//
// Image: 16-row tiles, per (tile, pair of units of 128 columns) one record of 2176 bytes: for each unit lane 16p + r's 16
// bytes, block p (columns 32p .. 32p + 31) of row r in column order; then 32 words of scales, word 16h + r's byte
// 2 (unit) + i that of block 2i + h of row r.  One 16-byte load a lane is the operand of one 16x16x128 block-scaled MFMA, of
// a 32x32x64 one (blocks 2i and 2i + 1 of 32 rows; the byte of its scales' word selected by the instruction), and,
// block by block turned into bf16, of four 16x16x32 bf16 MFMAs (their k order is that of the lanes, the same for both
// sides).  The unit that fills up the last pair holds zeros.
#include <algorithm>
#include <type_traits>

#include "nnq_device.h"
#include "nnq_internal.h"
#include "nnq_mxfp4.h"

namespace nnq {

namespace {

// ---- quantization ---------------------------------------------------------------------
// Bound: one read of x and one write of the codes.  A block of 32 columns belongs to 4 (bf16) or 8 (f32) adjacent
// lanes of 16 bytes each, so that loads and stores are contiguous over the wave; blocks do not cross rows, so
// contiguous rows are one array of blocks.
typedef u32x4 u32x4_2 __attribute__((aligned(2)));
typedef u32x4 u32x4_4 __attribute__((aligned(4)));
constexpr int kQuantPer = 4;  // 16-byte pieces of a thread
template <bool BF16>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const uint8_t *x, int64_t pieces, int64_t row_pieces,
                                                          int64_t row_bytes, int floor_rule, uint8_t *codes,
                                                          uint8_t *scales) {
    constexpr int G = BF16 ? 4 : 8;  // pieces of a block
    const int64_t first = (int64_t)blockIdx.x * (256 * kQuantPer) + threadIdx.x;
    u32x4 v[kQuantPer];
#pragma unroll
    for (int i = 0; i < kQuantPer; i++) {
        const int64_t at = first + i * 256;
        v[i] = u32x4{0, 0, 0, 0};
        if (at >= pieces) continue;  // (whole blocks: pieces is a multiple of G)
        const int64_t row = row_pieces ? at / row_pieces : 0;
        const uint8_t *p = x + row * row_bytes + (at - row * row_pieces) * 16;
        if constexpr (BF16) v[i] = *reinterpret_cast<const u32x4_2 *>(p);
        else v[i] = *reinterpret_cast<const u32x4_4 *>(p);
    }
#pragma unroll
    for (int i = 0; i < kQuantPer; i++) {
        uint32_t mx = mx_largest_bits<BF16>(mx_largest<BF16>(v[i], 0));
        mx = max(mx, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mx, 0xB1, 0xF, 0xF, true));
        mx = max(mx, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mx, 0x4E, 0xF, 0xF, true));
        if constexpr (!BF16) mx = max(mx, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mx, 0x141, 0xF, 0xF, true));
        const uint32_t byte = mx_scale_byte(mx, floor_rule);
        const int64_t at = first + i * 256;
        if (at >= pieces) continue;
        uint32_t q;
        if constexpr (BF16) {
            q = mx_codes_bf16x8(v[i], mx_scale(byte));
        } else {
            const float f[8] = {__uint_as_float(v[i][0]), __uint_as_float(v[i][1]), __uint_as_float(v[i][2]), __uint_as_float(v[i][3]), 0.f, 0.f, 0.f, 0.f};
            q = mx_codes_f32(f, mx_scale(byte));
        }
        if (byte == 255u) q = 0;
        if constexpr (BF16) reinterpret_cast<uint32_t *>(codes)[at] = q;
        else reinterpret_cast<uint16_t *>(codes)[at] = (uint16_t)q;
        if (at % G == 0) scales[at / G] = (uint8_t)byte;
    }
}

// where lane 16p + r of job (tile, unit; an even number of units a tile) finds its block's codes and scale
__device__ __forceinline__ int64_t mx_codes_at(int64_t job, int lane) { return (job >> 1) * kMxPair + (job & 1) * 1024 + 16 * lane; }
__device__ __forceinline__ int64_t mx_scale_at(int64_t job, int lane) {
    return (job >> 1) * kMxPair + 2048 + 4 * (16 * ((lane >> 4) & 1) + (lane & 15)) + 2 * (job & 1) + (lane >> 5);
}

// x rows (whole units) to the records of the image, for a product of 4-bit operands: lane 16p + r quantizes block p
// of row r, as a lane of the kernels below does.
template <bool BF16>
__global__ __launch_bounds__(256) void mx_quantize_image_kernel(const uint8_t *x, int64_t m, int64_t k, int64_t units,
                                                                int64_t jobs, int floor_rule, uint8_t *image) {
    constexpr int L = BF16 ? 4 : 8;
    const int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (job >= jobs) return;
    const int lane = threadIdx.x & 63;
    const int64_t row = job / units * kTile + (lane & 15), k0 = job % units * kMxUnit + 32 * (lane >> 4);
    u32x4 v[L];
#pragma unroll
    for (int i = 0; i < L; i++) v[i] = u32x4{0, 0, 0, 0};
    if (row < m && k0 < k) {
        const u32x4 *p = reinterpret_cast<const u32x4 *>(x + (row * k + k0) * (BF16 ? 2 : 4));
#pragma unroll
        for (int i = 0; i < L; i++) v[i] = p[i];
    }
    uint32_t byte;
    const u32x4 q = mx_quantize_block<BF16>(v, floor_rule, byte);
    *reinterpret_cast<u32x4 *>(image + mx_codes_at(job, lane)) = q;
    image[mx_scale_at(job, lane)] = (uint8_t)byte;
}

// The image of codes and scales that are on the device; one wave per (tile, unit).  Rows and columns past the end:
// zeros.  bad (start: all ones; null: not asked): the lowest index of a scale byte over 252.
__global__ __launch_bounds__(256) void mx_repack_kernel(const uint8_t *codes, const uint8_t *scales, int64_t n, int64_t k,
                                                        int64_t units, int64_t jobs, uint8_t *image, unsigned long long *bad) {
    const int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (job >= jobs) return;
    const int lane = threadIdx.x & 63;
    const int64_t row = job / units * kTile + (lane & 15), k0 = job % units * kMxUnit + 32 * (lane >> 4);
    u32x4 q = {0, 0, 0, 0};
    uint32_t s = 0;
    if (row < n && k0 < k) {
        q = *reinterpret_cast<const u32x4_2 *>(codes + row * (k / 2) + k0 / 2);
        const int64_t at = row * (k / 32) + k0 / 32;
        s = scales[at];
        if (bad && s > kMxScaleMax) atomicMin(bad, (unsigned long long)at);
    }
    *reinterpret_cast<u32x4 *>(image + mx_codes_at(job, lane)) = q;
    image[mx_scale_at(job, lane)] = (uint8_t)s;
}

// rows of codes -> values (f32 or bf16), eight of them a thread; exact but for f32 subnormals below bf16's 2^-133,
// which no code reaches.  A block with scale byte 255 is NaN.
template <bool BF16>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint32_t *codes, const uint8_t *scales, int64_t words,
                                                            void *out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const u32x4 b = mx_codes_bf16(codes[i], mx_scale(scales[i >> 2]));
        if constexpr (BF16) {
            reinterpret_cast<u32x4 *>(out)[i] = b;
        } else {
            floatx4 lo, hi;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                lo[2 * e] = __uint_as_float(b[e] << 16);
                lo[2 * e + 1] = __uint_as_float(b[e] & 0xFFFF0000u);
                hi[2 * e] = __uint_as_float(b[2 + e] << 16);
                hi[2 * e + 1] = __uint_as_float(b[2 + e] & 0xFFFF0000u);
            }
            reinterpret_cast<floatx4 *>(out)[2 * i] = lo;
            reinterpret_cast<floatx4 *>(out)[2 * i + 1] = hi;
        }
    }
}

// the image's values, f32 [n, k]; one wave per (tile, unit)
__global__ __launch_bounds__(256) void mx_dequant_image_kernel(const uint8_t *image, int64_t n, int64_t k, int64_t units,
                                                               int64_t jobs, float *out) {
    const int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (job >= jobs) return;
    const int lane = threadIdx.x & 63;
    const int64_t row = job / units * kTile + (lane & 15), k0 = job % units * kMxUnit + 32 * (lane >> 4);
    if (row >= n || k0 >= k) return;
    const u32x4 q = ldg128(image + mx_codes_at(job, lane));
    const float s = mx_scale(image[mx_scale_at(job, lane)]);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const u32x4 b = mx_codes_bf16(q[j], s);
#pragma unroll
        for (int e = 0; e < 8; e++)
            out[row * k + k0 + 8 * j + e] = __uint_as_float(e & 1 ? b[e / 2] & 0xFFFF0000u : b[e / 2] << 16);
    }
}

// f32 x -> three bf16 planes whose sum is x: each the leading 8 bits (cut, not rounded) of what the ones before
// leave.  Exact down to bf16's smallest subnormal.  (An infinity leaves NaN in the later planes.)
__device__ __forceinline__ void split3(float a, float b, uint32_t &h, uint32_t &m, uint32_t &l) {
    constexpr uint32_t kHigh = 0x07060302u;  // the high halves of two registers
    const uint32_t ab = __float_as_uint(a), bb = __float_as_uint(b);
    h = __builtin_amdgcn_perm(bb, ab, kHigh);
    const float ra = a - __uint_as_float(ab & 0xFFFF0000u), rb = b - __uint_as_float(bb & 0xFFFF0000u);
    const uint32_t rau = __float_as_uint(ra), rbu = __float_as_uint(rb);
    m = __builtin_amdgcn_perm(rbu, rau, kHigh);
    const float la = ra - __uint_as_float(rau & 0xFFFF0000u), lb = rb - __uint_as_float(rbu & 0xFFFF0000u);
    l = __builtin_amdgcn_perm(__float_as_uint(lb), __float_as_uint(la), kHigh);
}
__global__ __launch_bounds__(256) void mx_split_kernel(const float *x, int64_t count4, int64_t plane, uint16_t *out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count4; i += (int64_t)gridDim.x * 256) {
        const floatx4 v = reinterpret_cast<const floatx4 *>(x)[i];
        u32x2 h, m, l;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            uint32_t a, b, c;
            split3(v[2 * e], v[2 * e + 1], a, b, c);
            h[e] = a;
            m[e] = b;
            l[e] = c;
        }
        *reinterpret_cast<u32x2 *>(out + 4 * i) = h;
        *reinterpret_cast<u32x2 *>(out + plane + 4 * i) = m;
        *reinterpret_cast<u32x2 *>(out + 2 * plane + 4 * i) = l;
    }
}

// ---- one to sixteen token rows ----------------------------------------------------------
// Bound: the weight stream from HBM (17 / 32 of a byte for each weight), read once for all token rows.  A workgroup of
// up to 16 waves owns blocks of R tiles; wave w takes units w, w + waves, ..; the next step's loads are in flight
// while the current one is computed.  The waves' sums meet in LDS, one barrier per block of tiles.
// x: X_BF16 bf16 rows; X_TRI up to five f32 rows, row t as the MFMA's rows 3t .. 3t + 2 (the three bf16 planes above);
// X_PLANES three planes of bf16 rows; X_Q16 / X_Q32 rows to be quantized, each lane its own block; X_CODES codes and
// scales given.
enum { X_BF16, X_TRI, X_PLANES, X_Q16, X_Q32, X_CODES };
constexpr bool mx_both(int xf) { return xf >= X_Q16; }
constexpr int kTriRow = 272;  // LDS bytes of a plane's row of a unit (256 and a shift of the banks)
constexpr int kTriBuf = 16 * kTriRow;

__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
template <int CTRL>
__device__ __forceinline__ float row_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ uint64_t mx_argmax_key(float v, uint32_t idx) {
    if (v != v) return ~0ull;
    const uint32_t b = __float_as_uint(v);
    return ((uint64_t)((b & 0x80000000u) ? ~b : (b | 0x80000000u)) << 32) | (0xFFFFFFFFu - idx);
}

// the operands of a unit
template <int XF>
struct XOp {
    static constexpr int P = XF == X_PLANES ? 3 : 1;
    u32x4 a[mx_both(XF) ? 1 : P][mx_both(XF) ? 1 : 4];
    uint32_t s;
};

// (columns from k on, and rows past m: zeros)
template <int XF>
__device__ __forceinline__ void load_operand(const MxArgs &a, __amdgpu_buffer_rsrc_t rx, __amdgpu_buffer_rsrc_t rs, int u,
                                             int ue, int lane, uint8_t *buf, XOp<XF> &x) {
    const int r = lane & 15, k0 = u * kMxUnit + 32 * (lane >> 4);
    const bool in = r < (int)a.m && k0 < (int)a.k && u < ue;
    const int el = r * (int)a.k + k0;
    auto ld = [&](int off, int at) { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rx, off, at, 0)); };
    if constexpr (XF == X_BF16 || XF == X_PLANES) {
#pragma unroll
        for (int p = 0; p < XOp<XF>::P; p++)
#pragma unroll
            for (int q = 0; q < 4; q++) x.a[p][q] = ld(in ? 2 * el : 0x7FFFFFF0, 2 * p * (int)(a.m * a.k) + 16 * q);
    } else if constexpr (XF == X_TRI) {
        // lane l splits columns 2l, 2l + 1 of every row; row 3t + p of the buffer is plane p of token t
        const int c = u * kMxUnit + 2 * lane;
#pragma unroll
        for (int t = 0; t < 5; t++) {
            if (t >= (int)a.m) break;
            const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rx, c < (int)a.k && u < ue ? 4 * (t * (int)a.k + c) : 0x7FFFFFF0, 0, 0));
            uint32_t h, m, l;
            split3(__uint_as_float(v[0]), __uint_as_float(v[1]), h, m, l);
            uint32_t *o = reinterpret_cast<uint32_t *>(buf + 3 * t * kTriRow) + lane;
            o[0] = h;
            o[kTriRow / 4] = m;
            o[kTriRow / 2] = l;
        }
        wave_sync();
        // (rows past the tokens' read what the buffer holds: rows are independent, theirs are not stored)
#pragma unroll
        for (int q = 0; q < 4; q++) x.a[0][q] = *reinterpret_cast<const u32x4 *>(buf + r * kTriRow + 64 * (lane >> 4) + 16 * q);
        wave_sync();
    } else if constexpr (XF == X_CODES) {
        x.a[0][0] = ld(in ? el / 2 : 0x7FFFFFF0, 0);
        x.s = __builtin_amdgcn_raw_buffer_load_b8(rs, in ? el / 32 : 0x7FFFFFF0, 0, 0);
    } else {
        constexpr bool B = XF == X_Q16;
        u32x4 v[B ? 4 : 8];
#pragma unroll
        for (int i = 0; i < (B ? 4 : 8); i++) v[i] = ld(in ? el * (B ? 2 : 4) : 0x7FFFFFF0, 16 * i);
        x.a[0][0] = mx_quantize_block<B>(v, a.floor_rule, x.s);
    }
}

// Part kp = blockIdx.x % ks of the units, in passes of waves * UPW units, over blocks blockIdx.x / ks, + gridDim.x / ks,
// .. of R tiles.
template <int XF, int R, int UPW>
__global__ __launch_bounds__(1024) void mx_rows_kernel(MxArgs a) {
    constexpr bool BOTH = mx_both(XF);
    constexpr int P = XOp<XF>::P;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)(blockDim.x >> 6);
    // LDS: (X_TRI) a staging buffer a wave, then two reduction buffers [tile][MFMA row][column][17 waves]
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    uint8_t *buf = lds + wv * kTriBuf;
    float *red = reinterpret_cast<float *>(lds + (XF == X_TRI ? waves * kTriBuf : 0));
    const int m = (int)a.m, units = (int)a.units;
    const int rows = XF == X_TRI ? 3 * m : m;  // MFMA rows that count
    const int ks = a.ks, kp = (int)blockIdx.x % ks, step = (int)gridDim.x / ks;
    const int ub = (int)((int64_t)units * kp / ks), ue = (int)((int64_t)units * (kp + 1) / ks);
    const int npass = (ue - ub + waves * UPW - 1) / (waves * UPW);
    const int nblock = (int)((a.ntile + R - 1) / R);
    const int c = lane & 15, p4 = lane >> 4;
    const int64_t xel = a.m * a.k;
    const __amdgpu_buffer_rsrc_t rx = rsrc(a.x, XF == X_CODES ? xel / 2 : XF == X_PLANES ? 6 * xel : XF == X_BF16 || XF == X_Q16 ? 2 * xel : 4 * xel);
    const __amdgpu_buffer_rsrc_t rs = rsrc(a.xs, XF == X_CODES ? xel / 32 : 0);
    XOp<XF> x[UPW];
    u32x4 wq[R][UPW];
    uint32_t ws[R][UPW];
    const int64_t tile_bytes = (int64_t)((units + 1) / 2) * kMxPair;
    const int ls = 2048 + 4 * (16 * (p4 & 1) + c) + (p4 >> 1);
    // a unit that does not exist is read at the last that does (its x is zeros), a tile that does not exist as a
    // buffer of no bytes
    auto tile_buffer = [&](int b, int r) {
        const int64_t tile = (int64_t)b * R + r;
        return rsrc(a.w + min(tile, a.ntile - 1) * tile_bytes, tile < a.ntile ? tile_bytes : 0);
    };
    auto load_w = [&](__amdgpu_buffer_rsrc_t t, int pass, int r, int j) {
        const int u = min(ub + (pass * UPW + j) * waves + wv, ue - 1), at = (u >> 1) * kMxPair;
        wq[r][j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(t, 16 * lane, at + (u & 1) * 1024, 2));
        ws[r][j] = __builtin_amdgcn_raw_buffer_load_b8(t, ls, at + 2 * (u & 1), 2);
    };
    auto load_x = [&](int pass) {
#pragma unroll
        for (int j = 0; j < UPW; j++) load_operand<XF>(a, rx, rs, ub + (pass * UPW + j) * waves + wv, ue, lane, buf, x[j]);
    };
    uint64_t key = 0;
    int b = (int)blockIdx.x / ks, par = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const __amdgpu_buffer_rsrc_t t = tile_buffer(b, r);
#pragma unroll
        for (int j = 0; j < UPW; j++) load_w(t, 0, r, j);
    }
    load_x(0);
    for (; b < nblock; b += step) {
        floatx4 acc[R];
#pragma unroll
        for (int r = 0; r < R; r++) acc[r] = floatx4{0.f, 0.f, 0.f, 0.f};
        for (int pass = 0; pass < npass; pass++) {
            // the next step: the next pass, or the next block's first; a unit's registers are loaded for it as soon as
            // they have been used
            const bool last = pass + 1 == npass;
            const int nb = last ? b + step : b, np = last ? 0 : pass + 1;
#pragma unroll
            for (int r = 0; r < R; r++) {
                const __amdgpu_buffer_rsrc_t t = tile_buffer(nb, r);
#pragma unroll
                for (int j = 0; j < UPW; j++) {
                    if constexpr (BOTH) {
                        acc[r] = mfma_mx16(x[j].a[0][0], x[j].s, wq[r][j], ws[r][j], acc[r]);
                    } else {
                        const float s = mx_scale(ws[r][j]);
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const u32x4 bq = mx_codes_bf16(wq[r][j][q], s);
                            // (the lo plane first: added to a finished hi sum its low bits would be cut off)
#pragma unroll
                            for (int p = P - 1; p >= 0; p--) acc[r] = mfma16x16x32_bf16(x[j].a[p][q], bq, acc[r]);
                        }
                    }
                    load_w(t, np, r, j);
                }
            }
            if (npass > 1 && nb < nblock) load_x(np);
        }
        float *rb = red + par * R * 16 * 272;
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (4 * p4 + i < rows) rb[((r * 16 + 4 * p4 + i) * 16 + c) * 17 + wv] = acc[r][i];
        __syncthreads();  // also: every wave is past its reads of the other buffer
        // a wave takes four outputs at a time, a wave's part of each to a lane of 16
        for (int i = wv; i < R * m * 4; i += waves) {
            int r = 0, t = i >> 2;
#pragma unroll
            for (int q = 1; q < R; q++)
                if (t >= m) r++, t -= m;
            const int col = 4 * (i & 3) + p4;
            const float *o = rb + (r * 16 * 16 + col) * 17 + c;
            float v = 0.f;
            if (c < waves) {
                if constexpr (XF == X_TRI) v = (o[(3 * t + 2) * 272] + o[(3 * t + 1) * 272]) + o[3 * t * 272];
                else v = o[t * 272];
            }
            v = row_add<0xB1>(v);
            v = row_add<0x4E>(v);
            v = row_add<0x141>(v);
            v = row_add<0x140>(v);
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
                if (a.argmax_partial) key = max(key, mx_argmax_key(v, (uint32_t)row));
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
int rows_waves(const MxArgs &a) {
    const int64_t part = (a.units + a.ks - 1) / a.ks;
    int waves = 16;
    while (waves > 4 && waves / 2 >= part) waves /= 2;
    return waves;
}

template <int XF, int R, int UPW>
int launch_rows_t(const MxArgs &a, void *stream) {
    const int waves = rows_waves(a);  // the chip holds 16 / waves workgroups per CU
    const int64_t blocks = (a.ntile + R - 1) / R;
    const int64_t grid = std::min<int64_t>(blocks, std::max<int64_t>(1, (int64_t)cus() * (16 / waves) / a.ks)) * a.ks;
    const size_t lds = (size_t)(XF == X_TRI ? waves * kTriBuf : 0) + 2 * R * 16 * 272 * 4;
    if (a.argmax_count) *a.argmax_count = grid;
    auto *kernel = mx_rows_kernel<XF, R, UPW>;
    hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), lds);
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(waves * 64), lds, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

template <int XF>
int launch_rows_x(const MxArgs &a, void *stream) {
    const bool two = a.ntile > 2 * (int64_t)cus() * (16 / rows_waves(a));
    // (two units of three planes have no registers)
    if (XF == X_PLANES || (a.units + a.ks - 1) / a.ks <= 16) return two ? launch_rows_t<XF, 2, 1>(a, stream) : launch_rows_t<XF, 1, 1>(a, stream);
    if constexpr (XF != X_PLANES) return two ? launch_rows_t<XF, 2, 2>(a, stream) : launch_rows_t<XF, 1, 2>(a, stream);
    return (int)hipErrorInvalidValue;
}

unsigned wave_jobs(int64_t jobs) { return (unsigned)((jobs + 3) / 4); }

}  // namespace

int launch_mx_quantize(const void *x, int x_bf16, int64_t rows, int64_t k, int64_t row_stride, int floor_rule,
                       uint8_t *codes, uint8_t *scales, void *stream) {
    const int64_t el = x_bf16 ? 2 : 4, pieces = rows * k * el / 16, grid = (pieces + 256 * kQuantPer - 1) / (256 * kQuantPer);
    if (grid > INT32_MAX) return (int)hipErrorInvalidValue;
    const int64_t row_pieces = row_stride == k ? 0 : k * el / 16;
    if (x_bf16)
        hipLaunchKernelGGL(mx_quantize_kernel<true>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream,
                           reinterpret_cast<const uint8_t *>(x), pieces, row_pieces, row_stride * el, floor_rule, codes, scales);
    else
        hipLaunchKernelGGL(mx_quantize_kernel<false>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream,
                           reinterpret_cast<const uint8_t *>(x), pieces, row_pieces, row_stride * el, floor_rule, codes, scales);
    return (int)hipGetLastError();
}

int launch_mx_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t count, void *out, int out_bf16, void *stream) {
    const int64_t words = count / 8;
    const dim3 grid((unsigned)std::min<int64_t>((words + 255) / 256, 65536)), block(256);
    const uint32_t *c = reinterpret_cast<const uint32_t *>(codes);
    if (out_bf16) hipLaunchKernelGGL(mx_dequantize_kernel<true>, grid, block, 0, (hipStream_t)stream, c, scales, words, out);
    else hipLaunchKernelGGL(mx_dequantize_kernel<false>, grid, block, 0, (hipStream_t)stream, c, scales, words, out);
    return (int)hipGetLastError();
}

int launch_mx_quantize_image(const void *x, int x_bf16, int64_t m, int64_t k, int floor_rule, uint8_t *image, void *stream) {
    const int64_t units = 2 * mx_pairs(k), jobs = mx_tiles(m) * units;
    if ((jobs + 3) / 4 > INT32_MAX) return (int)hipErrorInvalidValue;
    const uint8_t *p = reinterpret_cast<const uint8_t *>(x);
    if (x_bf16)
        hipLaunchKernelGGL(mx_quantize_image_kernel<true>, dim3(wave_jobs(jobs)), dim3(256), 0, (hipStream_t)stream, p, m, k, units, jobs, floor_rule, image);
    else
        hipLaunchKernelGGL(mx_quantize_image_kernel<false>, dim3(wave_jobs(jobs)), dim3(256), 0, (hipStream_t)stream, p, m, k, units, jobs, floor_rule, image);
    return (int)hipGetLastError();
}

int launch_mx_repack(const uint8_t *codes, const uint8_t *scales, int64_t n, int64_t k, uint8_t *image,
                     unsigned long long *bad, void *stream) {
    const int64_t units = 2 * mx_pairs(k), jobs = mx_tiles(n) * units;
    if ((jobs + 3) / 4 > INT32_MAX) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(mx_repack_kernel, dim3(wave_jobs(jobs)), dim3(256), 0, (hipStream_t)stream, codes, scales, n, k, units, jobs, image, bad);
    return (int)hipGetLastError();
}

int launch_mx_dequant_image(const Layout &L, const uint8_t *image, float *out, void *stream) {
    const int64_t units = 2 * mx_pairs(L.k), jobs = L.ntile * units;
    hipLaunchKernelGGL(mx_dequant_image_kernel, dim3(wave_jobs(jobs)), dim3(256), 0, (hipStream_t)stream, image, L.n, L.k, units, jobs, out);
    return (int)hipGetLastError();
}

int launch_mx_split(const float *x, int64_t count, uint16_t *planes, void *stream) {
    const int64_t n4 = count / 4;
    hipLaunchKernelGGL(mx_split_kernel, dim3((unsigned)std::min<int64_t>((n4 + 255) / 256, 16384)), dim3(256), 0, (hipStream_t)stream, x, n4, count, planes);
    return (int)hipGetLastError();
}

int launch_mx_rows(const MxArgs &g, void *scratch, void *stream) {
    MxArgs a = g;
    const MxRowsPlan p = mx_rows_plan(a.m, a.n, a.k, a.x_kind);
    if (a.m < 1 || a.m > kMxRows || a.units < 1 || a.ntile < 1 || (a.argmax_partial && (a.m != 1 || p.ks != 1)) || (p.bytes && !scratch))
        return (int)hipErrorInvalidValue;
    a.ks = p.ks;
    a.slabs = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(scratch) + p.slabs);
    int e = 0;
    if (a.x_kind == kMxF32 && p.planes) {
        e = launch_mx_split(reinterpret_cast<const float *>(a.x), a.m * a.k, reinterpret_cast<uint16_t *>(scratch), stream);
        if (e) return e;
        a.x = scratch;
        e = launch_rows_x<X_PLANES>(a, stream);
    } else {
        e = a.x_kind == kMxBf16  ? launch_rows_x<X_BF16>(a, stream)
            : a.x_kind == kMxF32 ? launch_rows_x<X_TRI>(a, stream)
            : a.x_kind == kMxQuantBf16 ? launch_rows_x<X_Q16>(a, stream)
            : a.x_kind == kMxQuantF32  ? launch_rows_x<X_Q32>(a, stream) : launch_rows_x<X_CODES>(a, stream);
    }
    if (e || a.ks == 1) return e;
    return launch_int4_sum(a.slabs, a.ks, a.m, a.n, a.bias, a.y, a.y_bf16, stream);
}

}  // namespace nnq
