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
// Measured (MI355X): 2011 x 12288 f32 19 us, 5.8 TB/s, and its values back 17 us, 6.6 TB/s (a large copy moves 5.3); one
// row of 4096 1.4 us, an empty launch's time.
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
        // (quotients in 64 bits: 64 rows of 4096 apart from one another 3.0 us, 2.7 in 32)
        const int64_t row = !row_pieces ? 0 : pieces >> 32 ? at / row_pieces : (uint32_t)at / (uint32_t)row_pieces;
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
// of row r, so that nothing crosses lanes.  One wave a workgroup, so that few of them lie on all CUs (four: 0.3 to 0.5 us
// more).  (2048 x 4096 bf16 6.7 us, 301 x 2880 f32 3.4: the latter is two waves a CU.)
template <bool BF16>
__global__ __launch_bounds__(64) void mx_quantize_image_kernel(const uint8_t *x, int64_t m, int64_t k, int64_t units,
                                                               int floor_rule, uint8_t *image) {
    constexpr int L = BF16 ? 4 : 8;
    const int64_t job = (int64_t)blockIdx.x;
    const int lane = threadIdx.x;
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

// The image of codes and scales that are on the device: of a weight, and of quantized rows in each product of more than 16
// (2048 of 4096 -> 4096 28.2 us the call, 29.4 with x to be quantized); one wave per (tile, unit).  Rows and columns past the end:
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

// rows of codes -> values (f32 or bf16), 16 bytes of them a lane, four times: a wave's store is 1 KB without a gap, and only so
// do non-temporal ones pay (us of quantizing and decoding 2011 x 12288 f32: 38.9, plain stores 49.8, a lane's 32 bytes in a
// row non-temporal 59; 4096 x 4096 bf16 22.2 against 28.1).  Exact (f32 subnormals below bf16's 2^-133 are reached by no
// code).  A block with scale byte 255 is NaN.
template <bool BF16>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t *codes, const uint8_t *scales, int64_t pieces,
                                                            uint8_t *out) {
    constexpr int N = 4;
    const int64_t first = (int64_t)blockIdx.x * (256 * N) + threadIdx.x;
    uint32_t q[N], s[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int64_t at = min(first + i * 256, pieces - 1);
        if constexpr (BF16) q[i] = reinterpret_cast<const uint32_t *>(codes)[at];
        else q[i] = reinterpret_cast<const uint16_t *>(codes)[at];
        s[i] = scales[at / (BF16 ? 4 : 8)];
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int64_t at = first + i * 256;
        if (at >= pieces) return;
        const float sc = mx_scale(s[i]);
        u32x4 v;
        if constexpr (BF16) {
            v = mx_codes_bf16(q[i], sc);
        } else {
            const uint32_t lo = mx_pair_bf16<0>(q[i], sc), hi = mx_pair_bf16<1>(q[i], sc);
            v = u32x4{lo << 16, lo & 0xFFFF0000u, hi << 16, hi & 0xFFFF0000u};
        }
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(out + 16 * at));
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
// kw * nw waves takes nw tiles at a time; wave (i, j) sums pairs of units i, i + kw, .. of tile j, a step's pairs all
// in its registers, loaded for the next step as soon as they have been used.  x of the workgroup's
// part of K lies in LDS, as MFMA operands read it; the waves' sums meet there too, one barrier a step.
// Measured (MI355X, in a graph over copies of the weight that pass the Infinity Cache; in parentheses one weight again and
// again): 1 x 4096 -> 4096 5.5 us, -> 24576 14.1, 3.8 TB/s, -> 151936 66, 5.0 TB/s (loads alone, in this structure, 65); 1 f32 x
// 12288 -> 4096 11.0 (9.0); 12 x 4096 -> 24576 16.0 (13.9); in 4 bits 8 x 12288 -> 4096 12.6 (10.4): latency of the first
// loads, x of every workgroup from L2 (for 8 rows as many bytes as its weights) and the sums' barrier.  Two tiles a wave,
// x in registers and sums over all 16 waves were 20 to 40% slower beyond one row (12 x 4096 -> 24576 22.6).
// x: X_BF16 bf16 rows; X_TRI up to five f32 rows, row t as the MFMA's rows 3t .. 3t + 2 (the three bf16 planes above);
// X_PLANES more f32 rows, an MFMA for each plane; X_Q16 / X_Q32 rows to be quantized; X_CODES codes and scales given.
enum { X_BF16, X_TRI, X_PLANES, X_Q16, X_Q32, X_CODES };
constexpr bool mx_both(int xf) { return xf >= X_Q16; }
constexpr int kSumRow = 20;                       // floats of an MFMA row's 16 sums (and a shift of the banks)
constexpr int kSumWave = 16 * kSumRow * 4;        // bytes of a wave's sums of a tile

template <int CTRL>
__device__ __forceinline__ uint32_t row_lane(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ uint64_t mx_argmax_key(float v, uint32_t idx) {
    if (v != v) return ~0ull;
    const uint32_t b = __float_as_uint(v);
    return ((uint64_t)((b & 0x80000000u) ? ~b : (b | 0x80000000u)) << 32) | (0xFFFFFFFFu - idx);
}

// x in LDS.  bf16 rows (X_BF16: of the tokens, f32: 3t + plane) of `pairs` pairs of units and 16 bytes, so that the same
// columns of 16 rows lie in 16 different places of the banks; or rows of codes, 16 bytes a block and 16 more, and
// behind them words of scales in the image's order, [row][pair][2].
template <int XF>
struct XStage {
    static constexpr bool BOTH = mx_both(XF), F32 = XF == X_TRI || XF == X_PLANES;
    static constexpr int U = XF == X_BF16 ? 8 : F32 ? 3 : XF == X_Q16 ? 2 : XF == X_Q32 ? 1 : 4;  // pieces of a thread at a time
    static constexpr int L = XF == X_BF16 || XF == X_CODES ? 1 : F32 ? 2 : XF == X_Q16 ? 4 : 8;   // loads of a piece
    int pitch, pieces, row_pieces, k0;
    uint8_t *lds, *words;
    __amdgpu_buffer_rsrc_t rx, rs;
    u32x4 v[U][L];
    uint32_t s[XF == X_CODES ? U : 1];
    __device__ __forceinline__ XStage(const MxArgs &a, uint8_t *at) {
        const int64_t xel = a.m * a.k;
        rx = rsrc(a.x, XF == X_CODES ? xel / 2 : XF == X_BF16 || XF == X_Q16 ? 2 * xel : 4 * xel);
        rs = rsrc(a.xs, XF == X_CODES ? xel / 32 : 0);
        lds = at;
    }
    __device__ __forceinline__ void part(const MxArgs &a, int pair0, int pairs) {
        row_pieces = pairs * (BOTH ? 8 : 32);  // blocks, or 8 columns
        pieces = (int)a.m * row_pieces;
        pitch = pairs * (BOTH ? 128 : 512) + 16;
        k0 = pair0 * 2 * kMxUnit;
        words = lds + (int)a.m * pitch;
    }
    // (columns from K on: zeros)
    __device__ __forceinline__ void load(const MxArgs &a, int first) {
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int at = first + i * (int)blockDim.x, row = at / row_pieces, k = k0 + (at - row * row_pieces) * (BOTH ? 32 : 8);
            const int el = at < pieces && k < (int)a.k ? row * (int)a.k + k : -1;
            const int off = el < 0 ? 0x7FFFFFF0 : XF == X_CODES ? el / 2 : XF == X_BF16 || XF == X_Q16 ? 2 * el : 4 * el;
#pragma unroll
            for (int l = 0; l < L; l++) v[i][l] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rx, off, 16 * l, 0));
            if constexpr (XF == X_CODES) s[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, el < 0 ? 0x7FFFFFF0 : el / 32, 0, 0);
        }
    }
    __device__ __forceinline__ void store(const MxArgs &a, int first) {
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int at = first + i * (int)blockDim.x, row = at / row_pieces, piece = at - row * row_pieces;
            if (at >= pieces) continue;
            if constexpr (XF == X_BF16) {
                *reinterpret_cast<u32x4 *>(lds + row * pitch + 16 * piece) = v[i][0];
            } else if constexpr (F32) {
                u32x4 h, m, l;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t c[3];
                    split3(__uint_as_float(v[i][e / 2][2 * (e & 1)]), __uint_as_float(v[i][e / 2][2 * (e & 1) + 1]), c[0], c[1], c[2]);
                    h[e] = c[0];
                    m[e] = c[1];
                    l[e] = c[2];
                }
                uint8_t *o = lds + 3 * row * pitch + 16 * piece;
                *reinterpret_cast<u32x4 *>(o) = h;
                *reinterpret_cast<u32x4 *>(o + pitch) = m;
                *reinterpret_cast<u32x4 *>(o + 2 * pitch) = l;
            } else {
                u32x4 q = v[i][0];
                uint32_t byte = 0;
                if constexpr (XF == X_CODES) byte = s[i];
                else q = mx_quantize_block<XF == X_Q16>(v[i], a.floor_rule, byte);
                *reinterpret_cast<u32x4 *>(lds + row * pitch + 16 * piece) = q;
                // block 4 (unit) + 2i + h of a pair: word h, byte 2 (unit) + i
                words[row * row_pieces + (piece & ~7) + 4 * (piece & 1) + 2 * ((piece >> 2) & 1) + ((piece >> 1) & 1)] = (uint8_t)byte;
            }
        }
    }
    __device__ __forceinline__ void rest(const MxArgs &a, int first) {  // what one load does not hold
        for (int i = first + U * (int)blockDim.x; i < pieces; i += U * (int)blockDim.x) {
            load(a, i);
            store(a, i);
        }
    }
};

// Part kp = blockIdx.x % ks of the pairs, in chunks that LDS holds (as a rule one), over blocks blockIdx.x / ks, + gridDim.x
// / ks, .. of nw tiles.
template <int XF, int PP>
__global__ __launch_bounds__(1024) void mx_rows_kernel(MxArgs a) {
    constexpr bool BOTH = mx_both(XF);
    constexpr int P = XF == X_PLANES ? 3 : 1;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), kw = a.kw, nw = a.nw, wi = wv % kw, wj = wv / kw;
    // LDS: the sums of two steps, then x
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int sums = kw * nw * kSumWave;
    const int m = (int)a.m, rows = XF == X_TRI ? 3 * m : m;  // MFMA rows that count
    const int all = ((int)a.units + 1) / 2;
    const int ks = a.ks, kp = (int)blockIdx.x % ks, step = (int)gridDim.x / ks;
    const int pb = (int)((int64_t)all * kp / ks), pe = (int)((int64_t)all * (kp + 1) / ks);
    const int chunks = (pe - pb + kw * PP - 1) / (kw * PP);
    const int nblock = (int)((a.ntile + nw - 1) / nw);
    const int c = lane & 15, p4 = lane >> 4;
    const int64_t tile_bytes = (int64_t)all * kMxPair;
    XStage<XF> x(a, lds + 2 * sums);
    u32x4 wq[PP][2];
    uint32_t ws[PP];
    // a pair that does not exist is read at the last that does (and not used), a tile that does not exist as a buffer of
    // no bytes
    auto tile_buffer = [&](int b) {
        const int64_t tile = (int64_t)b * nw + wj;
        return rsrc(a.w + min(tile, a.ntile - 1) * tile_bytes, tile < a.ntile ? tile_bytes : 0);
    };
    auto load_w = [&](__amdgpu_buffer_rsrc_t t, int chunk, int j) {
        const int at = min(pb + (chunk * PP + j) * kw + wi, pe - 1) * kMxPair;
#pragma unroll
        for (int h = 0; h < 2; h++) wq[j][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(t, 16 * lane, at + 1024 * h, 2));
        ws[j] = __builtin_amdgcn_raw_buffer_load_b32(t, 2048 + 4 * (16 * (p4 & 1) + c), at, 2);
    };
    auto stage_part = [&](int chunk) {
        const int p0 = pb + chunk * kw * PP;
        x.part(a, p0, min(kw * PP, pe - p0));
    };
    uint64_t key = 0;
    int b = (int)blockIdx.x / ks, par = 0;
    // x before the weights: loads return in order, and x comes from L2
    stage_part(0);
    x.load(a, tid);
    {
        const __amdgpu_buffer_rsrc_t t = tile_buffer(b);
#pragma unroll
        for (int j = 0; j < PP; j++) load_w(t, 0, j);
    }
    x.store(a, tid);
    x.rest(a, tid);
    __syncthreads();
    const int xrow = min(XF == X_PLANES ? 3 * c : c, (XF == X_PLANES ? 3 * m - 3 : rows - 1));  // (MFMA rows past the last: the last again, not stored)
    for (; b < nblock; b += step) {
        floatx4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int chunk = 0; chunk < chunks; chunk++) {
            // the next step: the next chunk, or the next block's first
            const bool last = chunk + 1 == chunks;
            const int nb = last ? b + step : b, nc = last ? 0 : chunk + 1;
            const __amdgpu_buffer_rsrc_t t = tile_buffer(nb);
#pragma unroll
            for (int j = 0; j < PP; j++) {
                const bool there = pb + (chunk * PP + j) * kw + wi < pe;
                const int local = j * kw + wi;  // pair of the chunk
                if constexpr (BOTH) {
                    if (there) {
                        const uint32_t xs = *reinterpret_cast<const uint32_t *>(x.words + xrow * x.row_pieces + 8 * local + 4 * (p4 & 1)) >> (8 * (p4 >> 1));
                        const uint32_t s = ws[j] >> (8 * (p4 >> 1));
                        const uint8_t *xa = x.lds + xrow * x.pitch + 128 * local + 16 * p4;
                        acc = mfma_mx16<0>(*reinterpret_cast<const u32x4 *>(xa), xs, wq[j][0], s, acc);
                        acc = mfma_mx16<2>(*reinterpret_cast<const u32x4 *>(xa + 64), xs, wq[j][1], s, acc);
                    }
                } else if (there) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            u32x4 xa[P];
#pragma unroll
                            for (int p = 0; p < P; p++)
                                xa[p] = *reinterpret_cast<const u32x4 *>(x.lds + (xrow + p) * x.pitch + 512 * local + 256 * h + 64 * p4 + 16 * q);
                            const u32x4 bq = mx_codes_bf16(wq[j][h][q], mx_scale((ws[j] >> (8 * (p4 >> 1) + 16 * h)) & 0xFFu));
                            // (the lo plane first: added to a finished hi sum its low bits would be cut off)
#pragma unroll
                            for (int p = P - 1; p >= 0; p--) acc = mfma16x16x32_bf16(xa[p], bq, acc);
                        }
                }
                load_w(t, nc, j);
            }
            if (chunks > 1 && nb < nblock) {
                __syncthreads();
                stage_part(nc);
                x.load(a, tid);
                x.store(a, tid);
                x.rest(a, tid);
                __syncthreads();
            }
        }
        // lane 16p + c: rows 4p .. 4p + 3 of output column c -> [tile][wave along K][row][column]
        float *sb = reinterpret_cast<float *>(lds + par * sums);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (4 * p4 + i < rows) sb[(wj * kw + wi) * (kSumWave / 4) + (4 * p4 + i) * kSumRow + c] = acc[i];
        __syncthreads();  // also: every wave is past its reads of the other buffer
        const int outs = nw * m * 16;
        auto put = [&](int i, float v) {
            const int col = i & 15, t = (i >> 4) % m, tile = (i >> 4) / m;
            const int64_t row = ((int64_t)b * nw + tile) * kTile + col;
            if (row >= a.n) return;
            if (ks > 1) {
                a.slabs[((int64_t)kp * m + t) * a.n + row] = v;
                return;
            }
            if (a.bias) v += a.bias[row];
            if (a.y_bf16) reinterpret_cast<__bf16 *>(a.y)[t * a.n + row] = (__bf16)v;
            else reinterpret_cast<float *>(a.y)[t * a.n + row] = v;
            if (a.argmax_partial) key = max(key, mx_argmax_key(v, (uint32_t)row));
        };
        // waves w0, w0 + dw, .. of output i (three planes: the lo ones first)
        auto sum = [&](int i, int w0, int dw) {
            const int col = i & 15, t = (i >> 4) % m, tile = (i >> 4) / m;
            const float *o = sb + tile * kw * (kSumWave / 4) + (XF == X_TRI ? 3 * t : t) * kSumRow + col;
            float v = 0.f;
#pragma unroll
            for (int p = XF == X_TRI ? 2 : 0; p >= 0; p--) {
                float u = 0.f;
                for (int w = w0; w < kw; w += dw) u += o[w * (kSumWave / 4) + p * kSumRow];
                v += u;
            }
            return v;
        };
        if (outs * 8 <= (int)blockDim.x) {  // few outputs: eight lanes each
            const int i = tid >> 3;
            float v = i < outs ? sum(i, tid & 7, 8) : 0.f;
            v += __uint_as_float(row_lane<0xB1>(__float_as_uint(v)));
            v += __uint_as_float(row_lane<0x4E>(__float_as_uint(v)));
            v += __uint_as_float(row_lane<0x141>(__float_as_uint(v)));
            if (i < outs && (tid & 7) == 0) put(i, v);
        } else {
            for (int i = tid; i < outs; i += (int)blockDim.x) put(i, sum(i, 0, 1));
        }
        par ^= 1;
    }
    if (a.argmax_partial) {
        // m = 1: threads that stored outputs hold keys (0 elsewhere); one key per workgroup
        __syncthreads();
        unsigned long long *kr = reinterpret_cast<unsigned long long *>(lds);
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)key, o, 64);
            key = other > key ? other : key;
        }
        if (lane == 0) kr[wv] = key;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kw * nw; w++) key = max(key, (uint64_t)kr[w]);
            a.argmax_partial[blockIdx.x] = key;
        }
    }
}

template <int XF, int PP>
int launch_rows_t(const MxArgs &a, const MxRowsPlan &p, void *stream) {
    const int64_t blocks = (a.ntile + p.nw - 1) / p.nw;
    const int64_t grid = std::min<int64_t>(blocks, std::max(1, p.groups)) * p.ks;
    if (a.argmax_count) *a.argmax_count = grid;
    auto *kernel = mx_rows_kernel<XF, PP>;
    hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), (size_t)p.lds);
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3((unsigned)(p.kw * p.nw * 64)), (size_t)p.lds, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

template <int XF>
int launch_rows_x(const MxArgs &a, const MxRowsPlan &p, void *stream) {
    if (p.pp == 1) return launch_rows_t<XF, 1>(a, p, stream);
    if (p.pp == 2) return launch_rows_t<XF, 2>(a, p, stream);
    if constexpr (XF != X_PLANES) {  // (the planes of six rows leave LDS for 17 pairs: two a wave)
        if (p.pp == 3) return launch_rows_t<XF, 3>(a, p, stream);
        if (p.pp == 4) return launch_rows_t<XF, 4>(a, p, stream);
    }
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
    const int64_t pieces = count / (out_bf16 ? 8 : 4), grid = (pieces + 1023) / 1024;
    if (grid > INT32_MAX) return (int)hipErrorInvalidValue;
    uint8_t *o = reinterpret_cast<uint8_t *>(out);
    if (out_bf16) hipLaunchKernelGGL(mx_dequantize_kernel<true>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, codes, scales, pieces, o);
    else hipLaunchKernelGGL(mx_dequantize_kernel<false>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, codes, scales, pieces, o);
    return (int)hipGetLastError();
}

int launch_mx_quantize_image(const void *x, int x_bf16, int64_t m, int64_t k, int floor_rule, uint8_t *image, void *stream) {
    const int64_t units = 2 * mx_pairs(k), jobs = mx_tiles(m) * units;
    if (jobs > INT32_MAX) return (int)hipErrorInvalidValue;
    const uint8_t *p = reinterpret_cast<const uint8_t *>(x);
    if (x_bf16)
        hipLaunchKernelGGL(mx_quantize_image_kernel<true>, dim3((unsigned)jobs), dim3(64), 0, (hipStream_t)stream, p, m, k, units, floor_rule, image);
    else
        hipLaunchKernelGGL(mx_quantize_image_kernel<false>, dim3((unsigned)jobs), dim3(64), 0, (hipStream_t)stream, p, m, k, units, floor_rule, image);
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
    a.kw = p.kw;
    a.nw = p.nw;
    uint8_t *base = reinterpret_cast<uint8_t *>(scratch);
    a.slabs = reinterpret_cast<float *>(base + p.slabs);
    int e = 0;
    if (p.first) {  // quantized once, not by every workgroup
        uint8_t *scales = base + (size_t)a.m * a.k / 2;
        e = launch_mx_quantize(a.x, a.x_kind == kMxQuantBf16, a.m, a.k, a.k, a.floor_rule, base, scales, stream);
        if (e) return e;
        a.x = base;
        a.xs = scales;
        a.x_kind = kMxCodes;
    }
    e = a.x_kind == kMxBf16          ? launch_rows_x<X_BF16>(a, p, stream)
                  : a.x_kind == kMxF32         ? (a.m <= kMxTriRows ? launch_rows_x<X_TRI>(a, p, stream) : launch_rows_x<X_PLANES>(a, p, stream))
                  : a.x_kind == kMxQuantBf16   ? launch_rows_x<X_Q16>(a, p, stream)
                  : a.x_kind == kMxQuantF32    ? launch_rows_x<X_Q32>(a, p, stream) : launch_rows_x<X_CODES>(a, p, stream);
    if (e || a.ks == 1) return e;
    return launch_int4_sum(a.slabs, a.ks, a.m, a.n, a.bias, a.y, a.y_bf16, stream);
}

}  // namespace nnq
