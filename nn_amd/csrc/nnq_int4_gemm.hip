// Linear over 4-bit codes with group scales on gfx950 for more than sixteen token rows
// (nnq_int4.hip has the formula, the image and the exact f16 form of the codes).
//
// Bound: the 32x32x16 f16 MFMAs (f32 x: two per product, for the hi and lo parts), with the VALU
// that turns codes into operands and scales a group's sums close behind.  The scale cannot go into
// an operand: scale * (q - z) has up to 16 significant bits.
//  * int4_stage_kernel writes x once as f16 of x * 2^s_row (f32 x: a hi and a lo plane) in the order
//    of the MFMA's A operands, per 32 rows and unit of 128 k one 8 KB piece, and 2^-s_row per row.
//  * int4_gemm_kernel: a workgroup of W waves takes MT * 32 rows and W * 32 columns.  The A pieces of
//    a unit go through two LDS buffers, one barrier per unit; a wave's weights go from memory straight
//    into its registers and become the B operands of its own 32 columns, each used for MT MFMAs, so
//    no operand is dequantized twice in a workgroup and none passes through LDS.
//  * A group's MFMAs start from zero (results in VGPRs, the build's VGPR-form option for this file)
//    and are added to the totals times the scale of the lane's column: 16 FMAs per 32 x 32 tile and
//    group, beside 8 (group 128), 4 or 2 MFMAs of 32 cycles.
//  * With too few workgroups K is split: f32 slabs, added in order by int4_sum_kernel.
#include <algorithm>

#include "nnq_device.h"
#include "nnq_int4.h"
#include "nnq_internal.h"

namespace nnq {

namespace {

constexpr int kPiece = 8192;  // bytes of the A operands of 32 rows and one unit: 8 steps x 64 lanes x 16

__device__ __forceinline__ floatx16 mfma32(u32x4 a, u32x4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// Four rows a workgroup (thread % 4): the row's largest |x|, then its 8-column chunks, chunk c of the
// row at piece c / 16, step (c / 2) % 8, half c % 2.  Chunks past K are zeros.
template <bool XB>
__global__ __launch_bounds__(512) void int4_stage_kernel(const void *x, int m, int64_t k, int units, uint8_t *xa,
                                                         int64_t plane, float *rowback) {
    __shared__ uint32_t red[8][4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int row = (int)blockIdx.x * 4 + (tid & 3), t = min(row, m - 1);
    const int chunks = (int)(k / 8);
    auto load = [&](int c, float(&v)[8]) {
        if constexpr (XB) {
            const u32x4 r = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint16_t *>(x) + t * k + 8 * c);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[2 * e] = __uint_as_float(r[e] << 16);
                v[2 * e + 1] = __uint_as_float(r[e] & 0xFFFF0000u);
            }
        } else {
            const floatx4 *p = reinterpret_cast<const floatx4 *>(reinterpret_cast<const float *>(x) + t * k + 8 * c);
            const floatx4 r0 = p[0], r1 = p[1];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] = r0[e];
                v[4 + e] = r1[e];
            }
        }
    };
    uint32_t mx = 0;
    for (int c = tid >> 2; c < chunks; c += 128) {
        float v[8];
        load(c, v);
#pragma unroll
        for (int e = 0; e < 8; e++) mx = max(mx, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    }
    for (int o = 4; o < 64; o <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
    if (lane < 4) red[tid >> 6][lane] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) mx = max(mx, red[w][tid & 3]);
    float s, back;
    f16_prescale(__uint_as_float(mx), s, back);
    if (row >= m) return;
    if (tid < 4) rowback[row] = back;
    uint8_t *dst = xa + (int64_t)(row >> 5) * units * kPiece + (row & 31) * 16;
    for (int c = tid >> 2; c < units * 16; c += 128) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (c < chunks) load(c, v);
        u32x4 hi, lo;
        split8<!XB>(v, s, hi, lo);
        u32x4 *o = reinterpret_cast<u32x4 *>(dst + (int64_t)(c >> 1) * 1024 + (c & 1) * 512);
        *o = hi;
        if constexpr (!XB) *reinterpret_cast<u32x4 *>(reinterpret_cast<uint8_t *>(o) + plane) = lo;
    }
}

struct Int4GemmArgs {
    const uint8_t *w, *xa;
    const float *rowback, *bias;
    void *y;        // [m][n], or with ks > 1 f32 slabs [ks][m][n] without the bias
    int y_bf16, scale_bf16;
    int m, units, ntile, ks;
    int row_blocks, col_blocks;
    int64_t n, plane;
};

// The raw bytes of one unit of 32 columns (two tiles): lane 32h + 16b + r holds row r of tile b, its
// k groups h and 2 + h, i.e. the B operands of steps 2j + i at word j of q[i].
template <int GS, bool Z>
struct Unit32 {
    u32x4 q[2];
    uint32_t s[(GS + 1) / 2];
    uint32_t z;
};

template <int MT, int P, int GS, bool Z, int W>
__global__ __launch_bounds__(W * 64, 2) void int4_gemm_kernel(Int4GemmArgs a) {
    constexpr int UB = int4_unit_bytes(kInt4Unit / GS, Z);
    constexpr int BUF = MT * P * kPiece;
    constexpr int NA = BUF / (W * 64 * 16);  // 16-byte pieces of A per thread and unit
    static_assert(NA * W * 64 * 16 == BUF, "whole pieces");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    // workgroup ids go round the 8 XCDs: each takes a contiguous run, the row blocks of a column block
    // (which share its weights) one after another
    const int total = a.row_blocks * a.col_blocks * a.ks, bid = (int)blockIdx.x;
    const int per = total / 8, extra = total % 8, xcd = bid % 8, at = bid / 8;
    const int T = xcd * per + min(xcd, extra) + at;
    const int rb = T % a.row_blocks, cb = T / a.row_blocks % a.col_blocks, kp = T / (a.row_blocks * a.col_blocks);
    const int u0 = (int)((int64_t)a.units * kp / a.ks), u1 = (int)((int64_t)a.units * (kp + 1) / a.ks);

    const int c32 = lane & 31, h = lane >> 5, r = lane & 15;
    const int tile0 = (cb * W + wv) * 2;
    const int tile = min(tile0 + ((lane >> 4) & 1), a.ntile - 1);  // (past the last: not stored)
    const uint8_t *wp = a.w + (size_t)tile * a.units * UB;
    auto load_w = [&](int u, Unit32<GS, Z> &o) {
        const uint8_t *rec = wp + (size_t)u * UB;
        o.q[0] = *reinterpret_cast<const u32x4 *>(rec + 16 * (16 * h + r));
        o.q[1] = *reinterpret_cast<const u32x4 *>(rec + 16 * (16 * (2 + h) + r));
        load_scales<GS, Z>(rec, r, o.s, o.z);
    };
    // A pieces: (row block, plane) pairs of a unit, 8 KB each; rows past the last block: the last one
    const int row_pieces = (a.m + 31) / 32;
    u32x4 ar[NA];
    auto load_a = [&](int u) {
#pragma unroll
        for (int i = 0; i < NA; i++) {
            const int p = (i * W * 64 + tid) / 512, off = (i * W * 64 + tid) % 512;
            const int pc = min(rb * MT + p % MT, row_pieces - 1);
            ar[i] = *reinterpret_cast<const u32x4 *>(a.xa + (p / MT) * a.plane + ((int64_t)pc * a.units + u) * kPiece + off * 16);
        }
    };
    auto store_a = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NA; i++) *reinterpret_cast<u32x4 *>(lds + buf * BUF + (i * W * 64 + tid) * 16) = ar[i];
    };

    floatx16 tot[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int e = 0; e < 16; e++) tot[mt][e] = 0.f;
    Unit32<GS, Z> w, wn;
    load_a(u0);
    load_w(u0, w);
    store_a(0);
    __syncthreads();
    for (int u = u0; u < u1; u++) {
        const int buf = (u - u0) & 1;
        const bool more = u + 1 < u1;
        if (more) {
            load_a(u + 1);
            load_w(u + 1, wn);
        }
        const uint8_t *ab = lds + buf * BUF + lane * 16;
#pragma unroll
        for (int g = 0; g < GS; g++) {
            uint32_t c1, c2;
            zero_consts<Z>(w.z, g, c1, c2);
            floatx16 part[MT];
#pragma unroll
            for (int jj = 0; jj < 4 / GS; jj++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int j = g * (4 / GS) + jj, step = 2 * j + i;
                    const u32x4 b = codes_f16(w.q[i][j], c1, c2);
                    // (the lo plane first: added to a finished hi sum its low bits would be cut off)
#pragma unroll
                    for (int pl = P - 1; pl >= 0; pl--)
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            const u32x4 av = *reinterpret_cast<const u32x4 *>(ab + (pl * MT + mt) * kPiece + step * 1024);
                            floatx16 zero;
#pragma unroll
                            for (int e = 0; e < 16; e++) zero[e] = 0.f;
                            part[mt] = mfma32(av, b, jj == 0 && i == 0 && pl == P - 1 ? zero : part[mt]);
                        }
                }
            const float s = group_scale(w.s, g, a.scale_bf16);
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int e = 0; e < 16; e++) tot[mt][e] = fmaf(s, part[mt][e], tot[mt][e]);
            if (GS > 1) __builtin_amdgcn_sched_barrier(0);  // one group's sums at a time: two would spill
        }
        if (more) {
            store_a(buf ^ 1);  // (read by nobody since the barrier before this unit)
            w = wn;
        }
        __syncthreads();
    }

    // lane: column c32, rows 8 (e / 4) + 4h + e % 4 of each 32-row tile
    const int64_t col = (int64_t)tile0 * kTile + c32;
    if (col >= a.n) return;
    const bool slab = a.ks > 1;
    const float bias = a.bias && !slab ? a.bias[col] : 0.f;
    float *ys = reinterpret_cast<float *>(a.y) + (slab ? (int64_t)kp * a.m * a.n : 0);
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int row = (rb * MT + mt) * 32 + 8 * (e / 4) + 4 * h + e % 4;
            if (row < a.m) {
                const float v = fmaf(tot[mt][e], a.rowback[row], bias);
                if (!slab && a.y_bf16)
                    reinterpret_cast<uint16_t *>(a.y)[(int64_t)row * a.n + col] = (uint16_t)f32_to_bf16_bits(v);
                else
                    ys[(int64_t)row * a.n + col] = v;
            }
        }
}

// y[i] = sum of the ks slabs' [i] in order + bias[i % n]
__global__ __launch_bounds__(256) void int4_sum_kernel(const float *ys, int ks, int64_t count, int64_t n,
                                                       const float *bias, void *y, int y_bf16) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        float v = ys[i];
        for (int s = 1; s < ks; s++) v += ys[s * count + i];
        if (bias) v += bias[i % n];
        if (y_bf16)
            reinterpret_cast<uint16_t *>(y)[i] = (uint16_t)f32_to_bf16_bits(v);
        else
            reinterpret_cast<float *>(y)[i] = v;
    }
}

template <int MT, int P, int GS, bool Z, int W>
int launch_gemm_t(const Int4GemmArgs &a, void *stream) {
    constexpr size_t lds = 2 * MT * P * kPiece;
    auto *kernel = int4_gemm_kernel<MT, P, GS, Z, W>;
    hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), lds);
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.row_blocks * a.col_blocks * a.ks)), dim3(W * 64), lds,
                       (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

template <int P, int GS, bool Z, int W>
int launch_gemm_m(int mt, const Int4GemmArgs &a, void *stream) {
    switch (mt) {
    case 1: return launch_gemm_t<1, P, GS, Z, W>(a, stream);
    case 2: return launch_gemm_t<2, P, GS, Z, W>(a, stream);
    case 3: return launch_gemm_t<3, P, GS, Z, W>(a, stream);
    default: return launch_gemm_t<4, P, GS, Z, W>(a, stream);
    }
}

template <int P, int GS, bool Z>
int launch_gemm_w(int waves, int mt, const Int4GemmArgs &a, void *stream) {
    return waves == 8 ? launch_gemm_m<P, GS, Z, 8>(mt, a, stream) : launch_gemm_m<P, GS, Z, 4>(mt, a, stream);
}

template <int P>
int launch_gemm_g(int group, int zeros, int waves, int mt, const Int4GemmArgs &a, void *stream) {
    if (zeros) {
        if (group == 128) return launch_gemm_w<P, 1, true>(waves, mt, a, stream);
        if (group == 64) return launch_gemm_w<P, 2, true>(waves, mt, a, stream);
        return launch_gemm_w<P, 4, true>(waves, mt, a, stream);
    }
    if (group == 128) return launch_gemm_w<P, 1, false>(waves, mt, a, stream);
    if (group == 64) return launch_gemm_w<P, 2, false>(waves, mt, a, stream);
    return launch_gemm_w<P, 4, false>(waves, mt, a, stream);
}

}  // namespace

int launch_int4_gemm(const Int4Args &a, void *scratch, void *stream) {
    const Int4GemmPlan p = int4_gemm_plan(a.m, a.n, a.k, a.x_bf16);
    if (a.m < 1 || a.m > INT32_MAX / 2 || a.units < 1) return (int)hipErrorInvalidValue;
    uint8_t *base = reinterpret_cast<uint8_t *>(scratch);
    Int4GemmArgs g{};
    g.w = a.w;
    g.xa = base;
    g.plane = (int64_t)p.plane;
    float *rowback = reinterpret_cast<float *>(base + p.rowback);
    float *slabs = reinterpret_cast<float *>(base + p.slabs);
    g.rowback = rowback;
    g.bias = a.bias;
    g.y = p.ks > 1 ? (void *)slabs : a.y;
    g.y_bf16 = a.y_bf16;
    g.scale_bf16 = a.scale_bf16;
    g.m = (int)a.m;
    g.units = (int)a.units;
    g.ntile = (int)a.ntile;
    g.ks = p.ks;
    g.row_blocks = p.row_blocks;
    g.col_blocks = p.col_blocks;
    g.n = a.n;
    const dim3 sg((unsigned)((a.m + 3) / 4));
    if (a.x_bf16)
        hipLaunchKernelGGL((int4_stage_kernel<true>), sg, dim3(512), 0, (hipStream_t)stream, a.x, (int)a.m, a.k,
                           (int)a.units, base, g.plane, rowback);
    else
        hipLaunchKernelGGL((int4_stage_kernel<false>), sg, dim3(512), 0, (hipStream_t)stream, a.x, (int)a.m, a.k,
                           (int)a.units, base, g.plane, rowback);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    int rc = a.x_bf16 ? launch_gemm_g<1>(a.group, a.zeros, p.waves, p.mt, g, stream)
                      : launch_gemm_g<2>(a.group, a.zeros, p.waves, p.mt, g, stream);
    if (rc || p.ks == 1) return rc;
    const int64_t count = a.m * a.n;
    hipLaunchKernelGGL(int4_sum_kernel, dim3((unsigned)std::min<int64_t>((count + 255) / 256, 8192)), dim3(256), 0,
                       (hipStream_t)stream, slabs, p.ks, count, a.n, a.bias, a.y, a.y_bf16);
    return (int)hipGetLastError();
}

}  // namespace nnq
