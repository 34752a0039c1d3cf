// Linear over 4-bit codes with group scales on gfx950 for more than sixteen token rows
// (nnq_int4.hip has the formula, the image and the exact f16 form of the codes).
//
// Bound: the 32x32x16 f16 MFMAs (f32 x: two per product, for the hi and lo parts), with the VALU
// that turns codes into operands and scales a group's sums close behind.  The scale cannot go into
// an operand: scale * (q - z) has up to 16 significant bits.
//  * int4_stage_kernel writes x once as f16 of x * 2^s_row (f32 x: a hi and a lo plane) in the order
//    of the MFMA's A operands, per 32 rows and unit of 128 k one 8 KB piece, and 2^-s_row per row.
//  * int4_gemm_kernel: a workgroup of four waves takes MT * 32 rows and NT * 128 columns.  The A
//    pieces of a unit are copied straight to one of two LDS buffers, a unit ahead, with one barrier
//    per unit; a wave's weights go from memory into its registers, a unit ahead too, and become the B
//    operands of its own NT * 32 columns, each used for MT MFMAs, so no operand is dequantized twice
//    in a workgroup and none passes through LDS.  (An A operand read from LDS feeds NT MFMAs: with NT
//    = 1 the reads take as long as the MFMAs.)
//  * A group's MFMAs start from zero (results in VGPRs, the build's VGPR-form option for this file)
//    and are added to the totals times the scale of the lane's column: 16 FMAs per 32 x 32 tile and
//    group, beside 8 (group 128), 4 or 2 MFMAs of 32 cycles.
//  * With too few workgroups K is split: f32 slabs, added in order by int4_sum_kernel.
// Measured (MI355X, bf16 x, groups of 128): 512 x 4096 -> 12288 54 us + 6 of staging, 0.95 PFLOP/s;
// 300 x 4096 -> 151936 360 to 410 us, 1.04 to 0.91 PFLOP/s, the clock lower the longer it runs (the
// library's f16 product of 8192^3: 1.06 to 1.3).  The MFMAs alone, with nothing beside them, take
// 78 us of 512 x 4096 -> 24576 (1.3 PFLOP/s), all of the kernel 108.
#include <algorithm>
#include <type_traits>

#include "nnq_device.h"
#include "nnq_int4.h"
#include "nnq_internal.h"

namespace nnq {

namespace {

constexpr int W = 4;          // waves of a GEMM workgroup
constexpr int kPiece = 8192;  // bytes of the A operands of 32 rows and one unit: 8 steps x 64 lanes x 16

__device__ __forceinline__ floatx16 mfma32(u32x4 a, u32x4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// ROWS rows a workgroup (thread % ROWS): the row's largest |x|, then its 8-column chunks, chunk c of the
// row at piece c / 16, step (c / 2) % 8, half c % 2.  Chunks past K are zeros.  A thread's first kHold
// chunks stay in registers between the two (all of them up to K = 8192, two rows: 16384).  Four adjacent
// rows write 64 bytes together; two fill the chip from half as many rows, and the two halves of four go to
// one XCD, whose L2 joins them (us, two / four: 203 f32 rows of 12288 8.8 / 14.0, 512 bf16 rows of 4096
// 5.4 / 5.5, 2048 10.2 / 9.4).
template <int ROWS>
__device__ __forceinline__ int stage_row(int b) {
    return ROWS == 4 ? b * 4 : (b / 16 * 8 + b % 8) * 4 + b / 8 % 2 * 2;
}
constexpr int kStageThreads = 1024, kHold = 4;
template <bool XB, int ROWS>
__global__ __launch_bounds__(kStageThreads) void int4_stage_kernel(const void *x, int m, int64_t k, int units,
                                                                   uint8_t *xa, int64_t plane, float *rowback) {
    constexpr int WV = kStageThreads / 64, STEP = kStageThreads / ROWS;
    __shared__ uint32_t red[WV][ROWS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int row = stage_row<ROWS>((int)blockIdx.x) + tid % ROWS, t = min(row, m - 1);
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
    auto largest = [&](const float(&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) mx = max(mx, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    };
    float held[kHold][8];
#pragma unroll
    for (int i = 0; i < kHold; i++) {
        const int c = tid / ROWS + i * STEP;
#pragma unroll
        for (int e = 0; e < 8; e++) held[i][e] = 0.f;
        if (c < chunks) load(c, held[i]);
    }
#pragma unroll
    for (int i = 0; i < kHold; i++) largest(held[i]);
    for (int c = tid / ROWS + kHold * STEP; c < chunks; c += STEP) {
        float v[8];
        load(c, v);
        largest(v);
    }
    for (int o = ROWS; o < 64; o <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
    if (lane < ROWS) red[tid >> 6][lane] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WV; w++) mx = max(mx, red[w][tid % ROWS]);
    float s, back;
    f16_prescale(__uint_as_float(mx), s, back);
    if (row >= m) return;
    if (tid < ROWS) rowback[row] = back;
    uint8_t *dst = xa + (int64_t)(row >> 5) * units * kPiece + (row & 31) * 16;
    auto put = [&](int c, const float(&v)[8]) {
        u32x4 hi, lo;
        split8<!XB>(v, s, hi, lo);
        u32x4 *o = reinterpret_cast<u32x4 *>(dst + (int64_t)(c >> 1) * 1024 + (c & 1) * 512);
        *o = hi;
        if constexpr (!XB) *reinterpret_cast<u32x4 *>(reinterpret_cast<uint8_t *>(o) + plane) = lo;
    };
#pragma unroll
    for (int i = 0; i < kHold; i++) {
        const int c = tid / ROWS + i * STEP;
        if (c < units * 16) put(c, held[i]);
    }
    for (int c = tid / ROWS + kHold * STEP; c < units * 16; c += STEP) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (c < chunks) load(c, v);
        put(c, v);
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

template <int MT, int NT, int P, int GS, bool Z>
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
    const int tile0 = (cb * W + wv) * 2 * NT;
    // (buffers: one register of a lane's offset for all loads of a kind instead of a pair for each)
    __amdgpu_buffer_rsrc_t wb[NT];
    int pair[NT];  // from the first tile of a pair to the second; tiles past the last: not stored
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int t = min(tile0 + 2 * nt, a.ntile - 1);
        wb[nt] = rsrc(a.w + (size_t)t * a.units * UB, (int64_t)min(2, a.ntile - t) * a.units * UB);
        pair[nt] = (lane & 16) && t + 1 < a.ntile ? a.units * UB : 0;
    }
    auto load_w = [&](int u, Unit32<GS, Z>(&o)[NT]) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int lq = pair[nt] + 16 * (16 * h + r), ls = pair[nt] + 1024 + 2 * GS * r;
            const int lz = pair[nt] + 1024 + 32 * GS + GS * r;
            o[nt].q[0] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wb[nt], lq, u * UB, 0));
            o[nt].q[1] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wb[nt], lq + 512, u * UB, 0));
            load_scales<GS, Z, 0, true>(wb[nt], ls, lz, u * UB, o[nt].s, o[nt].z);
        }
    };
    // A pieces: (row block, plane) pairs of a unit, 8 KB each; rows past the last block: the last one
    const int row_pieces = (a.m + 31) / 32;
    const __amdgpu_buffer_rsrc_t xb = rsrc(a.xa, P * a.plane);
    auto copy_a = [&](int u, int buf) {
#pragma unroll
        for (int i = 0; i < NA; i++) {
            const int p = i / 2, pc = min(rb * MT + p % MT, row_pieces - 1);
            const int at = (p / MT) * (int)a.plane + (pc * a.units + u) * kPiece + i % 2 * 4096;
            copy16_lds(xb, lds + buf * BUF + (i * W + wv) * 1024, tid * 16, at);
        }
    };
    static_assert(W * 64 * 16 * 2 == kPiece, "two loads of the workgroup a piece");
    // The MFMAs of a step are issued one at a time with the forming of the next step's operands and the
    // scaling of a finished group's sums between them: a wave that issues MFMAs back to back waits for
    // the matrix pipe with its own VALU work behind them.  (32 cycles of an MFMA hide six VALU
    // instructions.)
    const CodeMasks km;
    const uint32_t sm = scale_mask(a.scale_bf16), zsel = kZeroSel + 0x00010001u * (uint32_t)(GS * r & 3);
    floatx16 tot[MT][NT], part[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 16; e++) tot[mt][nt][e] = part[mt][nt][e] = 0.f;
    float sc[NT];  // the scales of the sums in `part`
    uint32_t c1[NT], c2[NT];
    u32x4 af[2][P][MT], bf[2][NT];
    Unit32<GS, Z> w2[2][NT];  // this unit's weights and the next one's, in turn (copied, they would be waited for at once)
#pragma unroll
    for (int nt = 0; nt < NT; nt++) sc[nt] = 0.f;
    auto read_a = [&](int buf, int s, int q) {
        af[s & 1][q / MT][q % MT] = *reinterpret_cast<const u32x4 *>(lds + buf * BUF + lane * 16 + q * kPiece + s * 1024);
    };
    auto arrive = [&]() {
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto scale_part = [&](int mt, int nt) {
#pragma unroll
        for (int e = 0; e < 16; e++) tot[mt][nt][e] = fmaf(sc[nt], part[mt][nt][e], tot[mt][nt][e]);
        asm volatile("" : "+v"(tot[mt][nt]));  // here: moved on, the sums would keep `part` alive beside its next values
        __builtin_amdgcn_sched_barrier(0);
    };
    // A unit's last step already reads and forms the next unit's first, so that no MFMA waits at a unit's
    // edge.  The barrier before it is the unit's only one: this unit's A pieces have been read (the loads of
    // step 7's operands are waited for there) and the copies of the next one, issued a unit earlier, have
    // landed, as have the weights; copies and loads of the unit after that start behind it.  Past the last
    // unit the last one is loaded again.
    auto begin = [&](auto parity) {
        constexpr int buf = decltype(parity)::value;
        copy_a(u0, buf);
        load_w(u0, w2[buf]);
        copy_a(min(u0 + 1, u1 - 1), buf ^ 1);
        load_w(min(u0 + 1, u1 - 1), w2[buf ^ 1]);
        arrive();
#pragma unroll
        for (int q = 0; q < P * MT; q++) read_a(buf, 0, q);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            zero_consts<Z>(w2[buf][nt].z, 0, c1[nt], c2[nt], zsel);
            bf[0][nt] = codes_f16(w2[buf][nt].q[0][0], c1[nt], c2[nt], km);
        }
    };
    auto unit = [&](auto parity, int ahead) {
        constexpr int buf = decltype(parity)::value;
#pragma unroll
        for (int s = 0; s < 8; s++) {
            const Unit32<GS, Z>(&w)[NT] = w2[s == 7 ? buf ^ 1 : buf];  // of the operands to form
            const bool first = s % (8 / GS) == 0;
            const int sn = (s + 1) % 8;
            if (s == 7) {
                arrive();
                copy_a(ahead, buf);
                load_w(ahead, w2[buf]);
            }
            if (sn % (8 / GS) == 0)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) zero_consts<Z>(w[nt].z, sn / (8 / GS), c1[nt], c2[nt], zsel);
            constexpr int M = P * MT * NT;  // MFMAs of a step
#pragma unroll
            for (int q = 0; q < M; q++) {
                // (the lo plane first: added to a finished hi sum its low bits would be cut off)
                const int pl = P - 1 - q / (MT * NT), mt = q / NT % MT, nt = q % NT;
                const bool start = first && q < MT * NT;
                __builtin_amdgcn_sched_barrier(0);
                if (start) scale_part(mt, nt);
                floatx16 zero;
#pragma unroll
                for (int e = 0; e < 16; e++) zero[e] = 0.f;
                part[mt][nt] = mfma32(af[s & 1][pl][mt], bf[s & 1][nt], start ? zero : part[mt][nt]);
                if (q % NT == 0) read_a(s == 7 ? buf ^ 1 : buf, sn, q / NT);
#pragma unroll
                for (int j = 0; j < 4 * NT; j++)
                    if (j * M / (4 * NT) == q)
                        bf[sn & 1][j / 4][j % 4] = code_pair(w[j / 4].q[sn & 1][sn >> 1], j % 4, c1[j / 4], c2[j / 4], km);
            }
            if (first)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) sc[nt] = group_scale(w2[buf][nt].s, s / (8 / GS), sm);
        }
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> odd;
    int u = u0;
    if ((u1 - u0) & 1) {
        begin(odd);
        unit(odd, min(u0 + 2, u1 - 1));
        u++;
    } else {
        begin(even);
    }
    for (; u < u1; u += 2) {
        unit(even, min(u + 2, u1 - 1));
        unit(odd, min(u + 3, u1 - 1));
    }

    // lane: column c32 of each 32, rows 8 i + 4h + e of each 32-row tile.  Everything that is read comes
    // before the first store: a wait for a load waits for the stores before it, too.
    const bool slab = a.ks > 1;
    float bias[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int64_t col = (int64_t)(tile0 + 2 * nt) * kTile + c32;
        bias[nt] = a.bias && !slab && col < a.n ? a.bias[col] : 0.f;
    }
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        floatx4 back[4];  // (whole 32-row tiles are there)
#pragma unroll
        for (int i = 0; i < 4; i++)
            back[i] = *reinterpret_cast<const floatx4 *>(a.rowback + min(rb * MT + mt, row_pieces - 1) * 32 + 4 * h + 8 * i);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            scale_part(mt, nt);
#pragma unroll
            for (int e = 0; e < 16; e++) tot[mt][nt][e] = fmaf(tot[mt][nt][e], back[e / 4][e % 4], bias[nt]);
        }
    }
    auto store = [&](auto *y, auto &&as) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const int row0 = (rb * MT + mt) * 32 + 4 * h;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const int64_t col = (int64_t)(tile0 + 2 * nt) * kTile + c32;
                if (col >= a.n) continue;
                auto *p = y + (int64_t)row0 * a.n + col;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    if (row0 + 8 * (e / 4) + e % 4 < a.m) *p = as(tot[mt][nt][e]);
                    p += e % 4 == 3 ? 5 * a.n : a.n;
                }
            }
        }
    };
    if (!slab && a.y_bf16)
        store(reinterpret_cast<uint16_t *>(a.y), [](float v) { return (uint16_t)f32_to_bf16_bits(v); });
    else
        store(reinterpret_cast<float *>(a.y) + (slab ? (int64_t)kp * a.m * a.n : 0), [](float v) { return v; });
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

template <int MT, int NT, int P, int GS, bool Z>
int launch_gemm_t(const Int4GemmArgs &a, void *stream) {
    constexpr size_t lds = 2 * MT * P * kPiece;
    static_assert(lds <= 65536, "LDS of a launch without an attribute");
    hipLaunchKernelGGL((int4_gemm_kernel<MT, NT, P, GS, Z>), dim3((unsigned)(a.row_blocks * a.col_blocks * a.ks)),
                       dim3(W * 64), lds, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

template <int P, int GS, bool Z>
int launch_gemm_s(int mt, int nt, const Int4GemmArgs &a, void *stream) {
    if (mt == 1) return nt == 1 ? launch_gemm_t<1, 1, P, GS, Z>(a, stream) : launch_gemm_t<1, 2, P, GS, Z>(a, stream);
    if constexpr (P == 1 && GS != 4)
        return nt == 1 ? launch_gemm_t<2, 1, P, GS, Z>(a, stream) : launch_gemm_t<2, 2, P, GS, Z>(a, stream);
    else
        return launch_gemm_t<2, 1, P, GS, Z>(a, stream);
}

template <int P>
int launch_gemm_g(int group, int zeros, int mt, int nt, const Int4GemmArgs &a, void *stream) {
    if (zeros) {
        if (group == 128) return launch_gemm_s<P, 1, true>(mt, nt, a, stream);
        if (group == 64) return launch_gemm_s<P, 2, true>(mt, nt, a, stream);
        return launch_gemm_s<P, 4, true>(mt, nt, a, stream);
    }
    if (group == 128) return launch_gemm_s<P, 1, false>(mt, nt, a, stream);
    if (group == 64) return launch_gemm_s<P, 2, false>(mt, nt, a, stream);
    return launch_gemm_s<P, 4, false>(mt, nt, a, stream);
}

template <int ROWS>
void launch_stage(const Int4Args &a, uint8_t *xa, int64_t plane, float *rowback, void *stream) {
    const dim3 grid((unsigned)(ROWS == 4 ? (a.m + 3) / 4 : (a.m + 31) / 32 * 16)), block(kStageThreads);
    if (a.x_bf16)
        hipLaunchKernelGGL((int4_stage_kernel<true, ROWS>), grid, block, 0, (hipStream_t)stream, a.x, (int)a.m, a.k,
                           (int)a.units, xa, plane, rowback);
    else
        hipLaunchKernelGGL((int4_stage_kernel<false, ROWS>), grid, block, 0, (hipStream_t)stream, a.x, (int)a.m, a.k,
                           (int)a.units, xa, plane, rowback);
}

}  // namespace

int launch_int4_gemm(const Int4Args &a, void *scratch, void *stream) {
    const Int4GemmPlan p = int4_gemm_plan(a.m, a.n, a.k, a.group, a.x_bf16);
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
    if (a.m > 512) launch_stage<4>(a, base, g.plane, rowback, stream);
    else launch_stage<2>(a, base, g.plane, rowback, stream);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    int rc = a.x_bf16 ? launch_gemm_g<1>(a.group, a.zeros, p.mt, p.nt, g, stream)
                      : launch_gemm_g<2>(a.group, a.zeros, p.mt, p.nt, g, stream);
    if (rc || p.ks == 1) return rc;
    return launch_int4_sum(slabs, p.ks, a.m, a.n, a.bias, a.y, a.y_bf16, stream);
}

int launch_int4_sum(const float *slabs, int ks, int64_t m, int64_t n, const float *bias, void *y, int y_bf16, void *stream) {
    const int64_t count = m * n;
    hipLaunchKernelGGL(int4_sum_kernel, dim3((unsigned)std::min<int64_t>((count + 255) / 256, 8192)), dim3(256), 0,
                       (hipStream_t)stream, slabs, ks, count, n, bias, y, y_bf16);
    return (int)hipGetLastError();
}

}  // namespace nnq
