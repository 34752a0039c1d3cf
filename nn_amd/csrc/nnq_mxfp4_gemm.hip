// Linears over MXFP4 rows on gfx950 for more than sixteen token rows (nnq_mxfp4.hip has the formula and the image).
//  * mx_gemm16_kernel: x in bf16 (f32 x: three bf16 planes that sum to it), 32x32x16 bf16 MFMAs.  A code times its
//    scale is exact in bf16, one conversion for two of them, so nothing is scaled afterwards.
//  * mx_gemm4_kernel: x quantized to MXFP4, 32x32x64 block-scaled MFMAs on the codes and scales as they are.
// A workgroup of four waves takes MT * 32 rows and NT * 128 columns.  The A pieces of a stage of K are copied straight to
// LDS (three buffers, two stages ahead, in the bf16 kernel with stages of 128 k; two buffers with stages of 256 k), with one
// barrier a stage; a wave's weights go from memory into its registers as far ahead, and none passes through LDS.  With too
// few workgroups K is split: f32 slabs, added in order.
// Measured (MI355X, in a graph over copies of the weight that pass the Infinity Cache; the library's bf16 product of 8192^3
// reaches 1.14 PFLOP/s; the MFMAs alone from registers, on random data, 1.61 in bf16 and 6.4 in 4 bits):
//  * 512 bf16 rows of 4096 -> 12288 46 to 51 us, 1.0 to 1.1 PFLOP/s; 2048 rows 172 us, 1.2: bound by the MFMAs at the clock that
//    they leave.  f32 rows take three MFMAs for one: 512 of them 120 to 130 us, 1.2 PFLOP/s of MFMAs, 2048 469.
//  * 2048 rows of 4096 -> 24576 in 4 bits 104 to 113 us with 7 of quantization, 3.7 to 3.9 PFLOP/s (125 to 129 in
//    graphs of three such calls in later runs).  Variants that leave work out say what of the kernel's 103: the MFMAs alone 60, with
//    the LDS reads 65, the copies of A 72, the loads of B 91, the stores 103.  Counters: L1's address unit busy 83% of the
//    cycles, its data return 96%, the matrix pipe 50%, one 64-byte access in 46%: the loads' path, or what two waves a SIMD hide of
//    it.  256 x 256 outputs a CU with both operands through LDS have a third less loads, but one wave a SIMD (126 us), so they
//    do not tell these apart; 256 rows with the weights in registers (122), a third buffer (112) and eight waves that share A
//    (115 / 115) were no faster.
//  * 301 f32 rows of 2880 -> 5751 in 4 bits 18 us: latency of two launches, 12 stages and the first loads.
#include <algorithm>
#include <type_traits>

#include "nnq_device.h"
#include "nnq_internal.h"
#include "nnq_mxfp4.h"

namespace nnq {

namespace {

constexpr int W = 4;          // waves of a workgroup
constexpr int kPiece = 8192;  // bf16 bytes of 32 rows and one unit

__device__ __forceinline__ floatx16 mfma32_bf16(u32x4 a, u32x4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int BYTE>
__device__ __forceinline__ floatx16 mfma32_mx(u32x4 a, uint32_t sa, u32x4 b, uint32_t sb, floatx16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, BYTE, (int)sa, BYTE, (int)sb);
#else
    return c;
#endif
}

// bytes of a stage's A in LDS: 2 mt tiles' codes, and two tiles' scales of each of the four waves
constexpr int mx_gemm4_stage(int mt) { return 2 * mt * 2048 + 1024; }
// 4 bytes a lane from a buffer straight into LDS
__device__ __forceinline__ void copy4_lds(__amdgpu_buffer_rsrc_t t, uint8_t *lds, int voff, int soff) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(t, (__attribute__((address_space(3))) void *)lds, 4, voff, soff, 0, 0);
#endif
}

typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
// a wave's LDS for 32 rows of 128 bytes of outputs
constexpr int kOutRow = 144, kOutBuf = 32 * kOutRow;

struct MxGemmArgs {
    const uint8_t *w, *x;  // x: bf16 planes [P][m][k], or the records of the quantized rows
    const float *bias;
    void *y;               // [m][n], or with ks > 1 f32 slabs [ks][m][n] without the bias
    int y_bf16;
    int m, units, ntile, ks;
    int row_blocks, col_blocks;
    int64_t n, k;
};

// where a workgroup works: workgroup ids go round the 8 XCDs, each takes a contiguous run, the row blocks of a column
// block (which share its weights) one after another
struct MxPlace {
    int rb, cb, kp, u0, u1;
    __device__ __forceinline__ explicit MxPlace(const MxGemmArgs &a) {
        const int total = a.row_blocks * a.col_blocks * a.ks, bid = (int)blockIdx.x;
        const int per = total / 8, extra = total % 8, xcd = bid % 8, at = bid / 8;
        const int t = xcd * per + min(xcd, extra) + at;
        rb = t % a.row_blocks;
        cb = t / a.row_blocks % a.col_blocks;
        kp = t / (a.row_blocks * a.col_blocks);
        const int64_t pairs = (a.units + 1) / 2;  // parts of K are whole pairs of units
        u0 = (int)(pairs * kp / a.ks) * 2;
        u1 = min((int)(pairs * (kp + 1) / a.ks) * 2, a.units);
    }
};

// A wave's weights, NT * 32 columns: lane 32h + 16b + r holds row r of tile b of a pair of tiles.
template <int NT>
struct MxW {
    __amdgpu_buffer_rsrc_t buf[NT];
    int off[NT];  // of the lane's tile; tiles past the last are read as the last (not stored)
    int slot;
    __device__ __forceinline__ MxW(const MxGemmArgs &a, int tile0, int lane) {
        slot = 16 * (lane >> 5) + (lane & 15);
        const int bytes = (a.units + 1) / 2 * kMxPair;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int t = min(tile0 + 2 * nt, a.ntile - 1);
            buf[nt] = rsrc(a.w + (int64_t)t * bytes, (int64_t)min(2, a.ntile - t) * bytes);
            off[nt] = (lane & 16) && t + 1 < a.ntile ? bytes : 0;
        }
    }
    // blocks 2s + h of a pair of units (s from 0 to 3), and the word of their scales (byte s)
    __device__ __forceinline__ u32x4 codes(int nt, int pair, int s) const {
        return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(buf[nt], off[nt] + 16 * slot, pair * kMxPair + 512 * s, 0));
    }
    __device__ __forceinline__ uint32_t scales(int nt, int pair) const {
        return __builtin_amdgcn_raw_buffer_load_b32(buf[nt], off[nt] + 4 * slot, pair * kMxPair + 2048, 0);
    }
    // of one unit: bytes i for blocks 2i + h
    __device__ __forceinline__ uint32_t scales16(int nt, int u) const {
        return __builtin_amdgcn_raw_buffer_load_b16(buf[nt], off[nt] + 4 * slot, (u >> 1) * kMxPair + 2048 + 2 * (u & 1), 0);
    }
};

// every wave's copies into LDS, but for the N youngest loads and copies of each, have landed and can be read
template <int N>
__device__ __forceinline__ void arrive() {
    wait_vmcnt<N>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// lane: column lane % 32 of each 32, rows 8 i + 4h + e of each 32-row tile.  The bias is read and added before the first
// store: a wait for a load waits for the stores before it, too.
template <int MT, int NT>
__device__ __forceinline__ void mx_store(const MxGemmArgs &a, const MxPlace &at, int tile0, int wv, int lane, uint8_t *lds,
                                         floatx16 (&acc)[MT][NT]) {
    const bool slab = a.ks > 1;
    const int h = lane >> 5;
    if (a.bias && !slab) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int64_t col = (int64_t)(tile0 + 2 * nt) * kTile + (lane & 31);
            const float bias = a.bias[min(col, a.n - 1)];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[mt][nt][e] += bias;
        }
    }
    const bool bf16 = !slab && a.y_bf16;
    float *slabs = reinterpret_cast<float *>(a.y) + (slab ? (int64_t)at.kp * a.m * a.n : 0);
    wait_vmcnt<0>();  // (copies into LDS for stages past the last)
    // Through LDS, 32 rows of 128 bytes at a time, so that a store is eight rows' 16 bytes a lane.  The wave's own
    // part of what held A (every wave is past it), whose accesses stay in order.  Non-temporal: outputs in L2 would push
    // out the operands that the next workgroups share (2048 x 4096 -> 24576 in 4 bits: 109 us, 128 with plain stores).
    __syncthreads();
    uint8_t *mine = lds + wv * kOutBuf;
    auto flush = [&](auto bytes, int mt, uint8_t *y, int64_t col0, int elem) {  // rows of so many bytes; y: of element [0][0]
        constexpr int L = decltype(bytes)::value / 16;  // lanes of a row
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int64_t col = col0 + lane % L * (16 / elem);
#pragma unroll
        for (int i = 0; i < L / 2; i++) {
            const int r = 64 / L * i + lane / L;
            const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + r * kOutRow + lane % L * 16);
            const int64_t row = (at.rb * MT + mt) * 32 + r;
            uint8_t *o = y + (row * a.n + col) * elem;
            if (row >= a.m || col >= a.n) continue;
            if (col + 16 / elem <= a.n) {  // (16 bytes at the element's alignment: rows need not be whole pieces)
                if (elem == 4) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_at4 *>(o));
                else __builtin_nontemporal_store(v, reinterpret_cast<u32x4_at2 *>(o));
            } else {
                for (int e = 0; e < 16 / elem && col + e < a.n; e++) {
                    if (elem == 4) reinterpret_cast<uint32_t *>(o)[e] = v[e];
                    else reinterpret_cast<uint16_t *>(o)[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        if ((at.rb * MT + mt) * 32 >= a.m) return;
        const int64_t col0 = (int64_t)tile0 * kTile;
        uint8_t *p = mine + 4 * h * kOutRow;
        if (bf16) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    *reinterpret_cast<__bf16 *>(p + (8 * (e / 4) + e % 4) * kOutRow + (32 * (nt & 1) + (lane & 31)) * 2) = (__bf16)acc[mt][nt][e];
                if (nt & 1) flush(std::integral_constant<int, 128>(), mt, reinterpret_cast<uint8_t *>(a.y), col0 + 32 * (nt - 1), 2);
                else if (nt == NT - 1) flush(std::integral_constant<int, 64>(), mt, reinterpret_cast<uint8_t *>(a.y), col0 + 32 * nt, 2);
            }
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    *reinterpret_cast<float *>(p + (8 * (e / 4) + e % 4) * kOutRow + (lane & 31) * 4) = acc[mt][nt][e];
                flush(std::integral_constant<int, 128>(), mt, reinterpret_cast<uint8_t *>(slabs), col0 + 32 * nt, 4);
            }
        }
    }
}

template <int MT, int NT>
__device__ __forceinline__ void mx_clear(floatx16 (&acc)[MT][NT]) {
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[mt][nt][e] = 0.f;
}

// LDS of an A piece: row r's 16-byte chunk c (columns 8c .. 8c + 7 of the unit) at r * 256 + (c ^ r % 16) * 16: a copy
// moves whole 256-byte rows, and the 16 lanes that read one chunk of 16 rows together find it in 16 different
// places of the banks.
template <int MT, int NT, int P>
__global__ __launch_bounds__(W * 64, 2) void mx_gemm16_kernel(MxGemmArgs a) {
    constexpr int BUF = MT * P * kPiece, NA = BUF / (W * 1024);  // copies of a wave and unit
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const MxPlace at(a);
    const int tile0 = (at.cb * W + wv) * 2 * NT;
    const MxW<NT> w(a, tile0, lane);
    // Copy i of a wave: rows 4 (i W + wv) .. + 3 of the pieces [plane][row tile][32 rows].  Rows past m are not read (zeros);
    // they are not stored.
    const int k = (int)a.k;
    const int64_t plane = (int64_t)a.m * k * 2;
    const __amdgpu_buffer_rsrc_t xb = rsrc(a.x, P * plane);
    const int l16 = lane >> 4, swz = ((lane & 15) ^ ((4 * wv + l16) & 15)) * 8;  // (W = 4: row % 16 is the same for every i)
    auto copy_a = [&](int u, int buf) {
#pragma unroll
        for (int i = 0; i < NA; i++) {
            const int row = 4 * (i * W + wv), pl = row / (MT * 32);
            const int off = mx_x_offset(at.rb * MT * 32 + row % (MT * 32) + l16, a.m, k, u, swz);
            copy16_lds(xb, lds + buf * BUF + (i * W + wv) * 1024, off, pl * (int)plane + u * kMxUnit * 2);
        }
    };
    const int c32 = lane & 31, h = lane >> 5;
    floatx16 acc[MT][NT];
    mx_clear(acc);
    u32x4 bq[2][NT][2];
    uint32_t bs[2][NT];
    auto load_codes = [&](int u, int par, int i) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) bq[par][nt][i] = w.codes(nt, u >> 1, 2 * (u & 1) + i);
    };
    auto load_scales = [&](int u, int par) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) bs[par][nt] = w.scales16(nt, u);
    };
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int u = min(at.u0 + i, at.u1 - 1);
        copy_a(u, i);
        __builtin_amdgcn_sched_barrier(0);
        load_codes(u, i, 0);
        load_codes(u, i, 1);
        load_scales(u, i);
        __builtin_amdgcn_sched_barrier(0);
    }
    int cur = 0;  // this unit's LDS buffer of three
    // Operands are formed, and A read, a step ahead of the MFMAs; a unit's weights are loaded for the unit after next as soon
    // as they have been used.
    auto unit = [&](auto parity, int u) {
        constexpr int par = decltype(parity)::value;
        // this unit's copies have landed: behind them came its loads, and the next unit's copies and loads
        arrive<NA + 2 * 3 * NT>();
        const int next = min(u + 2, at.u1 - 1);
        const uint8_t *from = lds + cur * BUF + c32 * 256;
        copy_a(next, cur == 0 ? 2 : cur - 1);
        cur = cur == 2 ? 0 : cur + 1;
        __builtin_amdgcn_sched_barrier(0);
        u32x4 af[2][P][MT], bf[2][NT];
        auto form = [&](int s) {  // step s: word s % 4 of blocks 2 (s / 4) + h
            const int chunk = (2 * (s >> 2) + h) * 4 + (s & 3);
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
                    af[s & 1][p][mt] = *reinterpret_cast<const u32x4 *>(from + (p * MT + mt) * kPiece + ((chunk ^ (c32 & 15)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
                bf[s & 1][nt] = mx_codes_bf16(bq[par][nt][s >> 2][s & 3], mx_scale((bs[par][nt] >> (8 * (s >> 2))) & 0xFFu));
        };
        form(0);
#pragma unroll
        for (int s = 0; s < 8; s++) {
            if (s < 7) form(s + 1);
            if (s == 3) load_codes(next, par, 0);
            if (s == 7) {
                load_codes(next, par, 1);
                load_scales(next, par);
            }
            // (the lo plane first: added to a finished hi sum its low bits would be cut off)
#pragma unroll
            for (int p = P - 1; p >= 0; p--)
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) acc[mt][nt] = mfma32_bf16(af[s & 1][p][mt], bf[s & 1][nt], acc[mt][nt]);
            if (s == 3 || s == 7) __builtin_amdgcn_sched_barrier(0);
        }
    };
    int u = at.u0;
    for (; u + 1 < at.u1; u += 2) {
        unit(std::integral_constant<int, 0>(), u);
        unit(std::integral_constant<int, 1>(), u + 1);
    }
    if (u < at.u1) unit(std::integral_constant<int, 0>(), u);
    mx_store(a, at, tile0, wv, lane, lds, acc);
}

// A stage is a pair of units (256 k).  A wave's B operands are loaded for the next stage as soon as a step has used them;
// the A records are copied to the other LDS buffer.  Copies are issued before the loads of a stage, so that the wait for
// them at the next one leaves the loads in flight.
template <int MT, int NT>
__global__ __launch_bounds__(W * 64, 2) void mx_gemm4_kernel(MxGemmArgs a) {
    constexpr int REC = 2 * MT;                // 16-row tiles
    constexpr int BUF = mx_gemm4_stage(MT);    // codes [REC][2048], then scales [REC][128] (at least 1 KB of them)
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const MxPlace at(a);
    const int tile0 = (at.cb * W + wv) * 2 * NT;
    const MxW<NT> w(a, tile0, lane);
    const int mtiles = (a.m + 15) / 16, bytes = (a.units + 1) / 2 * kMxPair;
    const __amdgpu_buffer_rsrc_t xb = rsrc(a.x, (int64_t)mtiles * bytes);
    // (row tiles past the last: the last one again, not stored)
    auto copy_a = [&](int pair, int buf) {
#pragma unroll
        for (int i = 0; i < MT; i++) {  // 2 REC pieces of 1 KB
            const int piece = i * W + wv;
            copy16_lds(xb, lds + buf * BUF + piece * 1024, 16 * lane,
                       min(at.rb * REC + piece / 2, mtiles - 1) * bytes + pair * kMxPair + piece % 2 * 1024);
        }
        // two tiles' scales a wave
        const int rec = min(at.rb * REC + (2 * wv + (lane >> 5)) % REC, mtiles - 1);
        copy4_lds(xb, lds + buf * BUF + REC * 2048 + wv * 256, rec * bytes + 4 * (lane & 31), pair * kMxPair + 2048);
    };
    const int b16 = (lane >> 4) & 1;
    floatx16 acc[MT][NT];
    mx_clear(acc);
    u32x4 bq[NT][4];
    uint32_t bs[2][NT];
    auto load_scales = [&](int pair, int buf) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) bs[buf][nt] = w.scales(nt, pair);
    };
    const int v0 = at.u0 / 2, v1 = (at.u1 + 1) / 2;  // (parts of K are whole pairs)
    copy_a(v0, 0);
    __builtin_amdgcn_sched_barrier(0);
    load_scales(v0, 0);
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) bq[nt][s] = w.codes(nt, v0, s);
    auto stage = [&](auto parity, int v) {
        constexpr int buf = decltype(parity)::value;
        arrive<5 * NT>();  // this stage's copies: behind them came its loads
        const int next = min(v + 1, v1 - 1);
        copy_a(next, buf ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        load_scales(next, buf ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        uint32_t as[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
            as[mt] = *reinterpret_cast<const uint32_t *>(lds + buf * BUF + REC * 2048 + (2 * mt + b16) * 128 + 4 * w.slot);
        // The next step's A is read, and this step's B loaded anew, between the MFMAs: left to itself the scheduler moves
        // all the loads to the stage's end, where the next stage waits for them.
        u32x4 af[2][MT];
        auto read_a = [&](int s) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
                af[s & 1][mt] = *reinterpret_cast<const u32x4 *>(lds + buf * BUF + (2 * mt + b16) * 2048 + 512 * s + 16 * w.slot);
        };
        read_a(0);
        auto step = [&](auto which) {
            constexpr int s = decltype(which)::value;
            if constexpr (s < 3) read_a(s + 1);
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) acc[mt][nt] = mfma32_mx<s>(af[s & 1][mt], as[mt], bq[nt][s], bs[buf][nt], acc[mt][nt]);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) bq[nt][s] = w.codes(nt, next, s);
            __builtin_amdgcn_sched_barrier(0);
        };
        step(std::integral_constant<int, 0>());
        step(std::integral_constant<int, 1>());
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
        __builtin_amdgcn_sched_barrier(0);
    };
    int v = v0;
    for (; v + 1 < v1; v += 2) {
        stage(std::integral_constant<int, 0>(), v);
        stage(std::integral_constant<int, 1>(), v + 1);
    }
    if (v < v1) stage(std::integral_constant<int, 0>(), v);
    mx_store(a, at, tile0, wv, lane, lds, acc);
}

template <int MT, int NT, int P>
int launch16(const MxGemmArgs &a, void *stream) {
    constexpr size_t lds = std::max(3 * MT * P * kPiece, W * kOutBuf);
    auto *kernel = mx_gemm16_kernel<MT, NT, P>;
    hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), lds);
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.row_blocks * a.col_blocks * a.ks)), dim3(W * 64), lds, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}
template <int MT, int NT>
int launch4(const MxGemmArgs &a, void *stream) {
    constexpr size_t lds = std::max(2 * mx_gemm4_stage(MT), W * kOutBuf);
    auto *kernel = mx_gemm4_kernel<MT, NT>;
    hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), lds);
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.row_blocks * a.col_blocks * a.ks)), dim3(W * 64), lds, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

}  // namespace

int launch_mx_gemm(const MxArgs &a, void *scratch, void *stream) {
    const MxGemmPlan p = mx_gemm_plan(a.m, a.n, a.k, a.x_kind);
    if (a.m < 1 || a.m > INT32_MAX / 2 || a.units < 1 || (p.bytes && !scratch)) return (int)hipErrorInvalidValue;
    uint8_t *base = reinterpret_cast<uint8_t *>(scratch);
    float *slabs = reinterpret_cast<float *>(base + p.slabs);
    MxGemmArgs g{};
    g.w = a.w;
    g.x = reinterpret_cast<const uint8_t *>(a.x);
    g.bias = a.bias;
    g.y = p.ks > 1 ? (void *)slabs : a.y;
    g.y_bf16 = a.y_bf16;
    g.m = (int)a.m;
    g.units = (int)a.units;
    g.ntile = (int)a.ntile;
    g.ks = p.ks;
    g.row_blocks = p.row_blocks;
    g.col_blocks = p.col_blocks;
    g.n = a.n;
    g.k = a.k;
    int e = 0;
    if (a.x_kind != kMxBf16) {
        if (a.x_kind == kMxF32) e = launch_mx_split(reinterpret_cast<const float *>(a.x), a.m * a.k, reinterpret_cast<uint16_t *>(base), stream);
        else if (a.x_kind == kMxCodes) e = launch_mx_repack(reinterpret_cast<const uint8_t *>(a.x), a.xs, a.m, a.k, base, nullptr, stream);
        else e = launch_mx_quantize_image(a.x, a.x_kind == kMxQuantBf16, a.m, a.k, a.floor_rule, base, stream);
        if (e) return e;
        g.x = base;
    }
    const int tile = 10 * p.mt + p.nt;
    e = (int)hipErrorInvalidValue;
    if (a.x_kind == kMxBf16)
        e = tile == 12   ? launch16<1, 2, 1>(g, stream)
            : tile == 13 ? launch16<1, 3, 1>(g, stream)
            : tile == 22 ? launch16<2, 2, 1>(g, stream)
            : tile == 23 ? launch16<2, 3, 1>(g, stream) : e;
    else if (a.x_kind == kMxF32)
        e = tile == 12 ? launch16<1, 2, 3>(g, stream) : tile == 13 ? launch16<1, 3, 3>(g, stream) : e;
    else
        e = tile == 12   ? launch4<1, 2>(g, stream)
            : tile == 22 ? launch4<2, 2>(g, stream)
            : tile == 23 ? launch4<2, 3>(g, stream)
            : tile == 42 ? launch4<4, 2>(g, stream) : e;
    if (e || p.ks == 1) return e;
    return launch_int4_sum(slabs, p.ks, a.m, a.n, a.bias, a.y, a.y_bf16, stream);
}

}  // namespace nnq
