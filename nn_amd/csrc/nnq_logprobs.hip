// Log probabilities of given tokens on gfx950: for each row of logits l[0 .. n)
//   M = max l,  d_i = l_i - M,  R = sum of e^(d_i) over all but one element with d_i = 0,
//   S = sum of d_i e^(d_i),  log Z = log1p(R)
//   log p_t = d_t - log Z,  entropy = log Z - S / (1 + R)   (both terms >= 0: nothing cancels),
//   rank_t = #{l_i > l_t} + #{l_i = l_t, i < t},  and the N largest l_i (lowest index first among
//   equals) with their log probabilities.
// Keeping the maximum's own 1 out of R holds the log probability of a nearly certain token, and
// the entropy of such a row, to a relative 2^-23 where 1 + R would round R away.
//
// Bound: one read of the logits (HBM, or the cache that a GEMM left them in), with some fourteen
// VALU instructions and an exponential per logit beside it.  Two launches:
//   logprob_seg_kernel   one wave per 2048 logits of a row, all of them in registers: the segment's
//                        maximum, then (count of the maximum, R, S) against it, how many logits
//                        come before the token, and the candidates of the top N.
//   logprob_join_kernel  one workgroup per row: the segments' sums rescaled to the row's maximum
//                        and added in a fixed order, and the N largest candidates by rank.
// Candidates of a segment: the N-th largest of the 64 lanes' maxima is a lower bound of the N-th
// largest logit (N <= 32), found with ballots over its bits; on continuous logits about 1.2 N of
// the 2048 reach it (N = 20).  Where more do than there are slots (many equal logits, or a row's
// largest in few lanes) the exact N-th value, and among its equals the lowest indices, are
// found the same way over all 2048.
#include <algorithm>

#include "nnq_device.h"
#include "nnq_internal.h"

namespace nnq {

namespace {

constexpr int kSeg = 2048;          // logits of a wave
constexpr int kPer = kSeg / 64;     // logits of a lane
constexpr int kSegWaves = 4;
constexpr int kJoinThreads = 256;
constexpr int kJoinList = 1024;     // candidates that the join ranks in LDS
constexpr float kNegInf = -__builtin_huge_valf();
constexpr uint32_t kOrdNegInf = 0x007FFFFFu;

// what a wave leaves of its segment
struct SegStat {
    float mx;       // the maximum (-inf: no logit above -inf)
    float r, s;     // sums of e^d and d e^d over the elements below the maximum, d against it
    uint32_t cnt;   // elements equal to the maximum
};

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

struct LpArgs {
    const void *logits;
    const int64_t *tokens;
    int64_t row0, n, stride;  // row0: the launch's first row
    int64_t nseg;             // segments of a row (a multiple of kSegWaves)
    int top, slots, ranks;
    SegStat *stat;            // [rows][nseg]
    uint32_t *before;         // [rows][nseg] (ranks)
    uint64_t *cand;           // [rows][nseg][slots] (top)
    float *logprob, *entropy;
    int64_t *rank;
    float *top_lp;
    int64_t *top_id;
};

// The largest t with at least `want` lanes' or elements' keys >= t, count(t) counting them
// (non-increasing in t; count(0) >= want).
template <class F>
__device__ __forceinline__ uint32_t largest_with(int want, F &&count) {
    uint32_t t = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
        if (count(t | bit) >= want) t |= bit;
    return t;
}

template <class T, bool RANK, bool TOP>
__global__ __launch_bounds__(kSegWaves * 64) void logprob_seg_kernel(LpArgs a) {
    constexpr int V = 16 / (int)sizeof(T);  // logits of one 16-byte load
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t rl = blockIdx.y, row = a.row0 + rl;
    const int64_t seg = (int64_t)blockIdx.x * kSegWaves + wv;
    const T *p = reinterpret_cast<const T *>(a.logits) + row * a.stride;
    // 16-byte loads at aligned addresses: slot i of the row holds logit i - off, the slots before 0
    // and from n on hold none
    const int off = (int)(((uintptr_t)p / sizeof(T)) % V);
    const int64_t base = seg * kSeg + (int64_t)lane * V - off;  // logit of element 0
    float x[kPer];
#pragma unroll
    for (int v = 0; v < kPer / V; v++) {
        const int64_t i = base + v * 64 * V;
        if (i >= 0 && i + V <= a.n) {
            widen16<T>(*reinterpret_cast<const u32x4 *>(p + i), x + v * V);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) x[v * V + e] = i + e >= 0 && i + e < a.n ? widen<T>(p[i + e]) : kNegInf;
        }
    }
    int64_t tok = -1;
    float lt = 0.f;
    bool ask = false;
    if constexpr (RANK) {
        tok = a.tokens[row];
        ask = tok >= 0 && tok < a.n;
        if (ask) lt = widen<T>(p[tok]);
    }

    // (fmaxf passes over NaN; a NaN reaches R and S through its difference)
    float lm = x[0];
#pragma unroll
    for (int e = 1; e < kPer; e++) lm = fmaxf(lm, x[e]);
    const float mx = wave_max(lm);
    const float ref = mx == kNegInf ? 0.f : mx;
    float r = 0.f, s = 0.f;
    int cnt = 0;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const float d = x[e] - ref;
        const float ex = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
        const bool top = d == 0.f;
        cnt += __popcll(__ballot(top));
        r += top ? 0.f : ex;
        s = fmaf(fmaxf(d, -1e30f), ex, s);  // (d = -inf: its e^d is 0)
    }
    r = wave_sum(r);
    s = wave_sum(s);
    const int64_t at = rl * a.nseg + seg;
    if (lane == 0) a.stat[at] = SegStat{mx, r, s, (uint32_t)cnt};

    if constexpr (RANK) {
        uint32_t before = 0;
        if (ask) {
#pragma unroll
            for (int e = 0; e < kPer; e++) {
                before += __popcll(__ballot(x[e] > lt));
                const uint64_t same = __ballot(x[e] == lt);
                if (same) {  // (slots outside the row are -inf, as a masked token is)
                    const int64_t i = base + (e / V) * 64 * V + e % V;
                    before += __popcll(same & __ballot(i >= 0 && i < tok));
                }
            }
        }
        if (lane == 0) a.before[at] = before;
    }

    if constexpr (TOP) {
        __shared__ uint64_t list[kSegWaves][64];
        const int want = a.top;
        const uint32_t mine = lm == lm ? ord(lm) : 0;  // (no number in the lane)
        const uint32_t lanes = largest_with(want, [&](uint32_t k) { return __popcll(__ballot(mine >= k)); });
        float t = unord(max(lanes, kOrdNegInf));  // (-inf is no candidate)
        int total = 0;
#pragma unroll
        for (int e = 0; e < kPer; e++) total += __popcll(__ballot(x[e] >= t && x[e] > kNegInf));
        int32_t upto = 0x7FFFFFFF;  // logits equal to t count up to this place of the segment
        if (total > a.slots) {
            t = unord(largest_with(want, [&](uint32_t k) {
                const float f = unord(k);
                int c = 0;
#pragma unroll
                for (int e = 0; e < kPer; e++) c += __popcll(__ballot(x[e] >= f && x[e] > kNegInf));
                return c;
            }));
            int more = 0;
#pragma unroll
            for (int e = 0; e < kPer; e++) more += __popcll(__ballot(x[e] > t));
            // the lowest `need` of the logits equal to t: the largest bound with fewer, plus one
            const int need = want - more;
            uint32_t b = 0;
            for (uint32_t bit = kSeg / 2; bit; bit >>= 1) {
                int c = 0;
#pragma unroll
                for (int e = 0; e < kPer; e++)
                    c += __popcll(__ballot(x[e] == t && (uint32_t)((e / V) * 64 * V + lane * V + e % V) < (b | bit)));
                if (c < need) b |= bit;
            }
            upto = (int32_t)b;
        }
        int at_list = 0;
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const int place = (e / V) * 64 * V + lane * V + e % V;
            const bool in = x[e] > kNegInf && (x[e] > t || (x[e] == t && place <= upto));
            const uint64_t b = __ballot(in);
            if (b) {
                if (in) {
                    const int slot = at_list + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
                    if (slot < 64) list[wv][slot] = cand_key(x[e], (uint32_t)(base + (e / V) * 64 * V + e % V));
                }
                at_list += __popcll(b);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (lane < a.slots) a.cand[at * a.slots + lane] = lane < at_list ? list[wv][lane] : 0ull;
    }
}

// sum (or max) over the workgroup of kJoinThreads, the same value in every thread; `tmp` holds
// one value per wave and is free again after the call
template <class T, class F>
__device__ __forceinline__ T join_reduce(T v, T *tmp, F &&f) {
    for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    v = tmp[0];
#pragma unroll
    for (int w = 1; w < kJoinThreads / 64; w++) v = f(v, tmp[w]);
    return v;
}

template <class T>
__global__ __launch_bounds__(kJoinThreads) void logprob_join_kernel(LpArgs a) {
    __shared__ float tf[kJoinThreads / 64];
    __shared__ uint32_t tu[kJoinThreads / 64];
    __shared__ uint64_t list[kJoinList];
    __shared__ uint64_t maxima[kJoinThreads];
    __shared__ uint32_t listed, bound;
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t rl = blockIdx.x, row = a.row0 + rl;
    const SegStat *st = a.stat + rl * a.nseg;
    const auto add = [](auto u, auto v) { return u + v; };
    const auto larger = [](auto u, auto v) { return u > v ? u : v; };
    float mx = kNegInf;
    for (int64_t i = tid; i < a.nseg; i += kJoinThreads) mx = fmaxf(mx, st[i].mx);
    mx = join_reduce(mx, tf, larger);
    // each segment's sums move by e^(its maximum - the row's); a row without a logit above -inf gives
    // -inf - -inf = NaN here, and a NaN among the logits came with its segment's sums
    float r = 0.f, s = 0.f;
    uint32_t cnt = 0;
    for (int64_t i = tid; i < a.nseg; i += kJoinThreads) {
        const SegStat q = st[i];
        const float d = q.mx - mx;
        if (d == 0.f) {
            cnt += q.cnt;
            r += q.r;
            s += q.s;
        } else {
            const float f = expf(d), z = (float)q.cnt + q.r;
            r += f * z;
            s += f * fmaf(fmaxf(d, -1e30f), z, q.s);
        }
    }
    r = join_reduce(r, tf, add);
    s = join_reduce(s, tf, add);
    cnt = join_reduce(cnt, tu, add);
    r += (float)cnt - 1.f;  // (exact up to 2^24 equal maxima)
    if (mx == kNegInf) r = __uint_as_float(0x7FC00000u);
    const float lz = log1pf(r);
    const float nan = __uint_as_float(0x7FC00000u);
    if (tid == 0) {
        const int64_t tok = a.tokens[row];
        const bool ask = tok >= 0 && tok < a.n;
        const float lt = ask ? widen<T>(reinterpret_cast<const T *>(a.logits)[row * a.stride + tok]) : nan;
        a.logprob[row] = (lt - mx) - lz;
        if (a.entropy) a.entropy[row] = lz - s / (1.f + r);
    }
    if (a.rank) {
        uint32_t before = 0;
        for (int64_t i = tid; i < a.nseg; i += kJoinThreads) before += a.before[rl * a.nseg + i];
        before = join_reduce(before, tu, add);
        if (tid == 0) {
            const float lp = a.logprob[row];  // this thread's own store
            a.rank[row] = lp == lp ? (int64_t)before : -1;
        }
    }
    if (a.top == 0) return;

    // The top N of the segments' candidates.  As in a segment: the N-th largest of the maxima of 64
    // parts bounds the N-th largest key's value from below.
    const uint64_t *c = a.cand + rl * a.nseg * a.slots;
    const int64_t total = a.nseg * a.slots;
    uint64_t best = 0;
    for (int64_t i = tid; i < total; i += kJoinThreads) best = larger(best, c[i]);
    maxima[tid] = best;
    if (tid == 0) listed = 0;
    __syncthreads();
    if (tid < 64) {
        uint64_t m = maxima[lane];
#pragma unroll
        for (int w = 1; w < kJoinThreads / 64; w++) m = larger(m, maxima[64 * w + lane]);
        const uint32_t v = (uint32_t)(m >> 32);
        const uint32_t t = largest_with(a.top, [&](uint32_t k) { return __popcll(__ballot(v >= k)); });
        if (lane == 0) bound = t;
    }
    __syncthreads();
    uint64_t low = max((uint64_t)bound << 32, (uint64_t)1);
    const auto collect = [&]() {
        for (int64_t i = tid; i < total; i += kJoinThreads) {
            const uint64_t k = c[i];
            if (k >= low) {
                const uint32_t at = atomicAdd(&listed, 1u);
                if (at < kJoinList) list[at] = k;
            }
        }
        __syncthreads();
    };
    collect();
    if (listed > kJoinList) {
        // very many equal values: the exact N-th largest key (keys are unique), bit by bit
        __syncthreads();
        uint64_t t = 0;
        for (uint64_t bit = 1ull << 63; bit; bit >>= 1) {
            uint32_t k = 0;
            for (int64_t i = tid; i < total; i += kJoinThreads) k += c[i] >= (t | bit);
            if (join_reduce(k, tu, add) >= (uint32_t)a.top) t |= bit;
        }
        low = max(t, (uint64_t)1);
        if (tid == 0) listed = 0;
        __syncthreads();
        collect();
    }
    const int got = (int)listed;  // at most kJoinList: unique keys
    for (int i = tid; i < got; i += kJoinThreads) {
        const uint64_t k = list[i];
        int ahead = 0;
        for (int j = 0; j < got; j++) ahead += list[j] > k;
        if (ahead < a.top) {
            a.top_id[row * a.top + ahead] = (int64_t)(0xFFFFFFFFu - (uint32_t)k);
            a.top_lp[row * a.top + ahead] = (unord((uint32_t)(k >> 32)) - mx) - lz;
        }
    }
    // fewer logits above -inf than places
    if (tid >= got && tid < a.top) {
        a.top_id[row * a.top + tid] = -1;
        a.top_lp[row * a.top + tid] = lz == lz ? kNegInf : nan;
    }
}

template <class T>
int launch_lp(const LpArgs &a, int64_t rows, void *stream) {
    const dim3 grid((unsigned)(a.nseg / kSegWaves), (unsigned)rows), block(kSegWaves * 64);
    if (a.rank && a.top)
        hipLaunchKernelGGL((logprob_seg_kernel<T, true, true>), grid, block, 0, (hipStream_t)stream, a);
    else if (a.rank)
        hipLaunchKernelGGL((logprob_seg_kernel<T, true, false>), grid, block, 0, (hipStream_t)stream, a);
    else if (a.top)
        hipLaunchKernelGGL((logprob_seg_kernel<T, false, true>), grid, block, 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL((logprob_seg_kernel<T, false, false>), grid, block, 0, (hipStream_t)stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL((logprob_join_kernel<T>), dim3((unsigned)rows), dim3(kJoinThreads), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

}  // namespace

int launch_logprobs(const LogprobArgs &g, int64_t m, void *scratch, void *stream) {
    const LogprobPlan pl = logprob_plan(m, g.n, g.top, g.dtype == NNQ_F32 ? 4 : 2);
    LpArgs a{};
    a.logits = g.logits;
    a.tokens = g.tokens;
    a.n = g.n;
    a.stride = g.stride;
    a.nseg = pl.nseg;
    a.top = g.top;
    a.slots = pl.slots;
    a.logprob = g.logprob;
    a.entropy = g.entropy;
    a.rank = g.rank;
    a.top_lp = g.top_lp;
    a.top_id = g.top_id;
    uint8_t *p = reinterpret_cast<uint8_t *>(scratch);
    a.cand = reinterpret_cast<uint64_t *>(p);
    a.stat = reinterpret_cast<SegStat *>(p + (size_t)pl.rows * pl.nseg * pl.slots * 8);
    a.before = reinterpret_cast<uint32_t *>(a.stat + (size_t)pl.rows * pl.nseg);
    for (int64_t r = 0; r < m; r += pl.rows) {
        a.row0 = r;
        const int64_t rows = std::min(pl.rows, m - r);
        const int e = g.dtype == NNQ_F32 ? launch_lp<float>(a, rows, stream)
                      : g.dtype == NNQ_BF16 ? launch_lp<Bf16>(a, rows, stream) : launch_lp<F16>(a, rows, stream);
        if (e) return e;
    }
    return 0;
}

}  // namespace nnq
