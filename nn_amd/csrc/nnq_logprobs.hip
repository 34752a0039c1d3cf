// Log probabilities of given tokens on gfx950: for each row of logits l[0 .. n)
//   M = max l,  d_i = l_i - M,  R = sum of e^(d_i) over all but one element with d_i = 0,
//   S = sum of d_i e^(d_i),  log Z = log1p(R)
//   log p_t = d_t - log Z,  entropy = log Z - S / (1 + R)   (both terms >= 0: nothing cancels),
//   rank_t = #{l_i > l_t} + #{l_i = l_t, i < t},  and the N largest l_i (lowest index first among
//   equals) with their log probabilities.
// Keeping the maximum's own 1 out of R holds the log probability of a nearly certain token, and
// the entropy of such a row, to a few 2^-24 relative to themselves where 1 + R would round R away: each term
// has its d's rounding, 2^-24 |d|, and 2^-22, and the sums theirs.  (Down to d = -87; below, e^d is taken
// for 0.)
//
// Bound: one read of the logits (HBM, or the cache that a GEMM left them in), with some fifteen VALU
// instructions and an exponential per logit beside it, twenty-three with rank and alternatives.  Two
// launches:
//   logprob_seg_kernel   one wave per 2048 logits of a row, all of them in registers: the segment's
//                        maximum, then (count of the maximum, R, S) against it, how many logits
//                        come before the token, and the candidates of the top N.
//   logprob_join_kernel  one workgroup per row: the segments' sums rescaled to the row's maximum
//                        and added in a fixed order, and the N largest candidates by rank.
// Candidates of a segment: the N-th largest of the 64 lanes' maxima is a lower bound of the N-th
// largest logit (N <= 32), found with ballots over its bits; on continuous logits about 1.2 N of
// the 2048 reach it (N = 20).  Of more than there are slots the largest are kept; of more than 64 (many
// equal logits, or a row's largest in few lanes) the exact N-th value, and among its equals the lowest
// indices, are found the same way over all 2048.
// Measured (MI355X, f32 logits of 151936): 512 rows 53.5 + 5.0 us (5.8 TB/s, the streaming read's rate
// is 7.0); 301 rows with rank and 5 alternatives 36.4 + 4.7 us (5.0 TB/s; the VALU is busy 90% of it);
// one row with 20 alternatives 6.2 + 5.1 us, both latency, and 19 us from Python (five tensors and two
// launches).  48 bf16 rows of 50257 7.8 + 4.8 us.
#include <algorithm>

#include "nnq_device.h"
#include "nnq_internal.h"
#include "nnq_logits.h"

namespace nnq {

namespace {

constexpr int kSegWaves = 4;
constexpr int kJoinThreads = 256;
constexpr int kJoinList = 1024;     // candidates that the join ranks in LDS

// what a wave leaves of its segment
struct SegStat {
    float mx;       // the maximum (-inf: no logit above -inf)
    float r, s;     // sums of e^d and d e^d over the elements below the maximum, d against it
    uint32_t cnt;   // elements equal to the maximum
};

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
    const float mx = max64(lm);
    const float ref = mx == kNegInf ? 0.f : mx;
    float r = 0.f, s = 0.f;
    int cnt = kSeg;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const float d = __builtin_elementwise_maximum(x[e] - ref, -1e30f);  // (-inf: its e^d is 0; NaN stays)
        const float ex = exp_of(d);
        const bool below = d != 0.f;  // (or NaN)
        cnt -= __popcll(__ballot(below));
        r += below ? ex : 0.f;
        s = fmaf(d, ex, s);
    }
    r = sum64(r);
    s = sum64(s);
    const int64_t at = rl * a.nseg + seg;
    if (lane == 0) a.stat[at] = SegStat{mx, r, s, (uint32_t)cnt};

    if constexpr (RANK) {
        // a segment before the token's counts equal logits, one after it does not
        const int64_t first = seg * kSeg - off;
        uint32_t before = 0;
        if (ask && lt <= mx) {  // (a likely token: few segments reach its logit)
            if (first > tok) {
#pragma unroll
                for (int e = 0; e < kPer; e++) before += x[e] > lt;
            } else if (first >= 0 && first + kSeg <= tok) {
#pragma unroll
                for (int e = 0; e < kPer; e++) before += x[e] >= lt;
            } else {  // (slots outside the row are -inf, as a masked token is)
                const int64_t from = -base, to = tok - base;  // places of logits 0 and tok, from the lane's first
#pragma unroll
                for (int e = 0; e < kPer; e++) {
                    const int place = (e / V) * 64 * V + e % V;
                    before += x[e] > lt || (x[e] == lt && place >= from && place < to);
                }
            }
        }
        before = sum64u(before);
        if (lane == 0) a.before[at] = before;
    }

    if constexpr (TOP) {
        __shared__ uint64_t list[kSegWaves][64];
        segment_candidates<V>(x, lm, base, a.top, a.slots, lane, list[wv], a.cand + at * a.slots);
    }
}

// One workgroup per row.  What it needs is loaded at once (a thread's first segment, its first kHeld
// keys, the token and its logit), and three barriers separate: the maxima; the sums against the row's
// maximum, and the bound of the N-th largest key; the list of candidates at or above it.
constexpr int kHeld = 8;
template <class T, bool TOP>
__global__ __launch_bounds__(kJoinThreads) void logprob_join_kernel(LpArgs a) {
    constexpr int NW = kJoinThreads / 64;
    struct Part {
        float r, s;
        uint32_t cnt, before;
    };
    __shared__ float wmax[NW];
    __shared__ Part part[NW];
    __shared__ uint64_t list[TOP ? kJoinList : 1], maxima[TOP ? kJoinThreads : 1];
    __shared__ uint32_t listed, bound, counts[NW];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int64_t rl = blockIdx.x, row = a.row0 + rl;
    const SegStat *st = a.stat + rl * a.nseg;
    const uint64_t *c = a.cand + rl * a.nseg * a.slots;
    const int64_t keys = a.nseg * a.slots;
    const float nan = __uint_as_float(0x7FC00000u);
    const int64_t tok = a.tokens[row];
    const bool ask = tok >= 0 && tok < a.n;
    const float lt = ask ? widen<T>(reinterpret_cast<const T *>(a.logits)[row * a.stride + tok]) : nan;
    SegStat q{kNegInf, 0.f, 0.f, 0};
    if (tid < a.nseg) q = st[tid];
    uint64_t held[kHeld], best = 0;
    if constexpr (TOP) {
#pragma unroll
        for (int i = 0; i < kHeld; i++) held[i] = tid + i * kJoinThreads < keys ? c[tid + i * kJoinThreads] : 0ull;
#pragma unroll
        for (int i = 0; i < kHeld; i++) best = max(best, held[i]);
        for (int64_t i = tid + kHeld * kJoinThreads; i < keys; i += kJoinThreads) best = max(best, c[i]);
        maxima[tid] = best;
    }
    float mx = q.mx;
    for (int64_t i = tid + kJoinThreads; i < a.nseg; i += kJoinThreads) mx = fmaxf(mx, st[i].mx);
    mx = max64(mx);
    if (lane == 0) wmax[wv] = mx;
    if (tid == 0) listed = 0;
    __syncthreads();

    mx = wmax[0];
#pragma unroll
    for (int w = 1; w < NW; w++) mx = fmaxf(mx, wmax[w]);
    // each segment's sums move by e^(its maximum - the row's); a row without a logit above -inf gives
    // -inf - -inf = NaN here, and a NaN among the logits came with its segment's sums
    Part t{0.f, 0.f, 0, 0};
    auto add = [&](const SegStat &g) {
        const float d = g.mx - mx;
        if (d == 0.f) {
            t.cnt += g.cnt;
            t.r += g.r;
            t.s += g.s;
        } else {
            const float f = expf(d), z = (float)g.cnt + g.r;
            t.r += f * z;
            t.s += f * fmaf(fmaxf(d, -1e30f), z, g.s);
        }
    };
    if (tid < a.nseg) add(q);
    for (int64_t i = tid + kJoinThreads; i < a.nseg; i += kJoinThreads) add(st[i]);
    if (a.rank)
        for (int64_t i = tid; i < a.nseg; i += kJoinThreads) t.before += a.before[rl * a.nseg + i];
    t.r = sum64(t.r);
    t.s = sum64(t.s);
    t.cnt = sum64u(t.cnt);
    t.before = sum64u(t.before);
    if (lane == 0) part[wv] = t;
    if (TOP && wv == 0) {
        // as in a segment: the N-th largest of the maxima of 64 parts
        uint64_t m = maxima[lane];
#pragma unroll
        for (int w = 1; w < NW; w++) m = max(m, maxima[64 * w + lane]);
        const uint32_t v = (uint32_t)(m >> 32);
        const uint32_t b = largest_with<24>(a.top, [&](uint32_t k) { return __popcll(__ballot(v >= k)); });
        if (lane == 0) bound = b;
    }
    __syncthreads();

    t = part[0];
#pragma unroll
    for (int w = 1; w < NW; w++) {
        t.r += part[w].r;
        t.s += part[w].s;
        t.cnt += part[w].cnt;
        t.before += part[w].before;
    }
    float r = t.r + ((float)t.cnt - 1.f);  // (exact up to 2^24 equal maxima)
    if (mx == kNegInf) r = nan;
    const float lz = log1pf(r);
    if (tid == 0) {
        const float lp = (lt - mx) - lz;
        a.logprob[row] = lp;
        if (a.entropy) a.entropy[row] = lz - t.s / (1.f + r);
        if (a.rank) a.rank[row] = lp == lp ? (int64_t)t.before : -1;
    }
    if constexpr (!TOP) return;

    uint64_t low = max((uint64_t)bound << 32, (uint64_t)1);
    auto take = [&](uint64_t k) {
        if (k >= low) {
            const uint32_t at = atomicAdd(&listed, 1u);
            if (at < kJoinList) list[at] = k;
        }
    };
    auto collect = [&]() {
#pragma unroll
        for (int i = 0; i < kHeld; i++) take(held[i]);
        for (int64_t i = tid + kHeld * kJoinThreads; i < keys; i += kJoinThreads) take(c[i]);
        __syncthreads();
    };
    collect();
    if (listed > kJoinList) {
        // very many equal values: the exact N-th largest key (keys are unique), bit by bit
        uint64_t least = 0;
        for (uint64_t bit = 1ull << 63; bit; bit >>= 1) {
            uint32_t k = 0;
            for (int64_t i = tid; i < keys; i += kJoinThreads) k += c[i] >= (least | bit);
            k = sum64u(k);
            __syncthreads();  // (the counts of the last bit have been read)
            if (lane == 0) counts[wv] = k;
            __syncthreads();
            k = 0;
#pragma unroll
            for (int w = 0; w < NW; w++) k += counts[w];
            if (k >= (uint32_t)a.top) least |= bit;
        }
        low = max(least, (uint64_t)1);
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
    if (a.top)
        hipLaunchKernelGGL((logprob_join_kernel<T, true>), dim3((unsigned)rows), dim3(kJoinThreads), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL((logprob_join_kernel<T, false>), dim3((unsigned)rows), dim3(kJoinThreads), 0, (hipStream_t)stream, a);
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
