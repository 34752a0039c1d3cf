// Beam search on gfx950: the choice of continuations, and the states that follow it.
//
// nnq_beam_select: item b's beam j with score s_j offers token t the value
//   v = s_j + l_t - log sum_i e^(l_i),
// and the `keep` largest of an item's values are wanted.  Within a beam v has the order of l, so the keep largest
// logits of every beam hold them.  Two launches:
//   beam_seg_kernel   one wave per 2048 logits of a beam: the maximum, the sum of e^(l - maximum), and the candidates
//                     (nnq_logits.h).  Beams that offer nothing by themselves (ended
//                     ones, scores of -inf) are not read.
//   beam_join_kernel  one workgroup per item: log sum e^l of each beam from its segments, in 64 bits and in a fixed
//                     order, and the largest values of the beams' candidates, compared in 64 bits.
// A row's segments begin at its multiples of 2048 wherever it lies, so that equal rows have equal sums and their
// continuations tie exactly.
// Bound: one read of the logits; small calls by the latency of two launches.  Measured (MI355X): four beams of 151936 with 8
// kept 5.6 + 6.1 us, 24 x 8 bf16 beams of 50257 with 16 kept 11.8 + 8.1, 64 x 5 f32 beams of 151936 38 + 9.4 (5.2 TB/s in
// the segments); sixteen beams of 151936 with 32 kept, whose 68000 candidates one workgroup reads, 30 in all.  Of the join
// 1 us each are the loads, the exponentials and logarithm in 64 bits, the bound of the keep-th value, and the ranking.
#include <algorithm>
#include <type_traits>

#include "nnq_device.h"
#include "nnq_internal.h"
#include "nnq_logits.h"

namespace nnq {

namespace {

constexpr int kBeamWaves = 4;
constexpr int kBeamThreads = 1024;
constexpr int kBeamList = 1024;  // candidates that the join ranks in LDS
constexpr int kStats = 2;        // segments that a lane of it holds
constexpr int kHeld = 4;         // pairs of candidates that a thread of it holds

struct BeamStat {
    float mx, r;  // a segment's maximum, the sum of e^(l - mx)
};

struct BeamDev {
    BeamArgs a;
    int64_t item0, nseg;  // the launch's first item
    int slots;
    BeamStat *stat;       // [items][beams][nseg]
    uint64_t *cand;       // [items][beams][nseg][slots]
};

__device__ __forceinline__ bool beam_ended(const BeamArgs &a, int64_t row) { return a.finished && a.finished[row]; }
__device__ __forceinline__ bool finite_score(float s) { return (__float_as_uint(s) & 0x7F800000u) != 0x7F800000u; }

// 16 bytes at the element's own alignment
typedef u32x4 u32x4_by2 __attribute__((aligned(2)));
typedef u32x4 u32x4_by4 __attribute__((aligned(4)));
template <class T>
__device__ __forceinline__ u32x4 load16(const T *p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const u32x4_by4 *>(p);
    else return *reinterpret_cast<const u32x4_by2 *>(p);
}

template <class T>
__global__ __launch_bounds__(kBeamWaves * 64) void beam_seg_kernel(BeamDev g) {
    constexpr int V = 16 / (int)sizeof(T);  // logits of one 16-byte load
    const BeamArgs &a = g.a;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int64_t rl = blockIdx.y, item = g.item0 + rl / a.beams, beam = rl % a.beams;
    const int64_t seg = (int64_t)blockIdx.x * kBeamWaves + wv;
    if (!finite_score(a.scores[item * a.beams + beam]) || beam_ended(a, item * a.beams + beam)) return;
    const T *p = reinterpret_cast<const T *>(a.logits) + item * a.batch_stride + beam * a.beam_stride;
    // 16 bytes at a time; fewer logits than all lanes' first loads one at a time, so that as many lanes as can be have
    // some: with fewer lanes than `keep` their maxima bound nothing, and the exact search behind that takes 13 us
    // (7 x 16 f16 beams of 80084 = 39 segments and 212 with 31 kept: 44 us the call, so 30)
    const int64_t start = seg * kSeg;
    const bool few = a.n - start < 64 * V;
    const int64_t base = start + (few ? lane : lane * V);  // logit of element 0
    float x[kPer];
    if (few) {
#pragma unroll
        for (int e = 0; e < kPer; e++) x[e] = kNegInf;
#pragma unroll
        for (int e = 0; e < V; e++)
            if (base + 64 * e < a.n) x[e] = widen<T>(p[base + 64 * e]);
    } else {
#pragma unroll
        for (int v = 0; v < kPer / V; v++) {
            const int64_t i = base + v * 64 * V;
            if (i + V <= a.n) {
                widen16<T>(load16(p + i), x + v * V);
            } else {
#pragma unroll
                for (int e = 0; e < V; e++) x[v * V + e] = i + e < a.n ? widen<T>(p[i + e]) : kNegInf;
            }
        }
    }
    // (fmaxf passes over NaN; a NaN reaches the sum through its difference)
    float lm = x[0];
#pragma unroll
    for (int e = 1; e < kPer; e++) lm = fmaxf(lm, x[e]);
    const float mx = max64(lm);
    const float ref = mx == kNegInf ? 0.f : mx;
    float r = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        // e^d as exp_of has it, but for the constant's second part, 2^-29 of p: to 2^-22, and to 2^-21 where 2048 of them weigh
        // less than 2^-19 (d < -21).  2^p alone is off by 2^-21 ln 2 at d = -5.6, to the same side for equal logits, and row
        // sums by 2.8e-7 (24 x 8 bf16 beams of 50257 20.4 us, so 21.1; with the second part 21.4).
        const float d = __builtin_elementwise_maximum(x[e] - ref, -1e30f);  // (-inf: its e^d is 0; NaN stays)
        const float p = d * 1.44269504088896340736f, ex = __builtin_amdgcn_exp2f(p);
        r += fmaf(ex, fmaf(p, -0x1.62e43p-1f, d), ex);
    }
    r = sum64(r);
    const int64_t at = rl * g.nseg + seg;
    if (lane == 0) g.stat[at] = BeamStat{mx, r};
    __shared__ uint64_t list[kBeamWaves][64];
    constexpr int BITS = std::is_same<T, Bf16>::value ? 16 : 24;
    if (!few) segment_candidates<V, BITS>(x, lm, base, a.keep, g.slots, lane, list[wv], g.cand + at * g.slots);
    else segment_candidates<1, BITS>(x, lm, base, a.keep, g.slots, lane, list[wv], g.cand + at * g.slots);
}

// larger values have larger ones (v is a number)
__device__ __forceinline__ uint64_t ord64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double unord64(uint64_t o) {
    return __longlong_as_double((long long)(o >> 63 ? o & 0x7FFFFFFFFFFFFFFFull : ~o));
}

__device__ __forceinline__ double sum64d(double v) {  // as sum64
    auto with = [&](auto &&f) {
        const uint64_t u = (uint64_t)__double_as_longlong(v);
        const uint32_t lo = f((uint32_t)u), hi = f((uint32_t)(u >> 32));
        v += __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
    };
    with([](uint32_t x) { return lane_of<0xB1>(x); });
    with([](uint32_t x) { return lane_of<0x4E>(x); });
    with([](uint32_t x) { return lane_of<0x141>(x); });
    with([](uint32_t x) { return lane_of<0x140>(x); });
    for (int o = 16; o < 64; o += o) v += __shfl_xor(v, o, 64);
    return v;
}

// a candidate: its value's order (0: none), its beam and its key (logit, then index)
struct Cand {
    uint64_t v, key;
    int beam;
};
__device__ __forceinline__ bool ahead(const Cand &x, const Cand &y) {
    return x.v > y.v || (x.v == y.v && (x.beam < y.beam || (x.beam == y.beam && x.key > y.key)));
}
__device__ __forceinline__ Cand shfl_cand(const Cand &c, int o) {
    return Cand{(uint64_t)__shfl_xor((unsigned long long)c.v, o, 64), (uint64_t)__shfl_xor((unsigned long long)c.key, o, 64),
                __shfl_xor(c.beam, o, 64)};
}

__global__ __launch_bounds__(kBeamThreads) void beam_join_kernel(BeamDev g) {
    constexpr int NW = kBeamThreads / 64;
    __shared__ double off[kBeams];   // score - log sum e^(l - maximum) (NaN: the beam offers nothing from its logits)
    __shared__ float top[kBeams];    // the maximum (taken off a logit before anything is added: both may be far from 0)
    __shared__ uint64_t ended[kBeams];  // the order of an ended beam's score (0: not ended)
    __shared__ uint64_t maxima[kBeamThreads], bound;
    __shared__ Cand list[kBeamList], part[NW];
    __shared__ uint32_t listed;
    const BeamArgs &a = g.a;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int64_t item = g.item0 + blockIdx.x;
    const BeamStat *stat = g.stat + (int64_t)blockIdx.x * a.beams * g.nseg;
    const uint64_t *cand = g.cand + (int64_t)blockIdx.x * a.beams * g.nseg * g.slots;
    const int64_t keys = g.nseg * g.slots;
    const double nan = __longlong_as_double(0x7FF8000000000000ll);
    // A beam's keys belong to `share` waves (beams over the number of waves: to one, which has several beams); a wave's
    // beams are first, first + step, ..  The first kHeld keys of a lane are loaded at once, before the sums that they
    // wait for (beams that were not read leave what the scratch held: not looked at).
    const int share = a.beams >= NW ? 1 : NW / a.beams, step = NW / share;
    const int first = wv / share, at0 = (wv % share) * 64 + lane;
    const int64_t pieces = keys / 2;  // of 16 bytes (nseg and slots are multiples of 4)
    auto load2 = [&](int b, int64_t at, uint64_t(&k)[2]) {
        const u32x4 v = at < pieces ? *reinterpret_cast<const u32x4 *>(cand + b * keys + 2 * at) : u32x4{0, 0, 0, 0};
        k[0] = (uint64_t)v[1] << 32 | v[0];
        k[1] = (uint64_t)v[3] << 32 | v[2];
    };
    uint64_t held[kHeld][2];
#pragma unroll
    for (int i = 0; i < kHeld; i++) load2(min(first, a.beams - 1), at0 + i * 64 * share, held[i]);
    if (tid == 0) listed = 0;
    for (int b = wv; b < a.beams; b += NW) {
        const float score = a.scores[item * a.beams + b];
        const uint8_t end = a.finished ? a.finished[item * a.beams + b] : 0;
        const BeamStat *st = stat + b * g.nseg;
        BeamStat q[kStats];  // (the first of a lane's segments stay)
#pragma unroll
        for (int i = 0; i < kStats; i++) q[i] = lane + 64 * i < g.nseg ? st[lane + 64 * i] : BeamStat{kNegInf, 0.f};
        const bool fin = finite_score(score);
        float mx = kNegInf;
        double o = nan;
        if (fin && !end) {
#pragma unroll
            for (int i = 0; i < kStats; i++) mx = fmaxf(mx, q[i].mx);
            for (int64_t i = lane + 64 * kStats; i < g.nseg; i += 64) mx = fmaxf(mx, st[i].mx);
            mx = max64(mx);
            double r = 0.0;
            auto add = [&](const BeamStat &t) { r = fma(exp((double)t.mx - (double)mx), (double)t.r, r); };
#pragma unroll
            for (int i = 0; i < kStats; i++) add(q[i]);
            for (int64_t i = lane + 64 * kStats; i < g.nseg; i += 64) add(st[i]);
            // (a row without a logit above -inf: mx = -inf)
            o = mx == kNegInf ? nan : (double)score - log(sum64d(r));
        }
        if (lane == 0) {
            off[b] = o;
            top[b] = mx;
            ended[b] = fin && end ? ord64((double)score) : 0;
        }
    }
    __syncthreads();

    auto value = [&](int b, uint64_t key) { return ord64(off[b] + ((double)unord((uint32_t)(key >> 32)) - (double)top[b])); };
    auto each = [&](int b, auto &&f) {  // the lane's keys of beam b (0: none)
        if (b == first) {
#pragma unroll
            for (int i = 0; i < kHeld; i++) f(held[i][0]), f(held[i][1]);
        }
        // (many at once: a workgroup's reads of a long list wait for one another otherwise)
        constexpr int N = 8;
        for (int64_t i = at0 + (b == first ? kHeld : 0) * 64 * share; i < pieces; i += N * 64 * share) {
            uint64_t k[N][2];
#pragma unroll
            for (int e = 0; e < N; e++) load2(b, i + e * 64 * share, k[e]);
#pragma unroll
            for (int e = 0; e < N; e++) f(k[e][0]), f(k[e][1]);
        }
    };
    // candidates of a value of at least `low`: within a beam they are the logits from some bound on, and only what is near
    // it needs its value
    auto from = [&](uint64_t low, auto &&f) {
        for (int b = first; b < a.beams; b += step) {
            if (off[b] != off[b]) continue;
            const double lv = unord64(low), at = lv - off[b] + (double)top[b];  // (NaN where low is no value's)
            const float near = (float)(at - 1e-6 * fabs(at) - 1e-9 * (fabs(lv) + fabs(off[b]) + fabs((double)top[b])));
            const uint32_t bound = near > -3e38f ? ord(near) : 0u;
            each(b, [&](uint64_t k) {
                if (k && (uint32_t)(k >> 32) >= bound) {
                    const uint64_t v = value(b, k);
                    if (v >= low) f(Cand{v, k, b});
                }
            });
        }
        if (tid < a.beams && ended[tid] && ended[tid] >= low) f(Cand{ended[tid], 1, tid});
    };
    uint64_t best = tid < a.beams ? ended[tid] : 0;
    for (int b = first; b < a.beams; b += step) {
        if (off[b] != off[b]) continue;
        uint64_t k = 0;
        each(b, [&](uint64_t x) { k = max(k, x); });
        if (k) best = max(best, value(b, k));
    }
    maxima[tid] = best;
    __syncthreads();
    if (wv == 0) {
        // The keep-th largest of the maxima of 64 parts is a lower bound of the keep-th largest value (its leading 24 bits).
        // A part takes another lane of every wave: of short rows only the first lanes hold candidates (2 x 15 beams of
        // 1621 with 30 kept 16 us, 61 with the same lane of all; 4 x 32 of 1000 with 32 21 and 170)
        uint64_t m = maxima[lane];
#pragma unroll
        for (int w = 1; w < NW; w++) m = max(m, maxima[64 * w + ((lane + 64 / NW * w) & 63)]);
        const uint32_t v = (uint32_t)(m >> 32);
        const uint32_t b = largest_with<24>(a.keep, [&](uint32_t k) { return __popcll(__ballot(v >= k)); });
        if (lane == 0) bound = max((uint64_t)b << 32, (uint64_t)1);
    }
    __syncthreads();
    const uint64_t low = bound;
    from(low, [&](const Cand &c) {
        const uint32_t at = atomicAdd(&listed, 1u);
        if (at < kBeamList) list[at] = c;
    });
    __syncthreads();
    auto put = [&](int place, const Cand &c) {
        const int64_t at = item * a.keep + place;
        a.out_scores[at] = c.v ? (float)unord64(c.v) : kNegInf;
        a.parents[at] = c.v ? c.beam : -1;
        a.tokens[at] = !c.v ? -1 : ended[c.beam] ? a.end_token : (int64_t)(0xFFFFFFFFu - (uint32_t)c.key);
    };
    const int got = (int)min(listed, (uint32_t)kBeamList);
    if (got <= 64) {  // as a rule: one wave, a candidate a lane
        if (wv) return;
        const Cand c = lane < got ? list[lane] : Cand{0, 0, kBeams};
        int place = 0;
        auto lane_u64 = [&](uint64_t v, int j) {
            return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, j);
        };
        for (int j = 0; j < got; j++) {
            const uint64_t v = lane_u64(c.v, j);
            place += v > c.v;
            if (__ballot(v == c.v) & ~(1ull << j)) {  // uniform
                const Cand o{v, lane_u64(c.key, j), __builtin_amdgcn_readlane(c.beam, j)};
                place += v == c.v && ahead(o, c);
            }
        }
        if (lane < got && place < a.keep) put(place, c);
        if (lane >= got && lane < a.keep) put(lane, Cand{0, 0, 0});
        return;
    }
    if (listed <= kBeamList) {
        for (int i = tid; i < got; i += kBeamThreads) {
            const Cand c = list[i];
            int place = 0;
            for (int j = 0; j < got; j++) place += ahead(list[j], c);
            if (place < a.keep) put(place, c);
        }
        if (tid >= got && tid < a.keep) put(tid, Cand{0, 0, 0});
        return;
    }
    // very many equal values: one place after another, the first of what is behind the last one
    Cand last{~0ull, ~0ull, -1};
    for (int place = 0; place < a.keep; place++) {
        Cand c{0, 0, kBeams};
        from(1, [&](const Cand &x) {
            if (ahead(last, x) && ahead(x, c)) c = x;
        });
        for (int s = 32; s > 0; s >>= 1) {
            const Cand o = shfl_cand(c, s);
            if (ahead(o, c)) c = o;
        }
        if (lane == 0) part[wv] = c;
        __syncthreads();
        c = part[0];
        for (int w = 1; w < NW; w++)
            if (ahead(part[w], c)) c = part[w];
        if (tid == 0) put(place, c);
        last = c;
        __syncthreads();  // (part is written again)
        if (!c.v) last = Cand{0, 0, kBeams};
    }
}

template <class T>
int launch_select(const BeamDev &g, int64_t items, void *stream) {
    hipLaunchKernelGGL(beam_seg_kernel<T>, dim3((unsigned)(g.nseg / kBeamWaves), (unsigned)(items * g.a.beams)), dim3(kBeamWaves * 64), 0,
                       (hipStream_t)stream, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)items), dim3(kBeamThreads), 0, (hipStream_t)stream, g);
    return (int)hipGetLastError();
}

// ---- states -----------------------------------------------------------------------------
// Bound: the bytes of the slots that move, written once, and of their parents, read once.  A thread takes one piece (up
// to 16 bytes) of all slots of an item: it reads the pieces of the parents of all slots that move before it writes any,
// so that the copy is in place whatever the parents are, and a parent of several slots comes from HBM once.
// Measured (MI355X): 787 MB of 4 beams 135 to 142 us, 5.6 TB/s; of more beams, all but one slot moving / half of them, each
// from a parent of its own: 8 beams 140 / 158, 16 beams 146 / 165, 32 beams 168 / 167; small ones: 1.8 MB of 6 beams 4.0, 9.7 MB of
// 32 beams 9.7 (19 workgroups a tensor, 16 loads a thread).
template <int N>
struct Bytes {
    typedef uint8_t type;
};
template <>
struct Bytes<2> {
    typedef uint16_t type;
};
template <>
struct Bytes<4> {
    typedef uint32_t type;
};
template <>
struct Bytes<8> {
    typedef u32x2 type;
};
template <>
struct Bytes<16> {
    typedef u32x4 type;
};

// PER: pieces of a thread at a time, two where a thread may have a single one to read and the card has many rounds of
// workgroups all the same (us, one / two: 0.6 MB in 76 workgroups of one 3.0 / 3.4; 105 MB in 6400 19.6 / 21.2; 210 MB in
// 12800 36.8 / 37.8; 787 MB in 48000 151 / 138; 480 MB of two slots in 59000 135 / 106, of four pieces 108).
template <int VEC, int MOST, int PER>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a) {
    typedef typename Bytes<VEC>::type T;
    __shared__ int from[MOST];
    __shared__ int moves;
    const int tid = threadIdx.x;
    if (tid == 0) moves = 0;
    __syncthreads();
    for (int64_t item = blockIdx.y; item < a.batch; item += gridDim.y) {
        if (tid < a.beams) {
            const int64_t p = a.parents[item * a.beams + tid];
            const bool move = p >= 0 && p < a.beams && p != tid;
            from[tid] = move ? (int)p : -1;
            if (move) moves = 1;
        }
        __syncthreads();
        if (moves) {
            int f[MOST];
#pragma unroll
            for (int j = 0; j < MOST; j++) f[j] = j < a.beams ? __builtin_amdgcn_readfirstlane(from[j]) : -1;
            uint8_t *base = a.state[blockIdx.z] + item * a.beams * a.slot_stride;
            auto place = [&](int64_t i) {  // of piece i (as a rule in 32 bits)
                int64_t at = 0;
                if (a.pieces <= 0xFFFFFFFFll) {
                    uint32_t left = (uint32_t)i;
#pragma unroll
                    for (int d = kReorderDims - 1; d >= 0; d--) {
                        if (a.size[d] == 1) continue;
                        const uint32_t q = left / (uint32_t)a.size[d];
                        at += (int64_t)(left - q * (uint32_t)a.size[d]) * a.stride[d];
                        left = q;
                    }
                } else {
                    int64_t left = i;
#pragma unroll
                    for (int d = kReorderDims - 1; d >= 0; d--) {
                        if (a.size[d] == 1) continue;
                        const int64_t q = left / a.size[d];
                        at += (left - q * a.size[d]) * a.stride[d];
                        left = q;
                    }
                }
                return base + at;
            };
            for (int64_t i = (int64_t)blockIdx.x * (256 * PER) + tid; i < a.pieces; i += (int64_t)gridDim.x * (256 * PER)) {
                uint8_t *p[PER];
                T v[PER][MOST];
#pragma unroll
                for (int e = 0; e < PER; e++) p[e] = i + e * 256 < a.pieces ? place(i + e * 256) : nullptr;
#pragma unroll
                for (int j = 0; j < MOST; j++)
                    if (f[j] >= 0)
#pragma unroll
                        for (int e = 0; e < PER; e++)
                            if (p[e]) v[e][j] = *reinterpret_cast<const T *>(p[e] + f[j] * a.slot_stride);
#pragma unroll
                for (int j = 0; j < MOST; j++)
                    if (f[j] >= 0)
#pragma unroll
                        for (int e = 0; e < PER; e++)
                            if (p[e]) __builtin_nontemporal_store(v[e][j], reinterpret_cast<T *>(p[e] + j * a.slot_stride));
            }
        }
        __syncthreads();
        if (tid == 0) moves = 0;
        __syncthreads();
    }
}

template <int VEC, int MOST, int PER>
int launch_reorder_as(const ReorderArgs &a, int tensors, void *stream) {
    const dim3 grid((unsigned)std::min<int64_t>((a.pieces + 256 * PER - 1) / (256 * PER), 65536), (unsigned)std::min<int64_t>(a.batch, 65535), (unsigned)tensors);
    hipLaunchKernelGGL((beam_reorder_kernel<VEC, MOST, PER>), grid, dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}
template <int VEC>
int launch_reorder(const ReorderArgs &a, int tensors, void *stream) {
    if (a.beams > 16) return launch_reorder_as<VEC, 32, 1>(a, tensors, stream);
    if (a.beams > 8) return launch_reorder_as<VEC, 16, 1>(a, tensors, stream);
    if (a.beams > 4) return launch_reorder_as<VEC, 8, 1>(a, tensors, stream);
    const double groups = (double)((a.pieces + 255) / 256) * (double)a.batch * tensors;
    return groups >= 24576 ? launch_reorder_as<VEC, 4, 2>(a, tensors, stream) : launch_reorder_as<VEC, 4, 1>(a, tensors, stream);
}

}  // namespace

int launch_beam_select(const BeamArgs &a, void *scratch, void *stream) {
    const BeamPlan p = beam_plan(a.batch, a.beams, a.n, a.keep);
    BeamDev g{};
    g.a = a;
    g.nseg = p.nseg;
    g.slots = p.slots;
    g.cand = reinterpret_cast<uint64_t *>(scratch);
    g.stat = reinterpret_cast<BeamStat *>(g.cand + (size_t)p.items * a.beams * p.nseg * p.slots);
    for (int64_t i = 0; i < a.batch; i += p.items) {
        g.item0 = i;
        const int64_t items = std::min(p.items, a.batch - i);
        const int e = a.dtype == NNQ_F32 ? launch_select<float>(g, items, stream)
                      : a.dtype == NNQ_BF16 ? launch_select<Bf16>(g, items, stream) : launch_select<F16>(g, items, stream);
        if (e) return e;
    }
    return 0;
}

int launch_beam_reorder(const ReorderArgs &a, int tensors, void *stream) {
    if (tensors < 1 || tensors > kReorderTensors || a.beams < 1 || a.beams > kBeams) return (int)hipErrorInvalidValue;
    switch (a.vec) {
    case 16: return launch_reorder<16>(a, tensors, stream);
    case 8: return launch_reorder<8>(a, tensors, stream);
    case 4: return launch_reorder<4>(a, tensors, stream);
    case 2: return launch_reorder<2>(a, tensors, stream);
    default: return launch_reorder<1>(a, tensors, stream);
    }
}

}  // namespace nnq
