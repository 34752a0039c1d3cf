// Host arithmetic of the C ABI's calls: the byte sizes of token arrays, the layout of a
// call's workspace regions, how long batches are cut into launches, and the rules that choose
// a kernel by sizes alone.  It is kept apart
// from nnq_abi.cpp (which makes the HIP runtime calls) so that the sanitizer harness
// (tests/sanitize) runs the same code on the CPU over ragged and extreme shapes.
#include <algorithm>
#include <cmath>

#include "nnq_internal.h"

namespace nnq {

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

bool array_bytes(int64_t rows, int64_t cols, size_t elem, size_t *out) {
    *out = 0;
    if (rows < 0 || cols < 0) return false;
    size_t a = 0;
    if (__builtin_mul_overflow((size_t)rows, (size_t)cols, &a)) return false;
    return !__builtin_mul_overflow(a, elem, out);
}

bool plan_regions(const size_t *sizes, int n, size_t *offsets, size_t *total) {
    size_t at = 0;
    for (int i = 0; i < n; i++) {
        offsets[i] = at;
        if (sizes[i] == 0) continue;  // an absent region takes no space
        // the next region starts at the 256-byte boundary after this one
        size_t end = 0;
        if (__builtin_add_overflow(at, sizes[i], &end) || end > SIZE_MAX - 255) return false;
        at = align256(end);
    }
    *total = at;
    return true;
}

int64_t moe_chunk_tokens(int64_t tokens, int top_k) {
    if (tokens <= 0 || top_k <= 0) return 0;
    return std::max<int64_t>(1, std::min<int64_t>(tokens, kMoeChunkAssign / top_k));
}

int64_t gemm_chunk_rows(int64_t m, int64_t k) {
    if (m <= 0 || k <= 0) return 0;
    // the GEMMs address an activation plane (and its f32 hi + lo pair) with 32-bit byte
    // offsets: 2 planes * rows * K * 2 bytes stays below 2^31
    const int64_t lim = ((int64_t)1 << 31) - 1;
    int64_t rows = lim / (4 * k);
    if (rows >= 256) rows = rows / 256 * 256;  // whole 256-row tiles per launch
    return std::min(m, std::max<int64_t>(1, rows));
}

// Parts of K in a 4-bit call of up to 16 rows.  Sixteen waves hold 32 units of x at a time (16 with f32
// planes); five rows and more of a longer K split it over workgroups, each of which converts its part of x
// once for all its tiles and leaves f32 slabs to one launch more (us, split / in passes: 12 bf16 rows of
// 4096 x 12288 17.4 / 19.8, 8192 x 8192 17.8 / 25.3, 6 f32 rows of 4096 x 12288 16.4 / 18.3).  Up to eight
// bf16 rows over no more tiles than CUs convert too little for that (5 rows of 4096 x 12288 13.7 / 12.6,
// 1024 x 8192 10.1 / 8.7; 8192 x 8192 13.6 / 16.8), and up to four rows have the next pass's x in flight.
int int4_rows_split(int64_t m, int64_t n, int64_t k, int x_bf16) {
    const int64_t held = (!x_bf16 && m > 8 ? 16 : 32) * kInt4Unit;
    if (m <= 4 || (x_bf16 && m <= 8 && n <= 256 * kTile)) return 1;
    return (int)std::min<int64_t>(8, (k + held - 1) / held);
}

size_t int4_rows_scratch(int64_t m, int64_t n, int64_t k, int x_bf16) {
    const int ks = int4_rows_split(m, n, k, x_bf16);
    return ks > 1 ? (size_t)ks * (size_t)m * (size_t)n * 4 : 0;
}

// Whether a 4-bit call of up to 16 rows takes the kernel for rows: always up to four; above, the shorter of
// two estimates (us, U units of 128 k, T 16-row tiles per CU), fitted on MI355X to 22 weights of 1024 to
// 151936 rows and K 512 to 12288 at 5 to 16 token rows.  The rows kernel's grows with the token rows, each of
// which it sums over its waves and stores apart (8 bf16 rows of 151936 x 1024 40 us, GEMM 25; x 4096 72 and
// 77; 16 f32 rows of 24576 x 4096 33 and 25, of 4096 x 4096 12 and 13.6).  The mean choice takes 1% more
// than the better one, the worst 22% (2 us).
bool int4_takes_rows(int64_t m, int64_t n, int64_t k, int x_bf16) {
    if (m <= 4 || m > kInt4Rows) return m <= 4;
    static const double rows[2][2][5] = {{{3.3, 0.085, 0.033, 0.083, 0.14}, {5.1, 0.051, 0.084, 0.062, 0.0}},
                                         {{3.0, 0.05, 0.037, 0.07, 0.2}, {2.5, 0.11, 0.007, 0.105, 0.7}}};
    static const double gemm[2][3] = {{9.1, 0.05, 0.069}, {8.6, 0.044, 0.057}};
    const double units = (double)((k + kInt4Unit - 1) / kInt4Unit);
    const double tiles = std::max(1.0, (double)((n + kTile - 1) / kTile) / 256);
    const double *r = rows[x_bf16 ? 1 : 0][m > 8], *g = gemm[x_bf16 ? 1 : 0];
    return r[0] + r[1] * units + tiles * (r[2] * units + r[3] * (double)m + r[4]) <= g[0] + g[1] * units + g[2] * tiles * units;
}

// 4-bit prefill: the workgroup tile (mt x 32 rows, nt x 128 columns) and the K split of the least
// estimated time.  c workgroups on a CU take c * step + lag per unit of 128 k (fitted on MI355X to
// 20 to 1024 rows of 1024 to 40960 columns, K 1024 to 12288: the choice is within 6% of the best of
// all tiles and splits there, 10% where a call takes under 20 us); with K split the slabs are written
// and read back at 5.6 TB/s by one launch more.  2 x 2 is left out where its registers spill (f32 x,
// groups of 32).
Int4GemmPlan int4_gemm_plan(int64_t m, int64_t n, int64_t k, int group, int x_bf16) {
    Int4GemmPlan p{};
    const int64_t cus = 256, tiles = (m + 31) / 32, units = (k + kInt4Unit - 1) / kInt4Unit;
    static const double step[2][2][2] = {{{0.42, 0.74}, {0.80, 0}}, {{0.255, 0.47}, {0.41, 0.76}}};
    static const double lag[2][2][2] = {{{0.08, 0.01}, {0.00, 0}}, {{0.15, 0.09}, {0.05, 0.14}}};
    const int xb = x_bf16 ? 1 : 0;
    double best = 1e30;
    int64_t ks = 1;
    for (int mt = 1; mt <= 2; mt++)
        for (int nt = 1; nt <= 2; nt++) {
            if (mt == 2 && nt == 2 && (!xb || group == 32)) continue;
            for (int64_t s = 1; s <= 8 && (s == 1 || units / s >= 2); s++) {
                const int64_t wg = (tiles + mt - 1) / mt * ((n + 128 * nt - 1) / (128 * nt)) * s;
                const double c = wg > 4 * cus ? (double)wg / cus : (double)((wg + cus - 1) / cus);
                double us = (double)((units + s - 1) / s) * (c * step[xb][mt - 1][nt - 1] + lag[xb][mt - 1][nt - 1]);
                if (s > 1) us += 1.5 + (double)(2 * s) * (double)m * (double)n * 4 / 5.6e6;
                if (us < best) {
                    best = us;
                    p.mt = mt;
                    p.nt = nt;
                    ks = s;
                }
            }
        }
    p.row_blocks = (int)((tiles + p.mt - 1) / p.mt);
    p.col_blocks = (int)((n + 128 * p.nt - 1) / (128 * p.nt));
    p.ks = (int)ks;
    const size_t planes = x_bf16 ? 1 : 2;
    p.plane = (size_t)tiles * (size_t)units * 8192;
    p.rowback = p.plane * planes;
    p.slabs = align256(p.rowback + (size_t)tiles * 32 * 4);
    p.bytes = p.slabs + (ks > 1 ? (size_t)ks * (size_t)m * (size_t)n * 4 : 0);
    return p;
}

// launches of at most 2^30 bytes of staged x and 2^16 rows
int64_t int4_chunk_rows(int64_t m, int64_t k) {
    const int64_t rows = ((int64_t)1 << 30) / (4 * (k + kInt4Unit)) / 128 * 128;
    return std::min(m, std::max<int64_t>(128, std::min<int64_t>(rows, 65536)));
}

// ---- MXFP4 rows ----

// Up to 16 rows the kernel for rows, unless over eight rows and many tiles K would go over workgroups (us, rows / GEMM: 16
// bf16 rows of 4096 -> 24576 21.7 / 20.0, 16 f32 rows of 4096 -> 151936 184 / 111; 16 bf16 of 12288 -> 4096 14.5 / 16.8, 9 f32 of
// 1024 -> 24576 10.3 / 14.4).  Over 170 shapes of 9 to 16 rows, K of 1024 to 12288 and n of 4096 to 151936, this takes 0.2% more
// than the better of both in the mean for products of 4-bit operands (at most 5%), 5% for bf16 x (25%: 16 x 1024 -> 50304
// 12.6 / 10.1) and 7% for f32 x (48%: 12 x 1024 -> 151936 52 / 35, and the other way 31%: 9 x 4096 -> 8192 13.7 / 18.0).
bool mx_takes_rows(int64_t m, int64_t n, int64_t k, int x_kind) {
    return m <= 8 || (m <= kMxRows && (mx_tiles(n) <= 256 || mx_rows_plan(m, n, k, x_kind).ks == 1));
}

// LDS bytes of x of m rows and `pairs` pairs of units (XStage)
static int64_t mx_stage_bytes(int64_t m, int64_t pairs, int x_kind) {
    if (x_kind >= kMxQuantBf16) return m * (pairs * 128 + 16 + pairs * 8);
    return m * (x_kind == kMxF32 ? 3 : 1) * (pairs * 512 + 16);
}

// The most values of x that every workgroup quantizes for itself; beyond, a launch before costs less.  us, in the call /
// before, -> 4096: bf16 rows 4 x 8192 8.4 / 10.1, 8 x 8192 9.9 / 11.2, 12 x 8192 11.4 / 11.7, 8 x 12288 12.4 / 13.1; 16 x 8192 12.4 /
// 12.0, 12 x 12288 14.4 / 13.8, 8 x 24576 21.0 / 20.4, 16 x 12288 16.1 / 14.5.  f32 rows 2 x 4096 6.3 / 7.1, 8 x 2048 6.9 / 7.0, 4 x
// 4096 7.6 / 8.2, 2 x 8192 8.9 / 9.8; 2 x 12288 12.0 / 12.1, 8 x 4096 10.1 / 8.7, 4 x 8192 11.7 / 10.6, 8 x 12288 21.1 / 12.8.
// (n of 16384 moves the change to half of that, n of 1024 hardly.)
constexpr int64_t kMxFirstBf16 = 98304, kMxFirstF32 = 16384;

// A wave along K for every two pairs of units (up to 16: three or four pairs), as many more along the tiles as make four
// waves, and as many workgroups on a CU as its 16 waves and its LDS hold; where x leaves room for one only, more waves
// along the tiles instead (their loads are what is in flight).  Swept on MI355X over 17 shapes of 1 to 16 rows (us, waves
// along K x tiles): 1 x 4096 -> 4096 5.5 (8 x 1), 7.0 (16 x 1), 5.9 (4 x 1); 12 x 4096 -> 24576 16.0 (8 x 2), 16.5 (4 x 3),
// 20 (16 x 1); 1 x 512 -> 151936 11.9 (1 x 4), 25 (2 x 1).
MxRowsPlan mx_rows_plan(int64_t m, int64_t n, int64_t k, int x_kind) {
    MxRowsPlan p{};
    const int64_t all = mx_pairs(k), tiles = mx_tiles(n), cus = 256, cap = 163840;
    // K goes over workgroups where its x does not fit (one row: in chunks, without a second launch)
    int64_t ks = 1;
    while (m > 1 && ks < 8 && ks < all && mx_stage_bytes(m, (all + ks - 1) / ks, x_kind) + 2 * 16 * 1280 > cap) ks++;
    const int64_t part = (all + ks - 1) / ks, per_cu = (tiles * ks + cus - 1) / cus;  // tiles of a CU's part
    p.ks = (int)ks;
    p.kw = (int)std::min<int64_t>(16, (part + 1) / 2);
    p.pp = (int)std::min<int64_t>(4, (part + p.kw - 1) / p.kw);
    p.nw = (int)std::min<int64_t>(per_cu, std::max(1, 4 / p.kw));
    auto bytes = [&] { return 2 * (int64_t)p.kw * p.nw * 1280 + mx_stage_bytes(m, std::min<int64_t>(part, p.kw * p.pp), x_kind); };
    while (bytes() > cap && p.pp > 1) p.pp--;
    while (bytes() > cap && p.kw > 1) p.kw--;
    int64_t fit = std::min<int64_t>(16 / (p.kw * p.nw), cap / bytes());
    if (fit < 2 && per_cu > 1 && p.nw == 1 && p.kw <= 8) {
        const int64_t steps = (per_cu + 16 / p.kw - 1) / (16 / p.kw);
        p.nw = (int)((per_cu + steps - 1) / steps);
        while (bytes() > cap && p.nw > 1) p.nw--;
        fit = 1;
    }
    p.lds = (int)bytes();
    p.groups = (int)std::max<int64_t>(1, cus * std::max<int64_t>(1, fit) / ks);
    p.first = (x_kind == kMxQuantBf16 && m * k > kMxFirstBf16) || (x_kind == kMxQuantF32 && m * k > kMxFirstF32);
    p.slabs = p.first ? align256((size_t)m * (size_t)k / 2 + (size_t)m * (size_t)k / 32) : 0;
    p.bytes = p.slabs + (ks > 1 ? (size_t)ks * (size_t)m * (size_t)n * 4 : 0);
    return p;
}

// More rows: the workgroup tile (mt x 32 rows, nt x 128 columns) and the K split of the least estimated time.  c
// workgroups on a CU take c * step + lag for each stage of K (128 k, products of 4-bit operands 256), fitted on MI355X to 15
// shapes of 17 to 2048 rows with all tiles and splits: the choice takes 1% more than the best of them in the mean, 9% at
// most.  With K split the slabs are written and read back at 4 TB/s by one launch more.
MxGemmPlan mx_gemm_plan(int64_t m, int64_t n, int64_t k, int x_kind) {
    struct Tile {
        int mt, nt;
        double step, lag;
    };
    static const Tile four[] = {{1, 2, 0.274, 0.057}, {2, 2, 0.348, 0.068}, {2, 3, 0.493, 0.084}, {4, 2, 0.66, 0.0}};
    static const Tile bf16[] = {{1, 2, 0.306, 0.115}, {1, 3, 0.416, 0.184}, {2, 2, 0.445, 0.267}, {2, 3, 0.655, 0.358}};
    static const Tile f32[] = {{1, 2, 0.847, 0.316}, {1, 3, 1.198, 0.329}};  // (64 x 256: 2.12 a stage, two of 32 x 256 less)
    MxGemmPlan p{};
    const bool both = x_kind >= kMxQuantBf16;
    const Tile *tiles = both ? four : x_kind == kMxBf16 ? bf16 : f32;
    const int count = x_kind == kMxF32 ? 2 : 4;
    const int64_t cus = 256, rows = (m + 31) / 32, pairs = mx_pairs(k), stages = both ? pairs : mx_units(k);
    double best = 1e30;
    for (int i = 0; i < count; i++)
        for (int64_t s = 1; s <= 8 && (s == 1 || pairs / s >= 2); s++) {
            const Tile &t = tiles[i];
            const int64_t wg = (rows + t.mt - 1) / t.mt * ((n + 128 * t.nt - 1) / (128 * t.nt)) * s;
            const double c = wg > 4 * cus ? (double)wg / cus : (double)((wg + cus - 1) / cus);
            double us = (double)((stages + s - 1) / s) * (c * t.step + t.lag);
            if (s > 1) us += 2.5 + (double)(2 * s) * (double)m * (double)n * 4 / 4.1e6;
            if (us < best) {
                best = us;
                p.mt = t.mt;
                p.nt = t.nt;
                p.ks = (int)s;
            }
        }
    p.row_blocks = (int)((rows + p.mt - 1) / p.mt);
    p.col_blocks = (int)((n + 128 * p.nt - 1) / (128 * p.nt));
    const size_t x = both ? (size_t)(mx_tiles(m) * pairs) * kMxPair : x_kind == kMxF32 ? (size_t)m * (size_t)k * 6 : 0;
    p.slabs = align256(x);
    p.bytes = p.slabs + (p.ks > 1 ? (size_t)p.ks * (size_t)m * (size_t)n * 4 : 0);
    return p;
}

int nnq_rule_mx(int64_t m, int64_t n, int64_t k, int x_kind, int *f) {
    if (mx_takes_rows(m, n, k, x_kind)) {
        const MxRowsPlan p = mx_rows_plan(m, n, k, x_kind);
        f[0] = p.pp;
        f[1] = p.kw;
        f[2] = p.nw;
        f[3] = p.ks;
        return 1;
    }
    const MxGemmPlan p = mx_gemm_plan(m, n, k, x_kind);
    f[0] = p.mt;
    f[1] = p.nt;
    f[2] = p.ks;
    f[3] = (int)((x_kind >= kMxQuantBf16 ? mx_pairs(k) : mx_units(k)) / p.ks);
    return 0;
}

int nnq_rule_mx_x_offset(int row, int m, int k, int u, int col) { return mx_x_offset(row, m, k, u, col); }

// launches whose x the kernels reach with 32-bit offsets (three bf16 planes: 6 bytes a value), whole 128-row tiles
int64_t mx_chunk_rows(int64_t m, int64_t k) {
    const int64_t rows = ((int64_t)1 << 30) / (6 * (k + kMxUnit)) / 128 * 128;
    return std::min(m, std::max<int64_t>(128, std::min<int64_t>(rows, 65536)));
}

size_t mx_linear_scratch(int64_t m, int64_t n, int64_t k, int x_kind) {
    const int64_t mc = mx_chunk_rows(m, k), tail = m % mc;
    auto launch = [&](int64_t r) { return mx_takes_rows(r, n, k, x_kind) ? mx_rows_plan(r, n, k, x_kind).bytes : mx_gemm_plan(r, n, k, x_kind).bytes; };
    return std::max(launch(mc), tail ? launch(tail) : 0);
}

// ---- beam search ----

// Segments of 2048 logits, four waves to a workgroup; a launch's rows fit its grid and its scratch stays near 64 MiB.
BeamPlan beam_plan(int64_t batch, int beams, int64_t n, int keep) {
    BeamPlan p{};
    p.nseg = ((n + 2047) / 2048 + 3) / 4 * 4;
    p.slots = std::min(64, (keep + keep / 2 + 6 + 3) / 4 * 4);
    const int64_t per = beams * p.nseg * (8 + 8 * (int64_t)p.slots);
    p.items = std::max<int64_t>(1, std::min({batch, ((int64_t)64 << 20) / per, (int64_t)65535 / beams}));
    p.bytes = (size_t)(p.items * per);
    return p;
}

const char *reorder_geometry(int64_t slots, int64_t slot_stride, int ndim, const int64_t *sizes, const int64_t *strides,
                             int64_t elem, uintptr_t address_bits, ReorderArgs *out) {
    struct Dim {
        int64_t size, stride;
    };
    Dim d[16], all[17];
    int n = 0;
    out->pieces = 0;
    out->dims = 0;
    for (int i = 0; i < ndim; i++) {
        if (sizes[i] < 0 || strides[i] < 0) return "negative size or stride";
        if (sizes[i] == 0) return nullptr;  // (no pieces)
        if (sizes[i] > 1) d[n++] = Dim{sizes[i], strides[i] * elem};
    }
    std::sort(d, d + n, [](const Dim &a, const Dim &b) { return a.stride > b.stride; });
    // elements that lie apart: each stride covers what the smaller ones span
    for (int i = 0; i < n; i++) all[i] = d[i];
    all[n] = Dim{slots, slot_stride * elem};
    std::sort(all, all + n + 1, [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
    int64_t span = elem;
    for (int i = 0; i <= n; i++) {
        if (all[i].size <= 1) continue;
        if (all[i].stride < span) return "elements that overlap or interleave";
        if (__builtin_mul_overflow(all[i].stride, all[i].size - 1, &all[i].size) || __builtin_add_overflow(span, all[i].size, &span))
            return "a span beyond 2^63 bytes";
    }
    // dims that follow one another are one
    Dim c[17];
    int m = 0;
    c[m++] = Dim{elem, 1};  // bytes of an element, innermost
    for (int i = n - 1; i >= 0; i--) {
        if (d[i].stride == c[m - 1].size * c[m - 1].stride) c[m - 1].size *= d[i].size;
        else c[m++] = d[i];
    }
    if (m > kReorderDims) out->dims = -1;
    if (m > kReorderDims) return "more than 4 dimensions that do not follow one another";
    uintptr_t bits = address_bits | (uintptr_t)c[0].size | (uintptr_t)(slots > 1 ? slot_stride * elem : 0);
    for (int i = 1; i < m; i++) bits |= (uintptr_t)c[i].stride;
    out->vec = bits & 1 ? 1 : bits & 2 ? 2 : bits & 4 ? 4 : bits & 8 ? 8 : 16;
    out->slot_stride = slot_stride * elem;
    out->dims = m;
    out->pieces = 1;
    for (int i = 0; i < kReorderDims; i++) {
        out->size[i] = 1;
        out->stride[i] = 0;
    }
    for (int i = 0; i < m; i++) {  // innermost last
        out->size[kReorderDims - 1 - i] = i ? c[i].size : c[0].size / out->vec;
        out->stride[kReorderDims - 1 - i] = i ? c[i].stride : out->vec;
        out->pieces *= out->size[kReorderDims - 1 - i];
    }
    return nullptr;
}

// Rows of 2048-logit segments (one wave each, four to a workgroup; a row that does not start at a
// 16-byte address begins inside its first segment, by up to 16 / elem - 1 logits).  The candidate
// slots leave room over the 1.1 to 1.4 top that continuous logits fill.  A launch takes at most
// 65535 rows (its grid's second dimension) and its scratch stays near 64 MiB, whatever m.
LogprobPlan logprob_plan(int64_t m, int64_t n, int top, int elem) {
    LogprobPlan p{};
    const int64_t seg = (n + 16 / elem - 1 + 2047) / 2048;
    p.nseg = (seg + 3) / 4 * 4;
    p.slots = top ? std::min(64, (top + top / 2 + 6 + 3) / 4 * 4) : 0;
    const int64_t per = p.nseg * (20 + 8 * (int64_t)p.slots);
    p.rows = std::max<int64_t>(1, std::min({m, ((int64_t)64 << 20) / per, (int64_t)65535}));
    p.bytes = (size_t)(p.rows * per);
    return p;
}

// Chunks of at most 320 MiB of f32 logits (552 rows of 151936), as even as whole 64-row tiles of the
// GEMMs allow: every chunk reads the weight again, so a short last one costs almost as much as a full
// one (300 rows of 151936 x 4096 in 4 bits as 272 + 28: 618 us, in one 506).
int64_t head_chunk_rows(int64_t m, int64_t n) {
    const int64_t fit = ((int64_t)320 << 20) / (4 * n), tile = fit >= 64 ? 64 : 16;
    const int64_t most = std::max<int64_t>(tile, fit / tile * tile), chunks = (m + most - 1) / most;
    return std::min(m, ((m + chunks - 1) / chunks + tile - 1) / tile * tile);
}

// ---- dispatch rules ----------------------------------------------------------------

// The path of a linear call of m tokens, by measured crossovers on MI355X (us, x f32 / bf16):
//  - 1 and 2 tokens: one decode-GEMV pass;
//  - 3 to 16: the few-row GEMM (nnq_gemm_few.hip) from 5 tokens on (Q8_0 4096x4096, 12 tokens:
//    14.3 / 17.0 as passes / GEMM, 12.8 / 7.5 there; Q6_K 12288x4096, 8 tokens: 26.8 / 26.3 as
//    two passes, 14.0 / 12.1).  Below that a GEMV pass of 4 tokens has the shorter prologue
//    (Q6_K 4096x4096: 6.2 against 8.4 / 7.4), except over eight tiles per CU or more (3 f32 tokens,
//    pass against few rows: Q6_K 151936 x 4096 133 / 97, 40960 x 2048 19.9 / 17.6; Q8_0 40960 x 2048
//    19.0 / 16.8; Q4_K 40960 x 4096 29.2 / 24.5; under 2048 k the pass is faster, 40960 x 1024
//    11.3 / 12.1, 10.8 / 11.3 and 8.7 / 11.4, but its sums are the less exact ones, so that the
//    rule has no line there).  Q4_K with f32 x takes it from 7
//    tokens (4096x4096: 5 and 6 as two passes 8.6 and 9.0 against 9.1 and 9.3; 8: 10.5 against
//    9.6), from 5 with two tiles per CU (24576 rows: 30.0 against 19.3) or K over 8192 (6
//    tokens at 4096x12288: 19.0 against 17.2).  Q4_K with bf16 x keeps the thin GEMM, which
//    stages nothing, up to that many tiles (16 tokens: 12288x4096 10.0 against 13.0, 24576
//    rows 18.8 against 19.5, 60000 rows 45.2 against 37.6).  Over 8 tokens of Q6_K are two
//    launches there: four tiles per CU of one or two units leave them to the MFMA GEMM (16 bf16
//    tokens, GEMM against few rows: 65536 x 256 14.4 / 25.4, x 512 20.7 / 26.5, x 1024 33.9 / 29.4;
//    8192 x 512 13.7 / 11.3);
//  - other counts: the MFMA GEMM.
// 1 where the few-row GEMM takes the call.
int nnq_rule_few_rows(int fmt, int64_t ntile, int64_t k, int64_t m, int x_bf16) {
    if (m < 3 || m > 16 || k > ((int64_t)1 << 24) || ntile >= ((int64_t)1 << 31)) return 0;
    if (fmt == NNQ_FMT_Q6_K && m > 8 && ntile >= 1024 && k <= 512) return 0;
    if (ntile >= 2048) return 1;  // eight tiles per CU
    if (fmt != NNQ_FMT_Q4_K) return m > 4;
    if (x_bf16) return 0;
    return m > 6 || (m > 4 && (ntile >= 512 || k > 8192));
}

// Shapes the Q4_K ring kernel takes (N % 128 == 0; f32 activations run their staged hi and lo
// planes as two halves of the work, summed by the finalize):
// BM x BN tiles, BM the smallest of 32, 64, 128 holding M (128 beyond), BN 192 or 128
// (dividing N), K split 1, 2, 4, 8 or 16 ways (a divisor of the super-block count leaving
// at least 4 super-blocks per workgroup, 2 with BM < 128).  Of these, the plan with the
// least estimated time: rounds of workgroups (one resident per CU: the rings of the small
// row tiles are deepened to 6 stages, which LDS holds once) times stages per workgroup, a 128-wide
// stage at 0.8 of a 192-wide one, plus one stage for the split-K finalize.  (Assuming two
// resident workgroups with shallower rings measured 5-25% slower at M = 16 to 64.)
// Returns the K split, or 0 when the shape does not fit.
int nnq_rule_gemm_ring(int64_t m, int64_t ntile, int64_t nblk, int x_bf16, int *bn, int *bm) {
    if (m < 1 || nblk < 1) return 0;
    const int npl = x_bf16 ? 1 : 2;  // f32 activations: hi and lo planes, each a full pass
    const int rows = m <= 32 ? 32 : (m <= 64 ? 64 : 128);
    const int64_t ncols = ntile * 16, nrt = (m + rows - 1) / rows;
    const int min_sb = rows == 128 ? 4 : 2;
    double best_cost = 0.0;
    int best_bn = 0, best_ks = 0;
    for (int cand : {192, 128}) {
        if (ncols % cand) continue;
        for (int ks = 1; ks <= 16; ks *= 2) {
            if (nblk % ks || (ks > 1 && nblk / ks < min_sb)) continue;
            const int64_t rounds = (nrt * (ncols / cand) * ks * npl + 255) / 256;
            const double cost = (double)rounds * (double)(nblk / ks) * (cand == 192 ? 1.0 : 0.8) + (ks * npl > 1 ? 1.0 : 0.0);
            if (best_bn == 0 || cost < best_cost) {
                best_cost = cost;
                best_bn = cand;
                best_ks = ks;
            }
        }
    }
    if (best_bn == 0) return 0;
    if (bn) *bn = best_bn;
    if (bm) *bm = rows;
    return best_ks;
}

// The wide kernel's shape rules: more than 128 rows (below, half of a 256-row tile or more is
// padding: f32 x, 100 x 4096 x 12288 109 us against the ring's 51), whole 16-row weight tiles
// and a 16-byte aligned output (the epilogue writes 16-byte row chunks), K <= 4096 * 3 (the
// staging keeps the row in one workgroup's registers and its sub-block sums in LDS), and at
// least 128 workgroups.  Column tiles per workgroup (6, 4 or 8) and K split (1 to 8 equal parts
// of whole super-blocks) are the ones with the least estimated time: rounds of workgroups over
// the CUs, each 3 us and its super-blocks times the measured time of one (us, 6, 4 and 8 tiles: bf16 x
// 3.8, 3.0 and 5.0, f32 x 6.2, 5.2 and 7.8: more tiles read each A fragment less often), plus
// the slabs' write, read and launch.  With bf16 x a part of two super-blocks, whose prologue nothing
// hides, counts as 2.7 and each further part adds 1.8% (without the two: 400 x 2560 x 2560 in 8 tiles and
// K in five 27.9 us, in 4 tiles and K in two 25.0; 200 x 6144 x 2048 25.4 and 23.6; 129 x 8192 x 3072 28.7
// and 26.6).
// 512 rows of f32 x take 107 us at 12288 x 4096 (6 tiles; the ring kernel over two planes 153) and
// 115 at 4096 x 12288 (8 tiles, K in four; 4 tiles and K in two 134, ring 155), of bf16 x there 77
// (4 tiles 83); 203 rows of f32 x at 12288 x 4096 take 6 tiles and K in two (256 workgroups).
// With random x these rates are the chip's power limit for f16 products: a library f16 GEMM
// of 512 x 12288 x 4096 takes 58 us (44 with x = 0), this kernel 66 with its staging (60).
// With f32 x the ring kernel keeps what it does faster, above all K of a prime number of super-blocks,
// which cannot be split here (260 x 5376 x 11008 125 us there, 187 here; 384 x 4736 x 1792 34 and 39).
// Both sides' times are estimated with constants fitted to 288 calls of the ring and 713 of this
// kernel, 4% and 5% off in the mean: us, per million of x, per MB of slabs (the ring's two planes have
// one each), per round and per super-block of a round (the ring's 128-column tiles 0.8 of its wide ones).
// h_out: the call is an MLP's gate | up and wants h = silu(gate) * up, which this kernel writes itself
// where K is not split and the ring leaves to a launch of about 4 us (f32 forwards, ring / wide gate | up: 260
// tokens of 768 x 2048 49.5 / 44.4 us, 129 of 1792 x 4608 66.3 / 61.7; 129 of 2816 x 4096 72.0 / 78.8).
// Returns the column tiles per workgroup (0: the ring kernel takes the shape) and the K split.
int nnq_rule_gemm_wide(int64_t m, int64_t ntile, int64_t nblk, int x_bf16, int h_out, int *ks) {
    if (m <= 128 || nblk > 48) return 0;
    const int64_t nrt = (m + 255) / 256, n = ntile * 16;
    const int tiles[3] = {6, 4, 8};
    const float sb_us[2][3] = {{3.8f, 3.0f, 5.0f}, {6.2f, 5.2f, 7.8f}};
    const float y_mb = (float)(m * n) * 4.0e-6f;
    float best = 0.0f;
    int at = -1, best_ks = 0;
    for (int i = 0; i < 3; i++) {
        if (ntile % tiles[i]) continue;
        for (int split = 1; split <= 8; split++) {
            const int64_t wg = nrt * (ntile / tiles[i]) * split;
            if (wg < 128 || nblk % split || nblk / split < 2) continue;
            const float sb = x_bf16 ? std::max((float)(nblk / split), 2.7f) : (float)(nblk / split);
            float us = (float)((wg + 255) / 256) * (3.0f + sb * sb_us[x_bf16 ? 0 : 1][i]);
            if (split > 1) us += 3.0f + (float)(split + 1) * y_mb * 0.25f;
            if (x_bf16) us *= 1.0f + 0.018f * (float)(split - 1);
            if (at < 0 || us < best) {
                best = us;
                at = i;
                best_ks = split;
            }
        }
    }
    if (at < 0) return 0;
    int bn = 0;
    const int rks = x_bf16 ? 0 : nnq_rule_gemm_ring(m, ntile, nblk, 0, &bn, nullptr);
    if (rks) {
        const float x_m = (float)m * (float)(nblk * 256) * 1.0e-6f, f32_us[3] = {4.7f, 3.9f, 5.8f};
        const int64_t rounds = (nrt * (ntile / tiles[at]) * best_ks + 255) / 256;
        const int64_t rrounds = ((m + 127) / 128 * (n / bn) * rks * 2 + 255) / 256;
        const float slabs = best_ks > 1 ? 0.5f + 0.22f * (float)(best_ks + 1) * y_mb : 0.0f;
        const float wide = 7.1f + 1.37f * x_m + (float)rounds * (3.8f + (float)(nblk / best_ks) * f32_us[at]) + slabs;
        const float ring = 10.4f + 1.05f * x_m + 0.34f * (float)(2 * rks + 1) * y_mb +
                           3.15f * (float)(rrounds * (nblk / rks)) * (bn == 192 ? 1.0f : 0.8f);
        if (ring + (h_out && best_ks == 1 ? 4.0f : 0.0f) < wide) return 0;
    }
    if (ks) *ks = best_ks;
    return tiles[at];
}

// The wide Q6_K kernel's shape rules: bf16 activations, more than 128 rows, whole groups of 8 weight tiles, K up
// to 4096 * 3 (the activation staging), a 16-byte aligned output, and at least 192 workgroups, or
// 128 with 8 super-blocks each.  The K split (1 to 8 equal parts of two or more super-blocks) is
// the one with the least estimated time: rounds of workgroups over the CUs, each 3 us and 7.8 us
// per super-block, plus the slabs; where that is not below the block kernel's estimate, that
// kernel keeps the shape (1000 x 2048 x 2560: 57 us wide, 49 there; 274 x 19200 x 7168, whose
// second row tile is nearly all padding: 285 and 277).  A second 128-row tile of up to 32 rows
// costs the block kernel less than a full one, 12% in its estimate (256, 160 and 129 x 40960 x
// 1024: 88, 62 and 59 us, wide 69, 67 and 66; 129 x 9728 x 2560: 45.7, wide 47.9).  Measured (block kernel -> wide): 512 x
// 4096 x 12288 134 -> 105 us, 512 x 12288 x 4096 167 -> 123, 300 x 4096 x 4096 67 -> 49, 200 x
// 4096 x 12288 108 -> 66, 256 x 24576 x 1024 61 -> 42.
// Returns the K split (0: the block kernel takes the shape).
int nnq_rule_gemm_wide6(int64_t m, int64_t ntile, int64_t nblk) {
    if (m <= 128 || nblk > 48 || ntile % 8) return 0;
    const int64_t base = (m + 255) / 256 * (ntile / 8), n = ntile * 16;
    // the block kernel: 128-row tiles at about 350 TFLOP/s, its staging and slab sum 12 us
    float best = 12.0f + 2.0f * (float)((m + 127) / 128 * 128) * (float)n * (float)(nblk * 256) / 350.0e6f;
    if (m <= 160) best *= 0.88f;
    int ks = 0;
    for (int split = 1; split <= 8; split++) {
        const int64_t wg = base * split;
        if (nblk % split || wg < 128 || nblk / split < 2 || (wg < 192 && nblk / split < 8)) continue;
        const float slabs = split > 1 ? 3.0f + (float)(split + 1) * (float)(m * n) * 4.0f / 4.0e6f : 0.0f;
        const float us = (float)((wg + 255) / 256) * (3.0f + (float)(nblk / split) * 7.8f) + slabs;
        if (us < best) {
            best = us;
            ks = split;
        }
    }
    return ks;
}

// Whether a MoE layer's experts run as moe_few_kernel's items (up to kMoeFewT tokens and
// kMoeFewAssign assignments) rather than as moe_stream_kernel's workgroups.  The items' time grows
// with the passes of four rows over an expert's weights, expected here for even routing; the
// streams' hardly does (a pass of theirs is 64 rows), so there is a number of passes where they
// cross: 28 with bf16 x and 22.5 with f32 x (which the items split on each pass, the streams
// once) for 2880 x 2880 experts, 5 and 4.5 more with each halving of an expert (an item of a small
// one is mostly its fixed part).  Streams of over 32 experts are more workgroups than CUs, and over
// 96 column streams take a wave more than one each: both raise it.  Measured (us, streams / items,
// top 8): 32 experts of 2880 x 2880, 6 bf16 tokens 104 / 99, 12 108 / 123, 16 109 / 151, 4 f32 tokens
// 127 / 127, 16 132 / 238; 16 such experts, 10 bf16 tokens 100 / 96, 16 101 / 126; 32 of 2048 x 2048, 12
// bf16 tokens 94 / 90, 16 94 / 109; 64 of 1024 x 768, 16 f32 tokens 79 / 71.
int nnq_rule_moe_few(int64_t experts, int64_t hidden, int64_t inter, int64_t tokens, int top_k, int x_bf16) {
    if (tokens > kMoeFewT || tokens * top_k > kMoeFewAssign) return 0;
    // an expert's rows are binomial: P(n) from P(n - 1)
    const double p = (double)top_k / (double)experts;
    double passes = (double)((tokens + 3) / 4);
    if (p < 1.0) {
        double pn = std::pow(1.0 - p, (double)tokens);
        passes = 0.0;
        for (int64_t n = 1; n <= tokens; n++) {
            pn *= (double)(tokens - n + 1) / (double)n * p / (1.0 - p);
            passes += pn * (double)((n + 3) / 4);
        }
    }
    passes *= (double)experts;
    const double halvings = std::max(0.0, std::log2(2880.0 * 2880.0 / ((double)hidden * (double)inter)));
    const double cross = x_bf16 ? 28.0 + 5.0 * halvings : 22.5 + 4.5 * halvings;
    const int64_t sets = (experts + 31) / 32, rounds = (inter / 32 + 95) / 96 + (hidden / 32 + 95) / 96;
    return passes <= cross * (1.0 + 1.25 * (double)(sets - 1)) * 0.5 * (double)rounds;
}

}  // namespace nnq
