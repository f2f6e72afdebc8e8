// sampling.hip -- a token per row of logits from a given random number: temperature, top-k, top-p, min-p.
//
//   w_i = exp((x_i - M) / T), M the row's maximum; tokens in the order (x falling, index rising)
//   top-k: the first k.  top-p, S the sum of their w: those whose predecessors sum to less than p S.  min-p: w_i >= m.
//   the token: the first in order of index whose running sum of kept w exceeds u times the sum of all kept w
//
// Weights are whole multiples of 2^-43 (the largest is 1), added as 64-bit integers: sums do not depend on their order, so
// neither do results, and 2^20 of them stay inside 64 bits. A weight is off by 2^-44 then, of 2^20 of them the sum by 2^-24
// at the very worst and 2^-35 by chance; a token whose weight is below that is not drawn.
//
// Four launches; the host does not see the rules, so all four whatever they are:
//   sample_scan, chunks of 4096: maximum and minimum of each, and the maxima of each 64 values
//   sample_bins, pieces of 512 values per wave, by the row's rule:
//     top-k of up to 1024: the k-th largest of the maxima bounds the k-th largest value from below; the tokens above the
//       bound are listed (50 of 151936: about 55 tokens)
//     top-p (or a larger k) alone: weights (counts) by distance from the maximum, 2048 bins, in LDS and then by integer atomics
//     neither: there is no border, the pieces' weights are added up
//   sample_border: rows with bins only: the bins that hold the border; their tokens are listed, the weights in front of them
//     added up by piece (gathered in LDS first: of a wave's 64 values few are in front, and their exponentials are what costs)
//   sample_draw: one workgroup per row. A small top-k's tokens are sorted, cut, and sorted by index. Else the border is found
//     among the listed tokens by digits of (x, index), then the piece that u falls into, and the token in it. Where a list is too
//     short (each_listed), the row is read in its place.
// Why bins and lists, not a sort: a row is read three times whatever the rule, and nothing but the lists is ever ordered.
//
// Bound and measured (one MI355X; calls back to back, and each launch alone under a trace, where clocks are lower and launches do not
// follow each other closely: those do not add up to the call). Few rows: the launches, 2.6 us each, and the chain of steps in
// sample_draw (1 x 151936, top-p 0.9 with top-k 20 14.1 us, 50 14.5, 200 20.9, 1000 23.8, without a top-k 24.0; traced at 50: scan
// 3.2, bins 6.5, border 1.7, draw 6.1; 13 rows of 32001 with rules of their own 25 to 29; rows that fit a list are sorted whole, 500
// logits with a top-k of 50 18.9). Many rows: 64 x 151936 with top-p 56 us, 3 x 39 MB read; traced: scan 8.4 us (4.7 TB/s, a large
// copy's rate), bins 20.7 (40 vector instructions a logit, most of them of the 64-bit exponential; vector units busy 59%), border
// 18.5 (30, 52%), draw 10.9. Without a border 29, min-p alone 25, greedy 15.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"
#include "sample.hpp"

namespace llamd {
namespace {

typedef unsigned long long u64;

constexpr int THREADS = 256, EACH = 16, CHUNK = THREADS * EACH, DRAW = 1024, PIECE = 512;
constexpr int BINS = 2048, LIST = 2048, FEW = 1024, GROUP = 64, GROUPS = CHUNK / GROUP;
constexpr int MOST_CHUNKS = SAMPLE_MOST / CHUNK, MOST_PIECES = SAMPLE_MOST / PIECE;
static_assert(MOST_CHUNKS <= THREADS, "a thread per chunk");
constexpr double RANGE = 44.0;  // weights below 2^-44 are 0

enum Mode { GREEDY, WHOLE, SMALL, BINNED };  // the maximum alone; no border; a small top-k; top-p or a larger top-k

struct Extremes {
    float top, least;  // least: of the finite values
    int at;            // the maximum's first index
    int pad;
};
// Where the border lies.
struct Border {
    int k_bin;             // top-k's last token's bin; -1: there are fewer than k
    int lo, hi;            // the bins that may hold the last token kept; lo BINS, hi below: no border
    unsigned k_count;      // tokens in front of k_bin, and their weight
    u64 k_weight, weight;  // weight of the tokens in front of lo
    u64 total;             // of all; with k_bin >= 0, of the tokens up to its end
};
// NaN as -infinity (the greater of a NaN and a number is the number).
__device__ __forceinline__ float value(float x) { return fmaxf(x, -INFINITY); }

// A number's bits so that they rise with it, and back.
__device__ __forceinline__ uint32_t rising(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_rising(uint32_t r) { return __uint_as_float(r & 0x80000000u ? r ^ 0x80000000u : ~r); }

// Position in the order: x falling, then index rising. (-0 is 0.)
__device__ __forceinline__ u64 place(float x, uint32_t i) { return (u64)~rising(x + 0.0f) << 32 | i; }

// s g + c. (Left to the compiler, c is copied first, one move for each of the polynomial's steps: 64 x 151936 with top-p
// 59.8 us, so 56.6.)
__device__ __forceinline__ double step(double s, double g, double c) {
    double x;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(x) : "v"(s), "v"(g), "s"(c));
    return x;
}

// A row's rule.
struct Rule {
    double m, c;        // maximum, log2(e) / T
    double furthest;    // min-p's
    double p;
    float half, scale;  // half the maximum; bins per half a unit of x
    int k;              // 0: all
    Mode mode;

    bool infinite;      // the maximum is

    // Distance from the maximum in powers of two. INF: `infinite`, where only the maximum's equals are not infinitely far.
    template <bool INF> __device__ __forceinline__ double distance_as(float x) const {
        return INF ? (x == INFINITY ? 0.0 : INFINITY) : (m - (double)x) * c;
    }
    __device__ __forceinline__ double distance(float x) const { return infinite ? distance_as<true>(x) : distance_as<false>(x); }
    // 2^-y as a multiple of 2^-43, to the nearest; 0 for NaN (an infinite temperature, and a token ruled out)
    static __device__ __forceinline__ u64 weight(double y) {
        y = fmin(y, 64.0);
        constexpr double ROUND = 0x1.8p52;  // what is added to it is rounded to a whole number, which its low word then holds
        const double whole = ROUND - y, g = (whole - ROUND) + y;  // -rint(y); |g| <= 1/2
        // 2^(43 - g): the polynomial through 2^-g at the 11 Chebyshev points of [-1/2, 1/2], off by 2^-51 of it at most
        double s = step(0x1p43 * 0x1.e6063f7217bc6p-28, g, 0x1p43 * -0x1.b675bca4eeebbp-24);
        s = step(s, g, 0x1p43 * 0x1.62bfd47773353p-20);
        s = step(s, g, 0x1p43 * -0x1.ffcb54062e698p-17);
        s = step(s, g, 0x1p43 * 0x1.430913096fd9fp-13);
        s = step(s, g, 0x1p43 * -0x1.5d87fe9d7a584p-10);
        s = step(s, g, 0x1p43 * 0x1.3b2ab6fba1ddap-7);
        s = step(s, g, 0x1p43 * -0x1.c6b08d703ce49p-5);
        s = step(s, g, 0x1p43 * 0x1.ebfbdff82c598p-3);
        s = step(s, g, 0x1p43 * -0x1.62e42fefa3a19p-1);
        s = step(s, g, 0x1p43);
        // times 2^-rint(y), rounded to a whole number in the last places of 2^52
        const int exponent = __double2hiint(s) + (int)((unsigned)__double2loint(whole) << 20);
        const double w = __hiloint2double(exponent, __double2loint(s)) + 0x1p52;
        return (u64)__double_as_longlong(w) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ bool likely(double y) const { return y <= furthest; }
    // Rises as x falls; BINS and more: behind the bins. (Halves: the difference of any two numbers is finite.)
    template <bool INF> __device__ __forceinline__ int bin_as(float x) const {
        return INF ? (x == INFINITY ? 0 : BINS) : (int)fminf((half - 0.5f * x) * scale, (float)BINS);
    }
    __device__ __forceinline__ int bin(float x) const { return infinite ? bin_as<true>(x) : bin_as<false>(x); }
    // f<infinite>()
    template <class F> __device__ __forceinline__ void by_kind(F f) const {
        if (__builtin_amdgcn_readfirstlane(infinite)) f(std::true_type{});
        else f(std::false_type{});
    }
};

// A row's rule as far as it does not depend on the logits (sample_scan finds it while they are on their way; by every workgroup
// of sample_bins, the logarithms and divisions are a part of its vector instructions).
struct Wanted {
    double c, furthest, p, reach;  // reach: of the bins, in x
    int k;
    Mode mode;
};

// A row's scratch; behind it the maxima of its groups of 64 values.
struct alignas(16) Row {
    u64 weight[BINS];
    unsigned count[BINS];
    u64 sum[MOST_PIECES];  // of the kept weights of 512 values, or of those in front of the border's bins
    Border border;
    u64 far;               // weight of the tokens behind the bins
    unsigned listed;
    int best;              // the maximum's first index
    Rule rule;
    Wanted wanted;
    Extremes chunk[MOST_CHUNKS];
    uint2 list[LIST];      // (index, x's bits), in any order
};
struct Rows {
    char *base;
    size_t step;
    int chunks;
    __device__ __forceinline__ Row &row(int i) const { return *(Row *)(base + (size_t)i * step); }
    __device__ __forceinline__ float *maxima(int i) const { return (float *)(base + (size_t)i * step + sizeof(Row)); }
};

// What a row's rule is before its logits are seen.
__device__ __forceinline__ Wanted wanted_of(const SampleArgs &a, int number) {
    const SampleRule how = a.how[number];
    Wanted r;
    r.c = 1.4426950408889634074 / (double)how.temperature;
    r.furthest = how.min_p > 0.0f ? -log2((double)how.min_p) : INFINITY;  // (negative above 1: GREEDY)
    r.k = how.top_k > 0 && how.top_k < a.n ? how.top_k : 0;
    r.p = how.top_p < 1.0f ? fmax((double)how.top_p, 0.0) : 1.0;  // (NaN: all)
    // (a bound of the k-th largest needs k groups; a quarter more leaves it some choice. By list and by bins, 151936 logits, top-k
    // with top-p: 50 14.6 and 23.5 us, 600 22.4 and 24.0, 1000 24.5 and 23.8, in 64 rows 50 26.0 and 55.3, 1000 38.6 and 56.9)
    const bool few = r.k && r.k <= FEW && (a.n <= LIST || a.n / GROUP >= r.k + r.k / 4);
    // (no weight reaches a min-p above 1: the first token alone is kept, not all that are equal to it)
    r.mode = !(how.temperature > 0.0f) || how.min_p > 1.0f ? GREEDY : few ? SMALL : r.k || r.p < 1.0 ? BINNED : WHOLE;
    // How far the bins reach, in x: to the least value, or where weights end. Top-p alone: tokens beyond log2(n / (1 - p)) + 1
    // sum to less than half of (1 - p) S, S >= 1, and are not needed to reach p S.
    const double reach = r.k || r.p == 1.0 ? RANGE : fmin(RANGE, log2(a.n / (1.0 - r.p)) + 1.0);
    r.reach = reach / r.c;
    return r;
}

// The rule of a row from its chunks' extremes; `at`: the maximum's first index.
__device__ __forceinline__ Rule rule_of(const Row &row, int chunks, int &at) {
    constexpr int W = 4;  // waves that have chunks
    __shared__ float tops[W], leasts[W];
    __shared__ int places[W];
    const Wanted wanted = row.wanted;
    Extremes x = {-INFINITY, INFINITY, 0x7FFFFFFF, 0};
    if ((int)threadIdx.x < chunks) x = row.chunk[threadIdx.x];
    wave_argmax(x.top, x.at, -INFINITY);
    x.least = wave_reduce(x.least, INFINITY, [](float u, float v) { return fminf(u, v); });
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = x.top, leasts[threadIdx.x >> 6] = x.least, places[threadIdx.x >> 6] = x.at;
    __syncthreads();
    float top = tops[0], least = leasts[0];
    at = places[0];
#pragma unroll
    for (int w = 1; w < W; ++w) {
        argmax_step(top, at, tops[w], places[w]);
        least = fminf(least, leasts[w]);
    }
    Rule r;
    r.m = top;
    r.infinite = top == INFINITY;
    r.c = wanted.c;
    r.furthest = wanted.furthest;
    r.k = wanted.k;
    r.p = wanted.p;
    r.mode = top == -INFINITY ? GREEDY : wanted.mode;
    const double range = fmin(r.m - (double)least, wanted.reach);
    r.half = 0.5f * top;
    r.scale = range > 0.0 ? (float)fmin((2.0 * BINS - 1.0) / range, 3e38) : 0.0f;
    return r;
}

// EACH logits for each of T threads, those from `first` on. VEC: rows are 16-byte aligned.
template <bool VEC, int T, int EACH> struct Values {
    float v[EACH];
    int first, n;

    __device__ __forceinline__ void load(const float *x, int of_row, int from) {
        first = from;
        n = of_row;
        if (VEC && first + T * EACH <= n) {
#pragma unroll
            for (int j = 0; j < EACH / 4; ++j) *(float4 *)(v + 4 * j) = *(const float4 *)(x + index(4 * j));
        } else {
#pragma unroll
            for (int j = 0; j < EACH; ++j) v[j] = index(j) < n ? x[index(j)] : -INFINITY;
        }
    }
    __device__ __forceinline__ int index(int j) const {
        const int t = threadIdx.x % T;
        return first + (VEC ? (j / 4 * T + t) * 4 + j % 4 : j * T + t);
    }
    // f(x, index) for each; -infinity behind the row
    template <class F> __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int j = 0; j < EACH; ++j) f(value(v[j]), index(j));
    }
    // The same where NaN may be NaN: it has no weight, and lies behind the bins.
    template <class F> __device__ __forceinline__ void each_raw(F f) const {
#pragma unroll
        for (int j = 0; j < EACH; ++j) f(v[j], index(j));
    }
};

// Sums over the wave, lane by lane.
__device__ __forceinline__ unsigned wave_scan(unsigned x) { return (unsigned)wave_incl_sum_i((int)x); }
template <int CTRL, int ROWS> __device__ __forceinline__ u64 dpp64(u64 x) {
    return (u64)(unsigned)dpp<CTRL, ROWS, ROWS == 0xF>(0, (int)(x >> 32)) << 32 | (unsigned)dpp<CTRL, ROWS, ROWS == 0xF>(0, (int)x);
}
__device__ __forceinline__ u64 wave_scan(u64 x) {
    x += dpp64<DPP_ROW_SHR1, 0xF>(x);
    x += dpp64<DPP_ROW_SHR2, 0xF>(x);
    x += dpp64<DPP_ROW_SHR4, 0xF>(x);
    x += dpp64<DPP_ROW_SHR8, 0xF>(x);
    x += dpp64<DPP_BCAST15, 0xA>(x);
    x += dpp64<DPP_BCAST31, 0xC>(x);
    return x;
}
__device__ __forceinline__ u64 last_lane(u64 x) {
    return (u64)(unsigned)readlane63((int)(x >> 32)) << 32 | (unsigned)readlane63((int)x);
}

// Inclusive sums over the workgroup's T threads of a count and a weight, and the sums of all.
template <int T>
__device__ __forceinline__ void scan(unsigned &count, u64 &weight, unsigned &counts, u64 &weights) {
    constexpr int W = T / 64;
    __shared__ unsigned c[W];
    __shared__ u64 w[W];
    const int wave = threadIdx.x >> 6;
    count = wave_scan(count);
    weight = wave_scan(weight);
    __syncthreads();  // (what the scan before this one left is read)
    if ((threadIdx.x & 63) == 63) c[wave] = count, w[wave] = weight;
    __syncthreads();
    counts = 0;
    weights = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const unsigned ci = c[i];
        const u64 wi = w[i];
        if (i < wave) count += ci, weight += wi;
        counts += ci;
        weights += wi;
    }
}
template <int T> __device__ __forceinline__ void scan(u64 &weight, u64 &weights) {
    unsigned none = 0, all;
    scan<T>(none, weight, all, weights);
}

// blockIdx.x: a row's chunk.
template <bool VEC> __global__ __launch_bounds__(THREADS) void sample_scan(SampleArgs a, Rows rows) {
    __shared__ float tops[4], leasts[4];
    __shared__ int places[4];
    const int number = blockIdx.x / rows.chunks, chunk = blockIdx.x % rows.chunks;
    Row &row = rows.row(number);
    float top = -INFINITY, least = INFINITY;
    int at = 0x7FFFFFFF;
    Values<VEC, THREADS, EACH> c;
    c.load(a.logits + (size_t)number * a.ld, a.n, chunk * CHUNK);
    if (chunk == 0 && threadIdx.x == 0) row.wanted = wanted_of(a, number);
    c.each_raw([&](float v, int i) {  // (a thread's indices rise)
        if (v > top) top = v, at = i;
        least = fminf(least, v > -INFINITY ? v : INFINITY);
    });
    // what the next launches add to
    for (int i = chunk * THREADS + threadIdx.x; i < BINS; i += rows.chunks * THREADS) row.count[i] = 0, row.weight[i] = 0;
    if (chunk == 0 && threadIdx.x == 0) row.far = 0, row.listed = 0;
    float group = fmaxf(top, dpp<DPP_XOR1>(top, top));
    group = fmaxf(group, dpp<DPP_XOR2>(group, group));
    if (threadIdx.x % 4 == 0) rows.maxima(number)[chunk * GROUPS + threadIdx.x / 4] = group;
    wave_argmax(top, at, -INFINITY);
    least = wave_reduce(least, INFINITY, [](float u, float v) { return fminf(u, v); });
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top, leasts[threadIdx.x >> 6] = least, places[threadIdx.x >> 6] = at;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) argmax_step(top, at, tops[w], places[w]), least = fminf(least, leasts[w]);
        row.chunk[chunk] = {top, least, at, 0};
    }
}

// A row's maxima of groups, as many as a wave holds: four groups in a number. HELD: 163840 logits; of more, every round of bound_of
// reads the others again, but registers for more cost every row (top-k 50 with top-p, 10 and 16 of them: 1 x 151936 14.4 and 15.0 us,
// 201088 17.6 and 15.1, 262144 20.6 and 15.1; 64 rows 26.0 and 32.2, 34.8 and 36.2, 41.4 and 38.6).
struct Maxima {
    static constexpr int HELD = 10;
    float4 v[HELD];
    const float4 *from;
    int n;  // fours

    __device__ __forceinline__ void load(const float *maxima, int groups) {
        from = (const float4 *)maxima;
        n = groups / 4;
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int at = (threadIdx.x & 63) + 64 * i;
            v[i] = at < n ? from[at] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
    }
};

// A bound that k groups' maxima, and so k tokens, reach: as few more as a short search finds. Four bounds are counted at a
// time, one by each wave. 0: there are fewer than k, or more tokens
// would reach it than a list holds.
__device__ __forceinline__ uint32_t bound_of(const Maxima &m, float top, int k) {
    __shared__ int counts[4];
    constexpr int HELD = Maxima::HELD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, enough = k + k / 4;
    const bool fours = m.n >= enough;  // maxima of four groups where these are still enough
    const uint32_t none = rising(-INFINITY);
    uint32_t one[HELD], four[HELD][4], least = ~0u;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const float4 v = m.v[i];
        four[i][0] = rising(v.x), four[i][1] = rising(v.y), four[i][2] = rising(v.z), four[i][3] = rising(v.w);
        one[i] = max(max(four[i][0], four[i][1]), max(four[i][2], four[i][3]));
        least = min(least, one[i] > none ? one[i] : ~0u);
    }
    const auto count_of = [&](uint32_t at) {
        int count = 0;
        if (fours) {
#pragma unroll
            for (int i = 0; i < HELD; ++i) count += __popcll(__ballot(one[i] >= at));
        } else {
#pragma unroll
            for (int i = 0; i < HELD; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) count += __popcll(__ballot(four[i][j] >= at));
        }
        for (int i = lane + 64 * HELD; i < m.n + lane; i += 64) {  // (those that are not held)
            const float4 v = m.from[min(i, m.n - 1)];
            const bool x = rising(v.x) >= at, y = rising(v.y) >= at, z = rising(v.z) >= at, w = rising(v.w) >= at, in = i < m.n;
            if (fours) {
                count += __popcll(__ballot(in && (x || y || z || w)));
            } else {
                count += __popcll(__ballot(in && x)) + __popcll(__ballot(in && y)) + __popcll(__ballot(in && z)) +
                         __popcll(__ballot(in && w));
            }
        }
        return count;
    };
    // from the least finite maximum: it is reached by so many of them
    uint32_t lo = (uint32_t)wave_reduce((int)(least ^ 0x80000000u), 0x7FFFFFFF, [](int x, int y) { return min(x, y); }) ^ 0x80000000u;
    uint32_t hi = rising(top) + 1;  // count(lo) >= k, count(hi) < k
    int best = count_of(lo);
    if (best < k) {  // (there may be less ones)
        lo = none + 1;
        best = count_of(lo);
        if (best < k) return 0;
    }
    while (best > enough && hi - lo > 1) {
        const uint32_t step = (hi - lo) / 5 + 1;
        const int mine = count_of(min(lo + (wave + 1) * step, hi));
        __syncthreads();  // (what the round before left is read)
        if (lane == 0) counts[wave] = mine;
        __syncthreads();
        int reached = 0;  // bounds that k reach
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int c = counts[w];
            if (c >= k) reached = w + 1, best = c;
        }
        const uint32_t was = lo;
        if (reached) lo = min(was + reached * step, hi);
        if (reached < 4) hi = min(was + (reached + 1) * step, hi);
    }
    // How many tokens reach it: of `all` groups of tokens that are alike, `best` with one at least, -all log(1 - best / all).
    // (Up to a sixteenth of the list's length fit even if no group is without one, all log(all) then.)
    if (best > LIST / 16) {
        const int all = count_of(none + 1);
        if (best >= all || all * -log1pf(-(float)best / (float)all) > 0.9f * LIST) return 0;
    }
    return lo;
}

// f(values, piece) for this wave's pieces of a row: every `waves`-th from `wave` on, the next one on its way.
template <bool VEC> using Piece = Values<VEC, 64, PIECE / 64>;
template <bool VEC, class F>
__device__ __forceinline__ void each_piece(Piece<VEC> &now, const float *x, int n, int wave, int waves, F f) {
    const int pieces = (n + PIECE - 1) / PIECE;
#pragma unroll 1
    for (int piece = wave; piece < pieces; piece += waves) {
        Piece<VEC> next;
        next.load(x, n, min(piece + waves, pieces - 1) * PIECE);
        f(now, piece);
        now = next;
    }
}

// blockIdx.x: one of a row's `parts` workgroups.
template <bool VEC> __global__ __launch_bounds__(THREADS) void sample_bins(SampleArgs a, Rows rows, int parts) {
    __shared__ union {
        struct { unsigned count[BINS]; u64 weight[BINS]; } bins;
        uint2 list[LIST];
    } lds;
    __shared__ unsigned listed, first;
    const int number = blockIdx.x / parts, part = blockIdx.x % parts;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(part * (THREADS / 64) + (threadIdx.x >> 6));
    const int waves = parts * (THREADS / 64);
    Row &row = rows.row(number);
    const float *x = a.logits + (size_t)number * a.ld;
    // (on their way while the rule is made)
    Piece<VEC> c;
    c.load(x, a.n, wave * PIECE);
    Maxima maxima;
    const int k = a.how[number].top_k;
    if (k > 0 && k <= FEW) maxima.load(rows.maxima(number), rows.chunks * GROUPS);
    int at;
    Rule r = rule_of(row, rows.chunks, at);
    uint32_t bound = 0;
    if (r.mode == SMALL && a.n > LIST) {
        bound = bound_of(maxima, (float)r.m, r.k);
        // (all workgroups of the row alike; a list that is too short would have sample_draw read the row instead: 16 x 80383, a third
        // masked, top-k 1000, 38 us, so 276; the estimate costs other rows 0.3 to 0.8)
        if (!bound) r.mode = BINNED;
    }
    if (part == 0 && threadIdx.x == 0) row.rule = r, row.best = at;
    if (r.mode == GREEDY) return;
    if (r.mode == WHOLE) {
        each_piece<VEC>(c, x, a.n, wave, waves, [&](const Piece<VEC> &c, int piece) {
            u64 sum = 0;
            r.by_kind([&](auto inf) {
                c.each_raw([&](float v, int) {
                    const double y = r.template distance_as<inf>(v);
                    sum += r.likely(y) ? r.weight(y) : 0;
                });
            });
            sum = last_lane(wave_scan(sum));
            if (lane == 0) row.sum[piece] = sum;
        });
        return;
    }
    if (r.mode == SMALL) {
        if (threadIdx.x == 0) listed = 0;
        const float least = bound ? of_rising(bound) : -INFINITY;
        __syncthreads();
        each_piece<VEC>(c, x, a.n, wave, waves, [&](const Piece<VEC> &c, int) {
            c.each([&](float v, int i) {
                if (v >= least && v > -INFINITY) {
                    const unsigned to = atomicAdd(&listed, 1u);
                    if (to < LIST) lds.list[to] = make_uint2(i, __float_as_uint(v));
                }
            });
        });
        __syncthreads();
        if (threadIdx.x == 0) first = listed ? atomicAdd(&row.listed, listed) : 0;
        __syncthreads();
        for (unsigned i = threadIdx.x; i < min(listed, (unsigned)LIST); i += THREADS)
            if (first + i < LIST) row.list[first + i] = lds.list[i];
        return;
    }
    for (int i = threadIdx.x; i < BINS; i += THREADS) lds.bins.count[i] = 0, lds.bins.weight[i] = 0;
    __syncthreads();
    u64 far = 0;
    each_piece<VEC>(c, x, a.n, wave, waves, [&](const Piece<VEC> &c, int) {
        r.by_kind([&](auto inf) {
            c.each_raw([&](float v, int) {
                const u64 w = r.weight(r.template distance_as<inf>(v));
                const int b = r.template bin_as<inf>(v);
                if (b >= BINS) {
                    far += w;
                } else if (w) {
                    if (r.k) atomicAdd(&lds.bins.count[b], 1u);
                    atomicAdd(&lds.bins.weight[b], w);
                }
            });
        });
    });
    far = last_lane(wave_scan(far));
    if (lane == 0 && far) atomicAdd(&row.far, far);
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += THREADS)
        if (lds.bins.weight[i]) {
            if (r.k) atomicAdd(&row.count[i], lds.bins.count[i]);
            atomicAdd(&row.weight[i], lds.bins.weight[i]);
        }
}

constexpr int PER = BINS / THREADS;
__device__ __forceinline__ Border border_of(const Row &row, const Rule &r, const unsigned (&count)[PER], const u64 (&weight)[PER]) {
    __shared__ Border found;
    unsigned c = 0, all;
    u64 w = 0, total;
#pragma unroll
    for (int i = 0; i < PER; ++i) c += count[i], w += weight[i];
    const unsigned mine_c = c;
    const u64 mine_w = w;
    scan<THREADS>(c, w, all, total);
    c -= mine_c;
    w -= mine_w;
    if (threadIdx.x == 0) found = {-1, BINS, BINS - 1, 0, 0, 0, total + row.far};
    __syncthreads();
    if (r.k && all >= (unsigned)r.k) {
        u64 in_front = w;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (c < (unsigned)r.k && c + count[i] >= (unsigned)r.k) {
                found.k_bin = found.lo = found.hi = threadIdx.x * PER + i;
                found.k_count = c;
                found.k_weight = found.weight = in_front;
                found.total = in_front + weight[i];
            }
            c += count[i];
            in_front += weight[i];
        }
        __syncthreads();
    }
    if (r.p < 1.0) {
        // the sum that p is a share of lies between these
        const double least = r.p * (double)(found.k_bin < 0 ? found.total : found.k_weight), most = r.p * (double)found.total;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const u64 with = w + weight[i];
            const bool first = threadIdx.x == 0 && i == 0;
            if ((first || (double)w < least) && (double)with >= least) found.lo = threadIdx.x * PER + i, found.weight = w;
            if ((first || (double)w < most) && (double)with >= most) found.hi = threadIdx.x * PER + i;
            w = with;
        }
        __syncthreads();
    }
    return found;
}

// blockIdx.x: one of a row's `parts` workgroups.
template <bool VEC> __global__ __launch_bounds__(THREADS) void sample_border(SampleArgs a, Rows rows, int parts) {
    __shared__ unsigned listed, first;
    __shared__ uint2 list[LIST];
    __shared__ float queues[THREADS / 64][PIECE];
    const int number = blockIdx.x / parts, part = blockIdx.x % parts;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(part * (THREADS / 64) + (threadIdx.x >> 6));
    const int waves = parts * (THREADS / 64);
    Row &row = rows.row(number);
    if (row.rule.mode != BINNED) return;
    const float *x = a.logits + (size_t)number * a.ld;
    unsigned count[PER];
    u64 weight[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) count[i] = row.count[threadIdx.x * PER + i], weight[i] = row.weight[threadIdx.x * PER + i];
    Piece<VEC> c;
    c.load(x, a.n, wave * PIECE);
    const Rule r = row.rule;
    const Border b = border_of(row, r, count, weight);
    if (part == 0 && threadIdx.x == 0) row.border = b;
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    float *queue = queues[threadIdx.x >> 6];
    each_piece<VEC>(c, x, a.n, wave, waves, [&](const Piece<VEC> &c, int piece) {
        // the values in front of the border, close together: few of a wave's 64 are, and their weights are what costs
        int queued = 0;
        r.by_kind([&](auto inf) {
            c.each_raw([&](float v, int i) {
                const int bin = r.template bin_as<inf>(v);
                const unsigned long long in_front = __ballot(bin < b.lo);
                const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(in_front >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in_front, 0));
                if (bin < b.lo) queue[queued + before] = v;
                queued += __popcll(in_front);
                if (bin >= b.lo && (bin <= b.hi || bin == b.k_bin)) {
                    const unsigned to = atomicAdd(&listed, 1u);
                    if (to < LIST) list[to] = make_uint2(i, __float_as_uint(v));
                }
            });
        });
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        u64 sum = 0;
        for (int i = lane; i < queued; i += 64) {
            const double y = r.distance(queue[i]);
            if (r.likely(y)) sum += r.weight(y);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        if (queued) sum = last_lane(wave_scan(sum));
        if (lane == 0) row.sum[piece] = sum;
    });
    __syncthreads();
    if (threadIdx.x == 0) first = listed ? atomicAdd(&row.listed, listed) : 0;
    __syncthreads();
    for (unsigned i = threadIdx.x; i < min(listed, (unsigned)LIST); i += THREADS)
        if (first + i < LIST) row.list[first + i] = list[i];
}

// ---- the last launch: one workgroup of 1024 per row ---------------------------------------

// Tokens of the border's bins.
struct Listed {
    u64 at[LIST], weight[LIST];
    uint16_t bin[LIST];
    unsigned n;
};

// f(place, weight) for those of bins [lo, hi]: from the list, or where that is too short, from the row (then from all tokens). It is
// where the border's bins hold more than 2048 tokens: few different values, as 16-bit logits far from 0 have. One workgroup reads
// the row then, once for each digit: 151936 16-bit logits around 24, 0.125 apart, spread 2.5, temperature 1.4, top-p 0.9: 236 us, 64
// rows 398 (f32 logits alike 24 and 57; at temperature 1 the border lies among fewer: 42 and 69); all logits equal 660 to 830.
template <class F>
__device__ __forceinline__ void each_listed(const Listed &list, const Rule &r, const float *x, int n, int lo, int hi, F f) {
    if (list.n <= LIST) {
        for (unsigned i = threadIdx.x; i < list.n; i += DRAW)
            if (list.bin[i] >= lo && list.bin[i] <= hi) f(list.at[i], list.weight[i]);
    } else {
        for (int i = threadIdx.x; i < n; i += DRAW) {
            const float v = value(x[i]);
            const int bin = r.bin(v);
            if (bin < lo || bin > hi) continue;
            const u64 w = r.weight(r.distance(v));
            if (w) f(place(v, i), w);
        }
    }
}

// The place of the first token of bins [lo, hi] with which it is done(tokens up to it, their weight), counted from `count` and
// `weight`; `weight` becomes that weight. By digits of 8 bits of the place, from the highest that differs.
template <class Done>
__device__ __forceinline__ u64 last_place(const Listed &list, const Rule &r, const float *x, int n, int lo, int hi,
                                          unsigned count, u64 &weight, Done done) {
    __shared__ unsigned counts[256];
    __shared__ u64 weights[256], highest[256], least, most;
    __shared__ struct { unsigned digit, count, here; u64 weight, mine; } next;
    if (threadIdx.x == 0) least = ~0ull, most = 0, next = {0, count, 1, weight, 0};  // (a digit is always found)
    __syncthreads();
    u64 a = ~0ull, b = 0;
    each_listed(list, r, x, n, lo, hi, [&](u64 at, u64) { a = min(a, at), b = max(b, at); });
    if (b) atomicMin(&least, a), atomicMax(&most, b);
    __syncthreads();
    const u64 differ = least ^ most;
    u64 prefix = most;
    int shift = differ ? max(56 - (int)__builtin_clzll(differ), 0) : 0, known = shift + 8;  // bits of the prefix that are known
    for (;;) {
        if (threadIdx.x < 256) counts[threadIdx.x] = 0, weights[threadIdx.x] = 0, highest[threadIdx.x] = 0;
        __syncthreads();
        each_listed(list, r, x, n, lo, hi, [&](u64 at, u64 w) {
            if (known < 64 && (at ^ prefix) >> known) return;
            const int digit = at >> shift & 255;
            atomicAdd(&counts[digit], 1u);
            atomicAdd(&weights[digit], w);
            atomicMax(&highest[digit], at);
        });
        __syncthreads();
        // the first digit with which it is done; if rounding leaves none, the last that there is
        if (threadIdx.x < 64) {
            unsigned c[4], cs = 0;
            u64 w[4], ws = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) cs += c[i] = counts[4 * threadIdx.x + i], ws += w[i] = weights[4 * threadIdx.x + i];
            unsigned before = wave_scan(cs);
            const unsigned all = (unsigned)readlane63((int)before);
            u64 in_front = wave_scan(ws) - ws;
            before -= cs;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned upto = before + c[i];
                const bool is = done(count + upto, weight + in_front + w[i]);
                const bool was = before && done(count + before, weight + in_front);
                if (c[i] && !was && (is || upto == all))
                    next = {4 * threadIdx.x + i, count + before, c[i], weight + in_front, w[i]};
                before = upto;
                in_front += w[i];
            }
        }
        __syncthreads();
        count = next.count;
        weight = next.weight;
        prefix = highest[next.digit];
        if (next.here == 1 || shift == 0) {
            weight += next.mine;
            return prefix;
        }
        known = shift;
        shift = max(shift - 8, 0);
        __syncthreads();
    }
}

// The running sum that the token's exceeds: u times all, at most all but one.
__device__ __forceinline__ u64 target_of(double u, u64 total) {
    const double want = u * (double)total;
    return want > 0.0 ? (want < (double)total ? min((u64)want, total - 1) : total - 1) : u == u ? 0 : total - 1;
}

// The token drawn: one per thread that may be, `before` the kept weights in front of it.
__device__ __forceinline__ void drawn(const SampleArgs &a, int number, u64 target, u64 before, u64 w, u64 total, int at) {
    if (before <= target && before + w > target) {
        a.ids[number] = at;
        if (a.prob) a.prob[number] = (float)((double)w / (double)total);
    }
}

// Listed tokens in order, by bins of their bits: a token's place is its bin's beginning and those in front of it in the bin.
// CROWD: tokens of a cell from which on it is done by digits (last_place) instead. By cells and by digits: top-p alone, 1 row 25.3 and
// 27.1 us, 64 rows 55.8 and 61.2, top-k 1000 24.5 and 45.0; 64 rows of 16-bit logits, whose border's cell holds hundreds of equal
// ones: with this limit 66.7, with a limit of 1024 78.4, always by digits 66.9.
constexpr int CELLS = 2048, PER_CELL = CELLS / DRAW, CROWD = 64;
struct Ordered {
    unsigned begin[CELLS + 1];  // the cells' first tokens
    u64 weight[CELLS];          // the weight in front of them
    u64 at[LIST], own[LIST];    // places and weights, cell by cell
    unsigned least, most, crowd;
};
constexpr int HELD = LIST / DRAW;
struct Token {
    u64 at, w;        // place and weight; at ~0: none
    unsigned before;  // listed tokens in front of it, and their weight
    u64 weight;
};
// False: a cell has so many (equal logits) that this would take longer than last_place.
__device__ __forceinline__ bool order(Ordered &o, Token (&t)[HELD]) {
    unsigned least = ~0u, most = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (t[i].at != ~0ull) {
            least = min(least, (unsigned)(t[i].at >> 32));
            most = max(most, (unsigned)(t[i].at >> 32));
        }
    least = ~(unsigned)wave_reduce((int)(~least ^ 0x80000000u), (int)0x80000000, [](int x, int y) { return max(x, y); }) ^ 0x80000000u;
    most = (unsigned)wave_reduce((int)(most ^ 0x80000000u), (int)0x80000000, [](int x, int y) { return max(x, y); }) ^ 0x80000000u;
    if (threadIdx.x == 0) o.least = ~0u, o.most = 0, o.crowd = 0;
    for (int i = threadIdx.x; i < CELLS; i += DRAW) o.begin[i] = 0, o.weight[i] = 0;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) atomicMin(&o.least, least), atomicMax(&o.most, most);
    __syncthreads();
    least = o.least;
    const unsigned range = o.most - least;
    const int shift = range ? max(32 - (int)__builtin_clz(range) - 11, 0) : 0;
    int cell[HELD];
    unsigned slot[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (t[i].at != ~0ull) {
            cell[i] = (int)(((unsigned)(t[i].at >> 32) - least) >> shift);
            slot[i] = atomicAdd(&o.begin[cell[i]], 1u);
            atomicAdd(&o.weight[cell[i]], t[i].w);
        }
    __syncthreads();
    unsigned count[PER_CELL], c = 0, all;
    u64 weight[PER_CELL], w = 0, total;
#pragma unroll
    for (int i = 0; i < PER_CELL; ++i) {
        c += count[i] = o.begin[threadIdx.x * PER_CELL + i];
        w += weight[i] = o.weight[threadIdx.x * PER_CELL + i];
        if (count[i] > CROWD) o.crowd = 1;
    }
    const unsigned mine_c = c;
    const u64 mine_w = w;
    scan<DRAW>(c, w, all, total);
    c -= mine_c;
    w -= mine_w;
#pragma unroll
    for (int i = 0; i < PER_CELL; ++i) {
        o.begin[threadIdx.x * PER_CELL + i] = c;
        o.weight[threadIdx.x * PER_CELL + i] = w;
        c += count[i];
        w += weight[i];
    }
    if (threadIdx.x == DRAW - 1) o.begin[CELLS] = c;
    __syncthreads();
    if (o.crowd) return false;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (t[i].at != ~0ull) {
            const unsigned to = o.begin[cell[i]] + slot[i];
            o.at[to] = t[i].at;
            o.own[to] = t[i].w;
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (t[i].at != ~0ull) {
            const unsigned first = o.begin[cell[i]], end = o.begin[cell[i] + 1];
            t[i].before = first;
            t[i].weight = o.weight[cell[i]];
            for (unsigned j = first; j < end; ++j)
                if (o.at[j] < t[i].at) ++t[i].before, t[i].weight += o.own[j];
        }
    return true;
}

// A row whose small top-k has left few tokens: every token is compared with every other, by LANES lanes, first for its place in
// the order, then for its place among the kept ones' ids. Few barriers (1 x 151936, top-k 10, 50 and 100 with top-p: 13.2,
// 14.6 and 18.3 us, by order() 18.5, 19.6 and 19.7; 64 rows of 50 26.0 and 31.3; up to 256 tokens with 4 lanes each: top-k 190 20.4 to
// 21.1, by order() 19.7).
constexpr int LANES = 8, PAIRS = DRAW / LANES;
struct Few {
    ulonglong2 token[PAIRS];  // (place, weight), then (id, kept weight)
    u64 sum;
};
__device__ __forceinline__ u64 sum_lanes(u64 x) {
    static_assert(LANES == 8, "three steps");
    x += dpp64<DPP_XOR1, 0xF>(x);
    x += dpp64<DPP_XOR2, 0xF>(x);
    return x + dpp64<DPP_HALF_MIRROR, 0xF>(x);
}
__device__ __forceinline__ void draw_few(const SampleArgs &a, int number, const Rule &r, double u, uint2 listed, int n, Few &few) {
    if ((int)threadIdx.x < n) {
        const float v = __uint_as_float(listed.y);
        few.token[threadIdx.x] = make_ulonglong2(place(v, listed.x), r.weight(r.distance(v)));
    }
    __syncthreads();
    const int i = threadIdx.x / LANES, first = threadIdx.x % LANES;
    const ulonglong2 mine = few.token[min(i, n - 1)];
    // (the tokens in front of it, and their weight: 2^43 each at most, 128 of them below 2^50, the count above)
    u64 before = 0;
#pragma unroll 4
    for (int j = first; j < n; j += LANES) {
        const ulonglong2 x = few.token[j];
        before += x.x < mine.x ? x.y + (1ull << 52) : 0;
    }
    before = sum_lanes(before);
    const int place_of = (int)(before >> 52);
    const u64 weight = before & ((1ull << 52) - 1);
    if (i < n && first == 0 && place_of == min(r.k, n) - 1) few.sum = weight + mine.y;  // of the first k
    __syncthreads();
    const bool keep = i < n && place_of < r.k && (r.p == 1.0 || (double)weight < r.p * (double)few.sum || !weight) &&
                      r.likely(r.distance(of_rising(~(uint32_t)(mine.x >> 32))));
    const u64 w = keep ? mine.y : 0;
    if (i < n && first == 0) few.token[i] = make_ulonglong2((uint32_t)mine.x, w);
    __syncthreads();
    u64 upto = 0, total = 0;
#pragma unroll 4
    for (int j = first; j < n; j += LANES) {
        const ulonglong2 x = few.token[j];
        total += x.y;
        upto += x.x < (uint32_t)mine.x ? x.y : 0;
    }
    upto = sum_lanes(upto);
    total = sum_lanes(total);
    if (keep && first == 0) drawn(a, number, target_of(u, total), upto, w, total, (int)(uint32_t)mine.x);
}

__global__ __launch_bounds__(DRAW) void sample_draw(SampleArgs a, Rows rows) {
    __shared__ u64 sums[MOST_PIECES], highest, of_k;
    __shared__ struct { int piece; u64 before; } hit;
    __shared__ unsigned in_front, near;
    __shared__ union {
        Ordered ordered;
        Listed list;
        struct { u64 w[LIST]; uint32_t at[LIST]; } near;
        Few few;
    } lds;
    const int number = blockIdx.x;
    const Row &row = rows.row(number);
    const float *x = a.logits + (size_t)number * a.ld;
    // (everything that the steps below may want, in one trip to memory)
    const Rule r = row.rule;
    const unsigned listed = row.listed;
    const double u = a.u[number];
    Border b = row.border;
    constexpr int MINE = MOST_PIECES / DRAW;
    const int pieces = (a.n + PIECE - 1) / PIECE;
    u64 of_piece[MINE];
#pragma unroll
    for (int j = 0; j < MINE; ++j) of_piece[j] = row.sum[threadIdx.x * MINE + j];
    uint2 of_list[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) of_list[i] = row.list[threadIdx.x + i * DRAW];
    if (r.mode == GREEDY) {
        if (threadIdx.x == 0) {
            const bool some = r.m != -INFINITY;
            a.ids[number] = some ? row.best : -1;
            if (a.prob) a.prob[number] = some ? 1.0f : 0.0f;
        }
        return;
    }
    if (r.mode == SMALL && listed <= PAIRS) {
        draw_few(a, number, r, u, of_list[0], listed, lds.few);
        return;
    }
    // tokens in front of bin b.lo are kept, and of bins up to b.hi those up to the place `last`
    u64 last = 0;
    if (r.mode == WHOLE) b = {-1, BINS + 1, BINS, 0, 0, 0, 0};
    if (r.mode == SMALL) b = {0, 0, BINS, 0, 0, 0, 0};
    const int k_end = r.mode == SMALL ? b.hi : b.k_bin;  // bins k_bin .. k_end hold top-k's last token
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        const int piece = threadIdx.x * MINE + j;
        sums[piece] = piece < pieces && r.mode != SMALL ? of_piece[j] : 0;
    }
    Token t[HELD];
    int bin[HELD];
    bool keep[HELD], small = false;
    if (r.mode != WHOLE) {
        if (threadIdx.x == 0) highest = 0, of_k = 0, in_front = 0, near = 0;
        unsigned front = 0;
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const bool is = listed <= LIST && threadIdx.x + i * DRAW < listed;
            const float v = __uint_as_float(of_list[i].y);
            t[i] = {is ? place(v, of_list[i].x) : ~0ull, is ? r.weight(r.distance(v)) : 0, 0, 0};
            bin[i] = is ? r.bin(v) : BINS + 1;
            front += bin[i] < b.k_bin;
            keep[i] = false;
        }
        if (listed <= LIST && order(lds.ordered, t)) {
            // S: the weight of the first k
            u64 all = b.total;
            if (b.k_bin >= 0) {
                front = wave_scan(front);
                if ((threadIdx.x & 63) == 63 && front) atomicAdd(&in_front, front);
                __syncthreads();
                u64 w = 0;
#pragma unroll
                for (int i = 0; i < HELD; ++i) {
                    keep[i] = bin[i] < b.k_bin || (bin[i] <= k_end && b.k_count + (t[i].before - in_front) < (unsigned)r.k);
                    if (keep[i] && bin[i] >= b.k_bin) w += t[i].w;
                }
                w = last_lane(wave_scan(w));
                if ((threadIdx.x & 63) == 0 && w) atomicAdd(&of_k, w);
                __syncthreads();
                all = b.k_weight + of_k;
            } else {
#pragma unroll
                for (int i = 0; i < HELD; ++i) keep[i] = bin[i] <= BINS;
            }
            const double share = r.p * (double)all;
            u64 top = 0;
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                const u64 before = b.weight + t[i].weight;
                keep[i] = keep[i] && bin[i] <= b.hi && (r.p == 1.0 || (double)before < share || !before);
                if (keep[i]) top = max(top, t[i].at);
            }
            if (top) atomicMax(&highest, top);
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                keep[i] = keep[i] && t[i].w && r.likely(r.distance(of_rising(~(uint32_t)(t[i].at >> 32))));
                if (keep[i]) atomicAdd(&sums[(uint32_t)t[i].at / PIECE], t[i].w);
            }
            __syncthreads();
            last = highest;
            small = r.mode == SMALL;
        } else {
            if (threadIdx.x == 0) lds.list.n = listed;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < HELD; ++i)
                if (t[i].at != ~0ull) {
                    lds.list.at[threadIdx.x + i * DRAW] = t[i].at;
                    lds.list.weight[threadIdx.x + i * DRAW] = t[i].w;
                    lds.list.bin[threadIdx.x + i * DRAW] = (uint16_t)bin[i];
                }
            __syncthreads();
            u64 all = b.total;
            if (b.k_bin >= 0) {
                all = b.k_weight;
                last = last_place(lds.list, r, x, a.n, b.k_bin, k_end, b.k_count, all,
                                  [&](unsigned c, u64) { return c >= (unsigned)r.k; });
            }
            if (r.p < 1.0) {
                const double share = r.p * (double)all;
                u64 w = b.weight;
                last = last_place(lds.list, r, x, a.n, b.lo, b.hi, 0, w, [&](unsigned, u64 s) { return (double)s >= share; });
            }
            each_listed(lds.list, r, x, a.n, b.lo, b.hi, [&](u64 at, u64 w) {
                if (at <= last && r.likely(r.distance(of_rising(~(uint32_t)(at >> 32))))) atomicAdd(&sums[(uint32_t)at / PIECE], w);
            });
        }
    }
    __syncthreads();
    u64 total;
    u64 mine = 0;
#pragma unroll
    for (int j = 0; j < MINE; ++j) mine += of_piece[j] = sums[threadIdx.x * MINE + j];
    u64 upto = mine;
    scan<DRAW>(upto, total);
    if (!total) {  // (the maximum is kept and weighs 2^43: no row comes here, and none reads behind its end for want of a piece)
        if (threadIdx.x == 0) {
            a.ids[number] = -1;
            if (a.prob) a.prob[number] = 0.0f;
        }
        return;
    }
    const u64 target = target_of(u, total);
    upto -= mine;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        if (upto <= target && upto + of_piece[j] > target) hit = {(int)threadIdx.x * MINE + j, upto};
        upto += of_piece[j];
    }
    __syncthreads();
    if (small) {
        // all kept tokens are at hand: those of the piece
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (keep[i] && (int)((uint32_t)t[i].at / PIECE) == hit.piece) {
                const unsigned to = atomicAdd(&near, 1u);
                lds.near.at[to] = (uint32_t)t[i].at;
                lds.near.w[to] = t[i].w;
            }
        __syncthreads();
        for (unsigned i = threadIdx.x; i < near; i += DRAW) {
            u64 before = hit.before;
            for (unsigned j = 0; j < near; ++j) before += lds.near.at[j] < lds.near.at[i] ? lds.near.w[j] : 0;
            drawn(a, number, target, before, lds.near.w[i], total, (int)lds.near.at[i]);
        }
        return;
    }
    // the piece's values, one per thread
    const int at = hit.piece * PIECE + threadIdx.x;
    u64 w = 0;
    if (threadIdx.x < PIECE && at < a.n) {
        const float v = value(x[at]);
        const double y = r.distance(v);
        const int in = r.bin(v);
        if (r.likely(y) && (in < b.lo || (in <= b.hi && place(v, at) <= last))) w = r.weight(y);
    }
    u64 before = w, here;
    scan<DRAW>(before, here);
    drawn(a, number, target, hit.before + before - w, w, total, at);
}

template <bool VEC> void launch(const SampleArgs &a, const Rows &rows, int n, hipStream_t st) {
    const dim3 block(THREADS);
    // workgroups of a row: four for each CU in all, a piece for each wave at least (64 x 151936 with top-p 55.8 us, two for each CU
    // 60.0, three 56.8, five 57.1)
    const int pieces = (a.n + PIECE - 1) / PIECE, parts = std::max(1, std::min((pieces + 3) / 4, 1024 / n));
    hipLaunchKernelGGL((sample_scan<VEC>), dim3(n * rows.chunks), block, 0, st, a, rows);
    hipLaunchKernelGGL((sample_bins<VEC>), dim3(n * parts), block, 0, st, a, rows, parts);
    hipLaunchKernelGGL((sample_border<VEC>), dim3(n * parts), block, 0, st, a, rows, parts);
    hipLaunchKernelGGL(sample_draw, dim3(n), dim3(DRAW), 0, st, a, rows);
}

}  // namespace

// Rows at a time: a row's scratch is 61 KB and more, and so many fill the GPU.
constexpr int MOST_ROWS = 1024;

int launch_sample(const SampleArgs &a, int n, hipStream_t st) {
    Rows rows;
    rows.chunks = (a.n + CHUNK - 1) / CHUNK;
    rows.step = sizeof(Row) + (size_t)rows.chunks * GROUPS * sizeof(float);
    const std::lock_guard<std::mutex> lk(lib_scratch_mutex());
    rows.base = (char *)lib_scratch(std::min(n, MOST_ROWS) * rows.step);
    if (!rows.base) return -1;
    for (int first = 0; first < n; first += MOST_ROWS) {
        SampleArgs x = a;
        x.logits += (size_t)first * a.ld;
        x.how += first;
        x.u += first;
        x.ids += first;
        if (x.prob) x.prob += first;
        const int here = std::min(n - first, MOST_ROWS);
        // (four logits to a load where all rows allow it: 64 x 151936 with top-p 55.8 us, without a border 28.7, one at a time 57.2 and
        // 30.8)
        if (((uintptr_t)x.logits & 15) == 0 && a.ld % 4 == 0) launch<true>(x, rows, here, st);
        else launch<false>(x, rows, here, st);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace llamd
