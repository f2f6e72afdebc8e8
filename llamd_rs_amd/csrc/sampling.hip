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
// No sort: the tokens kept are those up to one border in that order, and the draw goes by index. Four launches over the
// row in chunks of 4096:
//   maxima: each chunk's maximum and minimum
//   bins: counts and weights by distance from the maximum (2048 bins), in LDS and then by integer atomics
//   border: the bins that hold the border, found by every workgroup for itself; their tokens are listed, the weights in front
//           of them added up by chunk
//   draw: one workgroup per row finds the border among the listed tokens by digits of (x, index), the chunk that u falls into,
//         and the token in it
// Rows without top-k and top-p need no border: bins adds up their chunks. A list that is too long (most logits equal) is
// replaced by the row itself.
//
// Bound: the launches and the chain inside them for few rows; reading the row three times (once from memory) and the 64-bit
// exponentials for many.
#include <algorithm>
#include <mutex>

#include "common.hpp"
#include "launch.hpp"
#include "sample.hpp"

namespace llamd {
namespace {

typedef unsigned long long u64;

constexpr int THREADS = 256, EACH = 16, CHUNK = THREADS * EACH, BINS = 2048, PER = BINS / THREADS, LIST = 2048;
constexpr int MOST_CHUNKS = SAMPLE_MOST / CHUNK;
static_assert(MOST_CHUNKS <= THREADS, "a thread per chunk");
constexpr double RANGE = 44.0;  // weights below 2^-44 are 0

struct Extremes {
    float top, least;  // least: of the finite values
    int at, pad;
};
// A row's scratch.
struct Row {
    unsigned count[BINS];
    u64 weight[BINS];
    u64 sum[MOST_CHUNKS];      // of the weights in front of the border's bins
    Extremes chunk[MOST_CHUNKS];
    unsigned listed, pad[3];
    uint2 list[LIST];          // (index, x's bits), in any order
};

__device__ __forceinline__ float value(float x) { return x == x ? x + 0.0f : -INFINITY; }  // (-0 is 0)

// Position in the order: x falling, then index rising.
__device__ __forceinline__ u64 place(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x);
    const uint32_t rising = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (u64)~rising << 32 | i;
}

// A row's rule, and the distance of its logits from the maximum in powers of two.
struct Rule {
    double m, c;       // maximum, log2(e) / T
    double furthest;   // min-p's
    double per_bin;
    double p;
    int k;             // 0: all
    bool greedy, cut;  // the maximum alone; top-k or top-p

    __device__ __forceinline__ double distance(float x) const { return (double)x == m ? 0.0 : (m - (double)x) * c; }
    // 2^-y as a multiple of 2^-43; 0 for NaN (an infinite temperature, and a token ruled out)
    static __device__ __forceinline__ u64 weight(double y) {
        if (!(y < RANGE)) return 0;
        const double r = rint(y), f = (r - y) * 0.69314718055994530942;  // |f| <= ln(2) / 2
        // e^f by its series: the next term is below 2^-46
        double s = 1.0 / 39916800.0;
        s = fma(s, f, 1.0 / 3628800.0);
        s = fma(s, f, 1.0 / 362880.0);
        s = fma(s, f, 1.0 / 40320.0);
        s = fma(s, f, 1.0 / 5040.0);
        s = fma(s, f, 1.0 / 720.0);
        s = fma(s, f, 1.0 / 120.0);
        s = fma(s, f, 1.0 / 24.0);
        s = fma(s, f, 1.0 / 6.0);
        s = fma(s, f, 0.5);
        s = fma(s, f, 1.0);
        s = fma(s, f, 1.0);
        // times 2^(43 - r), rounded to a whole number in the last places of 2^52
        const double w = __longlong_as_double(__double_as_longlong(s) + ((long long)(43 - (int)r) << 52)) + 4503599627370496.0;
        return (u64)__double_as_longlong(w) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ int bin(double y) const { return min((int)(y * per_bin), BINS - 1); }
    __device__ __forceinline__ bool likely(double y) const { return y <= furthest; }
};

// The rule of a row from its chunks' extremes. All threads of the workgroup; `at`: the maximum's first index.
__device__ __forceinline__ Rule rule_of(const SampleArgs &a, const Row &row, int number, int chunks, int &at) {
    __shared__ float tops[4], leasts[4];
    __shared__ int places[4];
    const SampleRule how = a.how[number];
    Extremes x = {-INFINITY, INFINITY, 0x7FFFFFFF, 0};
    if ((int)threadIdx.x < chunks) x = row.chunk[threadIdx.x];
    wave_argmax(x.top, x.at, -INFINITY);
    x.least = wave_reduce(x.least, INFINITY, [](float u, float v) { return fminf(u, v); });
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = x.top, leasts[threadIdx.x >> 6] = x.least, places[threadIdx.x >> 6] = x.at;
    __syncthreads();
    float top = tops[0], least = leasts[0];
    at = places[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
        argmax_step(top, at, tops[w], places[w]);
        least = fminf(least, leasts[w]);
    }
    Rule r;
    r.m = top;
    r.c = 1.4426950408889634074 / (double)how.temperature;
    r.greedy = !(how.temperature > 0.0f) || top == -INFINITY;
    r.furthest = how.min_p > 0.0f ? fmax(-log2((double)how.min_p), 0.0) : INFINITY;
    const double range = fmin(r.distance(least), RANGE);  // (a least of +inf: no finite value)
    r.per_bin = range > 0.0 ? (BINS - 1) / range : 0.0;
    r.k = how.top_k > 0 && how.top_k < a.n ? how.top_k : 0;
    r.p = how.top_p < 1.0f ? fmax((double)how.top_p, 0.0) : 1.0;  // (NaN: all)
    r.cut = r.k || r.p < 1.0;
    return r;
}

// f(x, index) for every logit of a chunk, 16 per thread. VEC: rows are 16-byte aligned.
template <bool VEC, class F> __device__ __forceinline__ void each(const float *x, int n, int chunk, F f) {
    const int first = chunk * CHUNK;
    if (first + CHUNK <= n) {
        float v[EACH];
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < EACH / 4; ++j) *(float4 *)(v + 4 * j) = *(const float4 *)(x + first + (j * THREADS + threadIdx.x) * 4);
        } else {
#pragma unroll
            for (int j = 0; j < EACH; ++j) v[j] = x[first + j * THREADS + threadIdx.x];
        }
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            f(value(v[j]), first + (VEC ? (j / 4 * THREADS + (int)threadIdx.x) * 4 + j % 4 : j * THREADS + (int)threadIdx.x));
    } else {
        for (int i = first + threadIdx.x; i < n; i += THREADS) f(value(x[i]), i);
    }
}

// Inclusive sums over the threads' numbers, and all threads' sum.
template <class T> __device__ __forceinline__ T scan(T mine, T &total) {
    __shared__ T waves[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const T x = __shfl_up(mine, s, 64);
        if (lane >= s) mine += x;
    }
    __syncthreads();  // (a scan before this one is read)
    if (lane == 63) waves[wave] = mine;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) mine += waves[w];
        total += waves[w];
    }
    return mine;
}

template <bool VEC> __global__ __launch_bounds__(THREADS) void sample_maxima(SampleArgs a, Row *rows, int chunks) {
    __shared__ float tops[4], leasts[4];
    __shared__ int places[4];
    const int number = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    Row &row = rows[number];
    float top = -INFINITY, least = INFINITY;
    int at = 0x7FFFFFFF;
    each<VEC>(a.logits + (size_t)number * a.ld, a.n, chunk, [&](float x, int i) {
        argmax_step(top, at, x, i);
        if (x > -INFINITY) least = fminf(least, x);
    });
    // what the next launches add to
    for (int i = chunk * THREADS + threadIdx.x; i < BINS; i += chunks * THREADS) row.count[i] = 0, row.weight[i] = 0;
    if (chunk == 0 && threadIdx.x == 0) row.listed = 0;
    wave_argmax(top, at, -INFINITY);
    least = wave_reduce(least, INFINITY, [](float u, float v) { return fminf(u, v); });
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top, leasts[threadIdx.x >> 6] = least, places[threadIdx.x >> 6] = at;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) argmax_step(top, at, tops[w], places[w]), least = fminf(least, leasts[w]);
        row.chunk[chunk] = {top, least, at, 0};
    }
}

template <bool VEC> __global__ __launch_bounds__(THREADS) void sample_bins(SampleArgs a, Row *rows, int chunks) {
    __shared__ unsigned count[BINS];
    __shared__ u64 weight[BINS];
    const int number = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    Row &row = rows[number];
    int at;
    const Rule r = rule_of(a, row, number, chunks, at);
    if (r.greedy) return;
    const float *x = a.logits + (size_t)number * a.ld;
    if (!r.cut) {
        u64 sum = 0, total;
        each<VEC>(x, a.n, chunk, [&](float v, int) {
            const double y = r.distance(v);
            if (r.likely(y)) sum += r.weight(y);
        });
        scan(sum, total);
        if (threadIdx.x == 0) row.sum[chunk] = total;
        return;
    }
    for (int i = threadIdx.x; i < BINS; i += THREADS) count[i] = 0, weight[i] = 0;
    __syncthreads();
    each<VEC>(x, a.n, chunk, [&](float v, int) {
        const double y = r.distance(v);
        const u64 w = r.weight(y);
        if (w) {
            const int b = r.bin(y);
            atomicAdd(&count[b], 1u);
            atomicAdd(&weight[b], w);
        }
    });
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += THREADS)
        if (count[i]) {
            atomicAdd(&row.count[i], count[i]);
            atomicAdd(&row.weight[i], weight[i]);
        }
}

// Where the border lies.
struct Border {
    int k_bin;             // top-k's last token's bin; -1: all tokens are among the first k
    int lo, hi;            // the bins that may hold the last token kept
    unsigned k_count;      // tokens in front of k_bin, and their weight
    u64 k_weight, weight;  // weight of the tokens in front of lo
    u64 total;             // of all
};
__device__ __forceinline__ Border border_of(const Row &row, const Rule &r) {
    __shared__ Border found;
    unsigned count[PER], counts = 0, all;
    u64 weight[PER], weights = 0, total;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        counts += count[i] = row.count[threadIdx.x * PER + i];
        weights += weight[i] = row.weight[threadIdx.x * PER + i];
    }
    const unsigned counts_before = scan(counts, all) - counts;
    const u64 before = scan(weights, total) - weights;
    if (threadIdx.x == 0) found = {-1, BINS, BINS, 0, 0, 0, total};  // (no border: fewer than top_k, no top-p)
    __syncthreads();
    // the bin where f(sum in front of it) is false and f(sum with it) is true
    if (r.k && all > (unsigned)r.k) {
        unsigned c = counts_before;
        u64 w = before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (c < (unsigned)r.k && c + count[i] >= (unsigned)r.k) {
                found.k_bin = found.lo = found.hi = threadIdx.x * PER + i;
                found.k_count = c;
                found.k_weight = found.weight = w;
                found.total = w + weight[i];  // (at the most, of those kept)
            }
            c += count[i];
            w += weight[i];
        }
    }
    __syncthreads();
    if (r.p < 1.0) {
        // the sum that p is a share of lies between these
        const double least = r.p * (double)(found.k_bin < 0 ? total : found.k_weight), most = r.p * (double)found.total;
        __syncthreads();
        u64 w = before;
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

template <bool VEC> __global__ __launch_bounds__(THREADS) void sample_border(SampleArgs a, Row *rows, int chunks) {
    __shared__ unsigned listed, first;
    __shared__ uint2 list[LIST];
    const int number = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    Row &row = rows[number];
    int at;
    const Rule r = rule_of(a, row, number, chunks, at);
    if (r.greedy || !r.cut) return;
    const Border b = border_of(row, r);
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    u64 sum = 0, total;
    each<VEC>(a.logits + (size_t)number * a.ld, a.n, chunk, [&](float v, int i) {
        const double y = r.distance(v);
        const u64 w = r.weight(y);
        if (!w) return;
        const int bin = r.bin(y);
        if (bin < b.lo && r.likely(y)) sum += w;
        if ((bin >= b.lo && bin <= b.hi) || bin == b.k_bin) {
            const unsigned to = atomicAdd(&listed, 1u);
            if (to < LIST) list[to] = make_uint2(i, __float_as_uint(v));
        }
    });
    scan(sum, total);
    if (threadIdx.x == 0) {
        row.sum[chunk] = total;
        first = listed ? atomicAdd(&row.listed, listed) : 0;
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < min(listed, (unsigned)LIST); i += THREADS)
        if (first + i < LIST) row.list[first + i] = list[i];
}

// The border's tokens: from the list, or where that is too short, from the row.
template <class F> __device__ __forceinline__ void each_listed(const SampleArgs &a, const Row &row, const Rule &r, const float *x, F f) {
    if (row.listed <= LIST) {
        for (unsigned i = threadIdx.x; i < row.listed; i += THREADS) {
            const float v = __uint_as_float(row.list[i].y);
            const double y = r.distance(v);
            f(v, row.list[i].x, y, r.weight(y));
        }
    } else {
        for (int i = threadIdx.x; i < a.n; i += THREADS) {
            const float v = value(x[i]);
            const double y = r.distance(v);
            const u64 w = r.weight(y);
            if (w) f(v, (uint32_t)i, y, w);
        }
    }
}

// The last place of bins [lo, hi] to keep: that of the first token with which it is done(tokens up to it, their weight),
// counted from `count` and `weight`, or one between it and the bins' next; `weight` becomes that weight. By digits of 8 bits of
// the place, the highest first.
template <class Done>
__device__ __forceinline__ u64 last_place(const SampleArgs &a, const Row &row, const Rule &r, const float *x, int lo, int hi,
                                          unsigned count, u64 &weight, Done done) {
    __shared__ unsigned counts[256];
    __shared__ u64 weights[256];
    __shared__ struct { unsigned digit, count, here; u64 weight, mine; } next;
    u64 prefix = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        counts[threadIdx.x] = 0;
        weights[threadIdx.x] = 0;
        __syncthreads();
        each_listed(a, row, r, x, [&](float v, uint32_t i, double y, u64 w) {
            const int bin = r.bin(y);
            const u64 at = place(v, i);
            if (bin < lo || bin > hi || (shift < 56 && at >> (shift + 8) != prefix >> (shift + 8))) return;
            atomicAdd(&counts[at >> shift & 255], 1u);
            atomicAdd(&weights[at >> shift & 255], w);
        });
        __syncthreads();
        unsigned all;
        u64 total;
        const unsigned c = counts[threadIdx.x], upto = scan(c, all) + count;
        const u64 w = weights[threadIdx.x], with = scan(w, total) + weight;
        // the first digit with which it is done; if rounding leaves none, the last that there is
        const bool here = c && done(upto, with);
        const bool none = c && upto == all + count && !done(upto, with);
        if ((here && !(upto - c > count && done(upto - c, with - w))) || none)
            next = {threadIdx.x, upto - c, c, with - w, w};
        __syncthreads();
        prefix |= (u64)next.digit << shift;
        count = next.count;
        weight = next.weight;
        const unsigned here_count = next.here;
        const u64 mine = next.mine;
        __syncthreads();
        if (here_count == 1 || shift == 0) {
            weight += mine;
            return prefix | ((1ull << shift) - 1);
        }
    }
    return prefix;
}

__global__ __launch_bounds__(THREADS) void sample_draw(SampleArgs a, Row *rows, int chunks) {
    __shared__ u64 sums[MOST_CHUNKS];
    __shared__ struct { int chunk; u64 before; } hit;
    const int number = blockIdx.x;
    const Row &row = rows[number];
    const float *x = a.logits + (size_t)number * a.ld;
    int best;
    const Rule r = rule_of(a, row, number, chunks, best);
    if (r.greedy) {
        if (threadIdx.x == 0) {
            const bool some = r.m != -INFINITY;
            a.ids[number] = some ? best : -1;
            if (a.prob) a.prob[number] = some ? 1.0f : 0.0f;
        }
        return;
    }
    int lo = BINS, hi = BINS;  // tokens of bins in front of lo are kept, and of bins up to hi those up to the place `last`
    u64 last = 0;
    if ((int)threadIdx.x < chunks) sums[threadIdx.x] = row.sum[threadIdx.x];
    if (r.cut) {
        const Border b = border_of(row, r);
        u64 all = b.total;
        lo = b.lo;
        hi = b.hi;
        if (b.k_bin >= 0) {
            all = b.k_weight;
            last = last_place(a, row, r, x, b.k_bin, b.k_bin, b.k_count, all,
                              [&](unsigned c, u64) { return c >= (unsigned)r.k; });
        }
        if (r.p < 1.0) {
            const double share = r.p * (double)all;
            u64 w = b.weight;
            last = last_place(a, row, r, x, b.lo, b.hi, 0, w, [&](unsigned, u64 s) { return (double)s >= share; });
        }
        __syncthreads();
        each_listed(a, row, r, x, [&](float v, uint32_t i, double y, u64 w) {
            const int bin = r.bin(y);
            if (bin >= lo && bin <= hi && place(v, i) <= last && r.likely(y)) atomicAdd(&sums[i / CHUNK], w);
        });
    }
    __syncthreads();
    u64 total;
    const u64 mine = (int)threadIdx.x < chunks ? sums[threadIdx.x] : 0, upto = scan(mine, total);
    // the running sum that is exceeded: u times all, at most all but one
    const double u = a.u[number], want = u * (double)total;
    const u64 target = want > 0.0 ? (want < (double)total ? min((u64)want, total - 1) : total - 1) : u == u ? 0 : total - 1;
    if (upto > target && upto - mine <= target) hit = {(int)threadIdx.x, upto - mine};
    __syncthreads();
    const int first = hit.chunk * CHUNK + threadIdx.x * EACH;
    u64 before = hit.before, w[EACH], sum = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        w[j] = 0;
        if (first + j < a.n) {
            const float v = value(x[first + j]);
            const double y = r.distance(v);
            w[j] = r.likely(y) ? r.weight(y) : 0;
            if (w[j]) {
                const int bin = r.bin(y);
                if (bin >= lo && (bin > hi || place(v, first + j) > last)) w[j] = 0;
            }
        }
        sum += w[j];
    }
    u64 here;
    before += scan(sum, here) - sum;
    if (before <= target && before + sum > target) {
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            if (before <= target && before + w[j] > target) {
                a.ids[number] = first + j;
                if (a.prob) a.prob[number] = (float)((double)w[j] / (double)total);
            }
            before += w[j];
        }
    }
}

}  // namespace

int launch_sample(const SampleArgs &a, int rows, hipStream_t st) {
    const int chunks = (a.n + CHUNK - 1) / CHUNK;
    const std::lock_guard<std::mutex> lk(lib_scratch_mutex());
    Row *scratch = (Row *)lib_scratch((size_t)rows * sizeof(Row));
    if (!scratch) return -1;
    const dim3 grid((unsigned)(rows * chunks)), block(THREADS);
    if (((uintptr_t)a.logits & 15) == 0 && a.ld % 4 == 0) {
        hipLaunchKernelGGL((sample_maxima<true>), grid, block, 0, st, a, scratch, chunks);
        hipLaunchKernelGGL((sample_bins<true>), grid, block, 0, st, a, scratch, chunks);
        hipLaunchKernelGGL((sample_border<true>), grid, block, 0, st, a, scratch, chunks);
    } else {
        hipLaunchKernelGGL((sample_maxima<false>), grid, block, 0, st, a, scratch, chunks);
        hipLaunchKernelGGL((sample_bins<false>), grid, block, 0, st, a, scratch, chunks);
        hipLaunchKernelGGL((sample_border<false>), grid, block, 0, st, a, scratch, chunks);
    }
    hipLaunchKernelGGL(sample_draw, dim3(rows), block, 0, st, a, scratch, chunks);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace llamd
