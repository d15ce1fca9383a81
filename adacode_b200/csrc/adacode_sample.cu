// One token per row of logits: temperature, top-k, top-p, min-p and the draw from a given uniform number.
//
// Every cut (the top_k first, the nucleus, min_p) keeps a prefix of the order (descending logit, ascending token); tokens are kept
// as 64-bit keys of that order.  A row has a cluster of 1 to 8 CTAs, whose warps own consecutive spans of the vocabulary.  Passes over the row, which
// after the first come from L2:
//   1  the largest logit, and of every thread the largest of its tokens, in two halves.
//   top_k up to kMostK: the k-th largest of those many maxima has at least k tokens above it, and hardly more.  Threads whose maxima reach it list
//      their tokens that do; the list is sorted, and all else happens in it.  No weight of any other token is computed.
//   top_p alone: 2 adds up weights, roughly, per interval of the logit (2048 intervals), which says where the nucleus about ends;
//      3 computes every weight once, in 64 bits, and adds up, per span, what lies above that interval, what does not, and lists what
//      lies in it.  These sums say exactly whether the interval was right (if not, the guess is made again from there); the sorted list says
//      where the nucleus ends.
//   neither: 3 alone.
//   Then the span in which the draw falls is walked again.
// Measured: 192 rows of 151936 with top_p and min_p 150 us (the weights take half of it: 29 million of eight operations of 64 bits; issue slots
// half busy), 64 rows of 128256 with top_k and top_p 22 us (33 MB, twice), one row of 32000 11 us (latency: four passes that wait for one another).
// What fits no list (thousands of equal logits at a border, a larger top_k) goes the slow way: bisection of the keys by one CTA.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "adacode.h"

#include <atomic>

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMostCtas = 8;             // per row
constexpr int kStep = 256;               // tokens that a warp takes at a time, eight per lane
constexpr int kBins = 2048;
constexpr int kList = 4096;
constexpr int kMostK = 1024;

struct SampleArgs {
    const void *logits;
    long long row_stride;
    int V;
    bool wide;                           // rows on 16-byte boundaries
    const float *uniforms, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int64_t *tokens;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
// plus infinity counts as the largest number
__device__ __forceinline__ float capped(float v) { return fminf(v, FLT_MAX); }
__device__ __forceinline__ float most_of(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));      // (passes NaN over)
    return r;
}
__device__ __forceinline__ float least_of(float a, float b, float c) {
    float r;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// NaN and minus infinity have key 0 (never drawn), both zeros one key.
__device__ __forceinline__ uint32_t key_of(float v) {
    if (!(v > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(capped(v) + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key); }
// the order: descending logit, ascending token
__device__ __forceinline__ uint64_t place_of(float v, int token) { return (uint64_t)key_of(v) << 32 | (0xFFFFFFFFu - (uint32_t)token); }
__device__ __forceinline__ int token_of(uint64_t place) { return (int)(0xFFFFFFFFu - (uint32_t)place); }

struct Shared {
    double roots[128];                   // 2**(j / 128)
    uint32_t count[kBins];               // (later: the span of every listed token)
    uint64_t list[kList];
    double line[kMostK];
    double span_all[kMostCtas * kWarps], span_kept[kMostCtas * kWarps];
    double scan[kWarps + 1];
    unsigned long long slow[kWarps];
    double cta_below;
    float low[kWarps], cta_low, cta_top, cut_low, edge[2];
    int scan_n[kWarps];
    int listed, found, decided;
    uint64_t border;
};

// What turns a logit into its weight: w = exp((x - largest) / T) = 2**(x k - largest k).  Below `floor` (600 T from the largest) it is 0.  (The largest
// logit's own is 1 but for a rounding; what is compared with it is compared with that.  Where k would take x k beyond 2**40, at temperatures
// that leave the largest logit alone, it is held there: its neighbours are then 2**16 powers of two away.)
struct Weights {
    double k, shift;
    float floor;
    const double *roots;
    __device__ Weights(float top, float t, const double *roots)
        : k(fmin(1.4426950408889634074 / (double)t, 1099511627776.0 / fabs((double)top))), shift(-(double)top * k), floor(fmaxf(top - 600.f * t, -FLT_MAX)), roots(roots) {}
    // The exponent rounded to 1/128; the power of the rest r by the Taylor series of 2**r (degree 3, |r| <= 1/256: the next term is below 2.3e-12);
    // 128 roots of 2.  Eight operations of 64 bits, less than half the time of exp(), whose last bits no draw needs.
    __device__ __forceinline__ double of(float v) const {           // (where there is any)
        const double t = fma((double)capped(v), k, shift);
        constexpr double kShift = 6755399441055744.0 / 128.0;      // 1.5 x 2**52 / 128
        const double shifted = t + kShift;
        const int n = __double2loint(shifted);
        const double r = t - (shifted - kShift);
        constexpr double kLn2 = 0.69314718055994530942;
        const double power = fma(fma(fma(r, kLn2 * kLn2 * kLn2 / 6.0, kLn2 * kLn2 / 2.0), r, kLn2), r, 1.0) * roots[n & 127];
        return __hiloint2double(__double2hiint(power) + ((n >> 7) << 20), __double2loint(power));
    }
    __device__ __forceinline__ bool any(float v) const { return v >= floor; }          // (not NaN)
    __device__ __forceinline__ double operator()(float v) const { return any(v) ? of(v) : 0.0; }
};

template <typename R, typename Op>
__device__ __forceinline__ R warp_reduce(R v, Op op) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = op(v, __shfl_xor_sync(kFull, v, d));
    return v;
}
template <typename R, typename Op>
__device__ R block_reduce(R v, Op op, R *shared) {
    v = warp_reduce(v, op);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    R r = shared[0];
    for (int w = 1; w < kWarps; ++w) r = op(r, shared[w]);
    return r;
}
struct Plus {
    template <typename R>
    __device__ __forceinline__ R operator()(R p, R q) const { return p + q; }
};
struct Most {
    template <typename R>
    __device__ __forceinline__ R operator()(R p, R q) const { return p > q ? p : q; }
};
struct Least {
    template <typename R>
    __device__ __forceinline__ R operator()(R p, R q) const { return p < q ? p : q; }
};

// Sum of all threads' values before this thread's; `total`: of all.
template <typename R>
__device__ R block_scan(R v, R &total, R *shared) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    R incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const R u = __shfl_up_sync(kFull, incl, d);
        if (lane >= d) incl += u;
    }
    __syncthreads();
    if (lane == 31) shared[warp] = incl;
    __syncthreads();
    R before = 0;
    total = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w == warp) before = total;
        total += shared[w];
    }
    return before + (incl - v);
}

// Descending sort of n (at most kList) different places.  Up to kThreads by counting what is larger, all others' bitonic, padded with zeros to a
// power of two: 300 places take 2000 cycles against 14 000.
__device__ void sort_places(uint64_t *list, int n) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (n <= kThreads) {
        const uint64_t mine = tid < n ? list[tid] : 0;
        int larger = 0;
        if (tid < n) {
#pragma unroll 8
            for (int i = 0; i < n; ++i) larger += list[i] > mine;
        }
        __syncthreads();
        if (tid < n) list[larger] = mine;
        __syncthreads();
        return;
    }
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kThreads) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = tid; i < size / 2; i += kThreads) {
                const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                const uint64_t p = list[lo], q = list[hi];
                if ((p < q) == ((lo & k) == 0)) list[lo] = q, list[hi] = p;
            }
            __syncthreads();
        }
}

// The smallest weight that stays; the largest weight, 1, always does.
__device__ __forceinline__ double smallest_of(const SampleArgs &a, int row) {
    const float p = a.min_p ? a.min_p[row] : a.min_p_all;
    return p > 0.f ? fminf(p, 1.f) : 0.f;
}

// Eight consecutive logits; NaN behind the row's end.
template <typename T>
__device__ __forceinline__ void load_eight(const T *x, int i, int V, bool wide, float (&v)[8]) {
    if (wide && i + 8 <= V) {
        T raw[8];
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4 *>(raw)[j] = __ldg(reinterpret_cast<const uint4 *>(x + i) + j);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = widen(raw[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = i + j < V ? widen(x[i + j]) : NAN;
    }
}

// A warp's tokens i0 .. i1 - 1, eight per lane and step, the loads of U steps under way at a time (with one, the first pass over 58 MB took 34 us).
template <int U, typename T, typename Use>
__device__ __forceinline__ void each_eight(const T *x, int i0, int i1, bool wide, Use &&use) {
    for (int i = i0 + (threadIdx.x & 31) * 8; i < i1; i += U * kStep) {
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) load_eight(x, i + u * kStep, i1, wide, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) use(v[u], i + u * kStep);
    }
}

// One CTA, bisection of the keys: (cut, ties) are a key and the number of its tokens that stay, lower tokens first.
template <typename T>
__device__ void sample_slowly(const SampleArgs &a, Shared &s, const T *x, int row, uint32_t top, const Weights &weight_of) {
    const int tid = threadIdx.x, V = a.V;
    const auto weight = [&](uint32_t key) { return key == 0 ? 0.0 : weight_of(value_of(key)); };
    const auto key_at = [&](int i) { return key_of(widen(x[i])); };
    uint32_t cut = 1;
    long long ties = V;
    const int k = a.top_k ? a.top_k[row] : a.top_k_all;
    if (k > 0 && k < V) {
        // the largest key that at least k tokens reach
        uint32_t lo = 1, hi = top;
        long long above = 0;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            unsigned long long n = 0;
            for (int i = tid; i < V; i += kThreads) n += key_at(i) >= mid;
            n = block_reduce(n, Plus(), s.slow);
            if ((long long)n >= k) lo = mid;
            else hi = mid - 1, above = (long long)n;
        }
        cut = lo;
        ties = k - above;
    }
    const float p = a.top_p ? a.top_p[row] : a.top_p_all;
    if (p < 1.f) {
        const auto total = [&](uint32_t from) {           // weight of the tokens of keys from `from` on, inside the cut
            double w = 0.0;
            unsigned long long n = 0;
            for (int i = tid; i < V; i += kThreads) {
                const uint32_t key = key_at(i);
                if (key >= from && key > cut) w += weight(key);
                n += key == cut;
            }
            w = block_reduce(w, Plus(), s.scan);
            n = block_reduce(n, Plus(), s.slow);
            if (from <= cut && n > 0) w += (double)((long long)n < ties ? (long long)n : ties) * weight(cut);   // (no token has a NaN's key)
            return w;
        };
        const double aim = (double)p * total(cut);
        // the largest key at which the weight reaches the aim
        uint32_t lo = cut, hi = top;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            if (total(mid) >= aim) lo = mid;
            else hi = mid - 1;
        }
        const double above = lo == 0xFFFFFFFFu ? 0.0 : total(lo + 1), w = weight(lo);
        // tokens of that key whose predecessors' weight is below the aim
        long long n = w > 0.0 ? (long long)fmin(ceil((aim - above) / w), 2147483647.0) : 0;
        if (n < 0) n = 0;
        if (lo == top && n < 1) n = 1;
        ties = lo == cut && ties < n ? ties : n;
        cut = lo;
    }
    const double least = smallest_of(a, row) * weight_of(value_of(top));
    // runs of consecutive tokens per thread: ties before it, weight before it, the token
    const int per = (V + kThreads - 1) / kThreads, i0 = min(tid * per, V), i1 = min(i0 + per, V);
    int same = 0, all_same = 0;
    for (int i = i0; i < i1; ++i) same += key_at(i) == cut;
    const long long before = block_scan(same, all_same, s.scan_n);
    const auto walk = [&](double from, double aim, int &found) {
        long long n = before;
        for (int i = i0; i < i1; ++i) {
            const uint32_t key = key_at(i);
            if (key == 0 || key < cut || (key == cut && n++ >= ties)) continue;
            const double w = weight(key);
            if (w < least || w == 0.0) continue;
            found = i;
            from += w;
            if (from > aim) return from;
        }
        return from;
    };
    int found = -1;
    const double mine = walk(0.0, INFINITY, found);
    double all = 0.0;
    const double from = block_scan(mine, all, s.scan);
    const double aim = (double)a.uniforms[row] * all;
    // the first run that ends behind the aim; rounding may leave none, then the last that has a token
    if (tid == 0) s.found = INT32_MAX;
    __syncthreads();
    if (mine > 0.0 && from + mine > aim) atomicMin(&s.found, tid);
    __syncthreads();
    if (s.found == INT32_MAX) {
        __syncthreads();
        if (tid == 0) s.found = -1;
        __syncthreads();
        if (mine > 0.0) atomicMax(&s.found, tid);
        __syncthreads();
    }
    if (tid == s.found) {
        walk(from, aim, found);
        a.tokens[row] = found;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared &s = *reinterpret_cast<Shared *>(raw);
    const cg::cluster_group cluster = cg::this_cluster();
    const int ctas = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / ctas, V = a.V;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = reinterpret_cast<const T *>(a.logits) + row * a.row_stride;
    Shared &first = *cluster.map_shared_rank(&s, 0);           // of the CTA that finishes the row
    // a warp's span: whole steps
    const int spans = ctas * kWarps, span = ((V + spans - 1) / spans + kStep - 1) / kStep * kStep;
    const int me = rank * kWarps + warp, i0 = min((long long)me * span, (long long)V), i1 = min((long long)i0 + span, (long long)V);
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- 1: the largest logit, the lowest token that has it
    const float p = a.top_p ? a.top_p[row] : a.top_p_all, t = a.temperature ? a.temperature[row] : a.temperature_all;
    const int k = a.top_k ? a.top_k[row] : a.top_k_all;
    const bool use_k = k > 0 && k < V, use_p = p < 1.f;
    float half_most[2] = {-INFINITY, -INFINITY}, low = INFINITY;
    each_eight<2>(x, i0, i1, a.wide, [&](const float (&v)[8], int) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) half_most[j / 4] = most_of(half_most[j / 4], v[j], v[j + 1]), low = least_of(low, v[j], v[j + 1]);
    });
    // (intervals reach down to the smallest finite logit, those of the top_k to the smallest of the maxima)
    if (use_k) {
        low = fminf(half_most[0] > -INFINITY ? half_most[0] : INFINITY, half_most[1] > -INFINITY ? half_most[1] : INFINITY);
    } else if (__any_sync(kFull, low == -INFINITY)) {
        low = INFINITY;
        each_eight<1>(x, i0, i1, a.wide, [&](const float (&v)[8], int) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (v[j] > -INFINITY && v[j] < low) low = v[j];
        });
    }
    if (tid < 128) s.roots[tid] = exp2((double)tid / 128.0);
    if (tid == 0) s.listed = 0, s.found = INT32_MAX;
    for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0;
    float top = block_reduce(fmaxf(half_most[0], half_most[1]), Most(), s.low);
    low = block_reduce(low, Least(), s.low);
    if (tid == 0) s.cta_top = top, s.cta_low = low;
    cluster.sync();
    for (int r = 0; r < ctas; ++r) {
        top = fmaxf(top, cluster.map_shared_rank(&s, r)->cta_top);
        low = fminf(low, cluster.map_shared_rank(&s, r)->cta_low);
    }
    if (!(top > -INFINITY) || !(t > 0.f)) {
        // nothing to draw, or the first token of the largest logit
        if (top > -INFINITY && fmaxf(half_most[0], half_most[1]) == top)
            each_eight<1>(x, i0, i1, a.wide, [&](const float (&v)[8], int i) {
#pragma unroll
                for (int j = 7; j >= 0; --j)
                    if (v[j] > -INFINITY && capped(v[j]) == capped(top)) atomicMin(&first.found, i + j);
            });
        cluster.sync();
        if (rank == 0 && tid == 0) a.tokens[row] = s.found == INT32_MAX ? -1 : s.found;
        return;
    }
    top = capped(top), low = capped(low);
    const uint32_t top_key = key_of(top);
    const Weights weight_of(top, t, s.roots);
    const double least = smallest_of(a, row) * weight_of(top);
    // (fewer maxima than tokens asked for, and too many tokens for the list: the slow way)
    bool slow = use_k && (k > kMostK || (V > kList && k > ctas * kThreads));
    if (slow) {
        cluster.sync();
        if (rank == 0) sample_slowly(a, s, x, row, top_key, weight_of);
        return;
    }
    float range = top - low;
    if (!use_k && range > 30.f * t) range = 30.f * t;           // (weights below e**-30 share an interval)
    // Tokens that a mask has given a type's lowest value would leave all others in one interval.  So the intervals of a top_k reach down to the
    // smallest maximum that weighs something (600 T from the top nothing does), and the last has all that lies below.
    const bool cut = use_k && range > 610.f * t;
    if (cut) {
        low = INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (capped(half_most[j]) >= top - 610.f * t) low = fminf(low, capped(half_most[j]));
        low = block_reduce(low, Least(), s.low);
        if (tid == 0) s.cut_low = low;
        cluster.sync();
        for (int r = 0; r < ctas; ++r) low = fminf(low, cluster.map_shared_rank(&s, r)->cut_low);
        range = fmaxf((top - low) * 1.01f, t);
    }
    const float per_bin = range > 0.f ? fminf(kBins / range, FLT_MAX) : 0.f;
    // (rounded by an addition: the conversion unit is slow; of NaN the last)
    const auto bin_of = [&](float v) { return (int)(__float_as_uint(fminf((top - capped(v)) * per_bin, kBins - 1) + 8388608.f) & (kBins - 1)); };
    constexpr int kEach = kBins / kThreads;
    // counts of all CTAs (complete behind a cluster.sync()), of this thread's intervals
    const auto gather = [&](auto (&c)[kEach]) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) c[j] = 0;
        for (int r = 0; r < ctas; ++r) {
            const uint4 v = *reinterpret_cast<const uint4 *>(&cluster.map_shared_rank(&s, r)->count[tid * kEach]);
            c[0] += v.x, c[1] += v.y, c[2] += v.z, c[3] += v.w;
        }
        static_assert(kEach == 4, "one 16-byte load");
    };
    // tokens of a group of eight that are listed, with the CTA that finishes the row
    const auto list = [&](unsigned in, const float (&v)[8], int i) {
        if (in == 0) return;
        int n = atomicAdd(&first.listed, __popc(in));
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (in >> j & 1) {
                if (n < kList) first.list[n] = place_of(v[j], i + j);
                ++n;
            }
    };

    if (use_k) {
        int lowest = kBins;                                      // the lowest interval that is listed (all, of a short row)
        bool weighty = false;                                    // or, instead, all that weighs anything
        if (V > kList) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (half_most[j] > -INFINITY) atomicAdd(&s.count[bin_of(half_most[j])], 1u);
            uint32_t c[kEach];
            cluster.sync();
            gather(c);
            int total, sum = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) sum += c[j];
            if (tid == 0) s.decided = kBins;
            int before = block_scan(sum, total, s.scan_n);
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                if (before < k && before + (int)c[j] >= k) s.decided = tid * kEach + j;
                before += c[j];
            }
            __syncthreads();
            lowest = s.decided;
            // Fewer than k maxima lie above the last interval, so tokens among the first k may lie in it, in the shadow of a neighbour that is a
            // maximum.  What weighs something does (what does not is never drawn, and takes no part in any sum).
            weighty = cut && lowest >= kBins - 1;
        }
        const auto listed = [&](float v) { return weighty ? weight_of.any(v) : v > -INFINITY && (lowest == kBins || bin_of(v) <= lowest); };
        const bool look = lowest == kBins || listed(half_most[0]) || listed(half_most[1]);
        if (look)
            for (int i = i0 + lane * 8; i < i1; i += kStep) {
                float v[8];
                load_eight(x, i, i1, a.wide, v);
                unsigned in = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) in |= (listed(v[j]) ? 1u : 0u) << j;
                list(in, v, i);
            }
        cluster.sync();
        if (rank != 0) return;
        const int n = s.listed;
        if (n > kList) {
            sample_slowly(a, s, x, row, top_key, weight_of);
            return;
        }
        sort_places(s.list, n);
        const int kept_k = n < k ? n : k;
        // weights of the first k, two consecutive ones per thread; all cuts keep a prefix
        double w[2], sum_w = 0.0, all;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * tid + j;
            w[j] = i < kept_k ? weight_of(value_of((uint32_t)(s.list[i] >> 32))) : 0.0;
            sum_w += w[j];
        }
        double before_w = block_scan(sum_w, all, s.scan);
        int kept = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * tid + j;
            if (i < kept_k && (i == 0 || !use_p || before_w < (double)p * all) && w[j] >= least && w[j] > 0.0) {
                ++kept;
                s.line[i] = w[j];
            }
            before_w += w[j];
        }
        int total_kept;
        block_scan(kept, total_kept, s.scan_n);
        __syncthreads();
        // in the order of the vocabulary: descending complement of the token, with the place in the sorted list
        for (int i = tid; i < total_kept; i += kThreads) s.list[i] = s.list[i] << 32 | (uint32_t)i;
        __syncthreads();
        sort_places(s.list, total_kept);
        sum_w = 0.0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * tid + j;
            w[j] = i < total_kept ? s.line[(uint32_t)s.list[i]] : 0.0;
            sum_w += w[j];
        }
        before_w = block_scan(sum_w, all, s.scan);
        const double aim = (double)a.uniforms[row] * all;
        if (tid == 0) s.found = total_kept - 1;                  // (rounding may leave no sum above the aim)
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * tid + j;
            before_w += w[j];
            if (i < total_kept && before_w > aim) atomicMin(&s.found, i);
        }
        __syncthreads();
        // (the largest weight, 1, always stays, so there is one)
        if (tid == 0) a.tokens[row] = (int64_t)(0xFFFFFFFFu - (uint32_t)(s.list[s.found] >> 32));
        return;
    }

    // ---- 2: the interval in which the nucleus about ends
    int edge = kBins, lowest_edge = 0, highest_edge = kBins - 1; // everything lies above it
    // A token counts with its weight in units of 2**-15 of that of its interval's middle: with 1 for each, a few large weights half an
    // interval from the middle, or the steps of a 16-bit type, let the guess miss by some intervals, a pass over the row each.  (Sums that
    // pass 32 bits, of a hundred thousand tokens in an interval, and all else that is rounded here cost a better guess, nothing more.)
    const float fall = per_bin > 0.f ? -1.442695f / (per_bin * t) : 0.f;
    // the interval in which the weights of all intervals, from the first on, add up to what aim_of(all) says; the sum before interval `at`
    const auto interval_of = [&](auto &&aim_of) {
        float c[kEach], w[kEach], sum = 0.f, total;
        gather(c);
#pragma unroll
        for (int j = 0; j < kEach; ++j) w[j] = c[j] * exp2f((tid * kEach + j) * fall - 15.f), sum += w[j];
        if (tid == 0) s.decided = kBins - 1;
        float before = block_scan(sum, total, s.low);
        if (tid == edge / kEach) {
            float from = before;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                if (j == edge % kEach) s.edge[0] = from, s.edge[1] = from + w[j];
                from += w[j];
            }
        }
        __syncthreads();
        const float aim = aim_of(total);
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            if (before + w[j] >= aim) atomicMin(&s.decided, tid * kEach + j);
            before += w[j];
        }
        __syncthreads();
        return s.decided;
    };
    if (use_p) {
        each_eight<4>(x, i0, i1, a.wide, [&](const float (&v)[8], int) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // (what lies behind the intervals, masked tokens not least, has no weight to speak of)
                const float behind = (top - v[j]) * per_bin;
                if (behind < kBins) {                            // (not NaN)
                    const float at = fminf(fmaxf(behind, 0.f), kBins - 1), middle = at + 8388608.f;
                    const float units = fmaf(exp2_fast((at - (middle - 8388608.f)) * fall), 32768.f, 8388608.f);
                    atomicAdd(&s.count[__float_as_uint(middle) & (kBins - 1)], __float_as_uint(units) & 0x7FFFFFu);
                }
            }
        });
        cluster.sync();
        // (every CTA finds the same from the same numbers in the same order)
        edge = interval_of([&](float total) { return p * total; });
    }

    // the smallest logit for which `is` holds, which then holds for all larger ones, by a search of the keys 32 at a time; NaN if for none
    const auto smallest = [&](auto &&is) {
        uint32_t lo = key_of(-FLT_MAX), hi = top_key + 1;       // (one of lo .. hi)
        while (lo < hi) {
            const uint32_t stride = (hi - lo) / 32 + 1, mid = lo + lane * stride;
            const unsigned holds = __ballot_sync(kFull, mid >= hi || is(value_of(mid)));
            if (holds == kFull) hi = lo;
            else if (holds == 0) lo += 31 * stride + 1;
            else {
                const uint32_t at = lo + (__ffs(holds) - 1) * stride;
                lo = at - stride + 1, hi = at < hi ? at : hi;
            }
        }
        return lo > top_key ? NAN : value_of(lo);
    };
    // (weights of neighbours differ by far more than the rounding)
    const float kept_from = least > 0.0 ? smallest([&](float v) { return weight_of(v) >= least; }) : -FLT_MAX;

    // ---- 3: what lies above the interval, per span, below it, and what lies in it
    uint64_t border = 0;                                         // the last place that stays
    for (int tries = 0;; ++tries) {
        // (intervals as logits: one comparison each instead of the interval's number)
        const float above_from = edge < kBins ? smallest([&](float v) { return bin_of(v) < edge; }) : -FLT_MAX;
        const float in_from = edge < kBins ? smallest([&](float v) { return bin_of(v) <= edge; }) : NAN;
        const float stays_from = kept_from > above_from ? kept_from : above_from;
        double above = 0.0, kept = 0.0, below = 0.0;
        // (one step at a time: two under way cost more registers than there are, 64 for two CTAs on an SM)
        each_eight<1>(x, i0, i1, a.wide, [&](const float (&v)[8], int i) {
            unsigned in = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double w = weight_of.of(v[j]);
                if (weight_of.any(v[j])) {
                    if (v[j] >= above_from) above += w;
                    else below += w;
                    if (v[j] >= stays_from) kept += w;
                }
                in |= (v[j] >= in_from && !(v[j] >= above_from) ? 1u : 0u) << j;
            }
            list(in, v, i);
        });
        above = warp_reduce(above, Plus()), kept = warp_reduce(kept, Plus());
        if (lane == 0) first.span_all[me] = above, first.span_kept[me] = kept;
        if (use_p) {
            below = block_reduce(below, Plus(), s.scan);
            if (tid == 0) s.cta_below = below;
        }
        cluster.sync();
        if (!use_p) break;
        if (rank == 0) {
            const int n = s.listed;
            int next = -1;                                       // -1: done, -2: the slow way, else: the interval to look at
            if (n > kList) {
                next = -2;
            } else {
                sort_places(s.list, n);
                double over = 0.0, rest = 0.0, total, running = 0.0;     // (rest: in the interval and below it)
                over = block_reduce(tid < spans ? s.span_all[tid] : 0.0, Plus(), s.scan);
                for (int r = 0; r < ctas; ++r) rest += cluster.map_shared_rank(&s, r)->cta_below;
                // eight consecutive places per thread
                constexpr int kPlaces = kList / kThreads;
                double sum = 0.0;
                for (int j = 0; j < kPlaces; ++j) {
                    const int i = tid * kPlaces + j;
                    if (i < n) sum += weight_of(value_of((uint32_t)(s.list[i] >> 32)));
                }
                running = over + block_scan(sum, total, s.scan);
                const double aim = (double)p * (over + rest);
                const bool early = over >= aim && edge > 0, late = !early && over + total < aim && edge < kBins - 1;
                if (early || late) {
                    // the guess again, from where the exact sums are known
                    if (early) highest_edge = edge - 1;
                    else lowest_edge = edge + 1;
                    next = interval_of([&](float) { return early ? s.edge[0] - (float)(over - aim) : s.edge[1] + (float)(aim - (over + total)); });
                    next = max(lowest_edge, min(next, highest_edge));
                    if (tries == 6 || lowest_edge > highest_edge) next = -2;
                } else {
                    int inside = 0, total_inside;
                    for (int j = 0; j < kPlaces; ++j) {
                        const int i = tid * kPlaces + j;
                        if (i >= n) break;
                        inside += running < aim || (edge == 0 && i == 0);       // (the very first always stays)
                        running += weight_of(value_of((uint32_t)(s.list[i] >> 32)));
                    }
                    block_scan(inside, total_inside, s.scan_n);
                    if (tid == 0) s.border = total_inside > 0 ? s.list[total_inside - 1] : 1;
                    // the weights that stay count in their spans, in a fixed order: a warp each
                    uint8_t *span_of = reinterpret_cast<uint8_t *>(s.count);
                    for (int i = tid; i < total_inside; i += kThreads) span_of[i] = (uint8_t)(token_of(s.list[i]) / span);
                    __syncthreads();
                    for (int sp = warp; sp < spans; sp += kWarps) {
                        double more = 0.0;
                        for (int i = lane; i < total_inside; i += 32)
                            if (span_of[i] == sp) {
                                const double w = weight_of(value_of((uint32_t)(s.list[i] >> 32)));
                                if (w >= least) more += w;
                            }
                        more = warp_reduce(more, Plus());
                        if (lane == 0) s.span_kept[sp] += more;
                    }
                }
            }
            __syncthreads();
            if (tid == 0) s.listed = 0, s.decided = next;
        }
        cluster.sync();
        const int next = first.decided;
        border = first.border;
        cluster.sync();
        if (next == -2) {
            if (rank == 0) sample_slowly(a, s, x, row, top_key, weight_of);
            return;
        }
        if (next == -1) break;
        edge = next;
    }
    if (rank != 0) return;

    // ---- the span in which the draw falls, a step of it per warp, and then the step
    __syncthreads();
    double total;
    const double mine = tid < spans ? s.span_kept[tid] : 0.0, before = block_scan(mine, total, s.scan);
    const double aim = (double)a.uniforms[row] * total;
    // the first part that has a weight and ends above the aim; rounding may leave none, then the last that has one
    const auto first_above = [&](bool any, bool over, int i) {
        if (tid == 0) s.found = INT32_MAX, s.decided = -1;
        __syncthreads();
        if (any) atomicMax(&s.decided, i);
        if (any && over) atomicMin(&s.found, i);
        __syncthreads();
        const int r = s.found == INT32_MAX ? s.decided : s.found;
        __syncthreads();
        return r;
    };
    const int chosen = first_above(mine > 0.0, before + mine > aim, tid);
    if (tid == chosen) s.scan[kWarps] = before;
    const int j0 = chosen * span, j1 = min(j0 + span, V);
    double from = 0.0;
    // (the eight weights of a lane, those that stay)
    const auto weights_at = [&](int i, double (&w)[8], int &last) {
        float v[8];
        load_eight(x, i, j1, a.wide, v);
        double sum = 0.0;
        last = -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = v[j] > -INFINITY && place_of(v[j], i + j) >= border ? weight_of(v[j]) : 0.0;
            if (w[j] < least) w[j] = 0.0;
            if (w[j] > 0.0) last = i + j;
            sum += w[j];
        }
        return sum;
    };
    // the step of the span: sums of sixteen steps at a time, the last of which has what rounding leaves over
    int step = -1;
    double step_from = 0.0;
    __syncthreads();
    from = s.scan[kWarps];
    for (int s0 = j0; s0 < j1; s0 += kWarps * kStep) {
        double w[8];
        int last;
        const double sum = warp_reduce(weights_at(s0 + warp * kStep + lane * 8, w, last), Plus());
        __syncthreads();
        if (lane == 0) s.span_all[warp] = sum;
        __syncthreads();
        bool over = false;
        for (int i = 0; i < kWarps && !over; ++i)
            if (s.span_all[i] > 0.0) {
                step = s0 + i * kStep, step_from = from;
                over = from + s.span_all[i] > aim;
                from += s.span_all[i];
            }
        if (over) break;
    }
    if (warp != 0) return;
    double w[8];
    int last;
    const double sum = weights_at(step + lane * 8, w, last);
    double incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double u = __shfl_up_sync(kFull, incl, d);
        if (lane >= d) incl += u;
    }
    const unsigned over = __ballot_sync(kFull, sum > 0.0 && step_from + incl > aim), any = __ballot_sync(kFull, sum > 0.0);
    const int who = over ? __ffs(over) - 1 : 31 - __clz(any);
    if (lane == who) {
        double f = step_from + (incl - sum);
        int token = last;
#pragma unroll
        for (int j = 7; j >= 0; --j) f += w[j];
        // (backwards: the first that ends above the aim)
#pragma unroll
        for (int j = 7; j >= 0; --j) {
            if (w[j] > 0.0 && f > aim) token = step + lane * 8 + j;
            f -= w[j];
        }
        a.tokens[row] = token;
    }
}

template <typename T>
cudaError_t launch(const SampleArgs &a, int B, int ctas, cudaStream_t st) {
    static_assert(sizeof(Shared) <= 64 * 1024, "three CTAs per SM");
    // the kernel's limit of dynamic shared memory is raised once per device
    static std::atomic<bool> done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(k_sample<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)B * ctas), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = sizeof(Shared), cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k_sample<T>, a);
}

}  // namespace

extern "C" int adacode_sample_tokens(const void *logits, int64_t row_stride, int dtype, int B, int V, const float *uniforms,
                                     const float *temperature, float temperature_all, const int32_t *top_k, int top_k_all, const float *top_p,
                                     float top_p_all, const float *min_p, float min_p_all, int64_t *tokens, void *stream) {
    if (B < 0 || V <= 0 || (B > 0 && (!logits || !uniforms || !tokens))) return ADACODE_ERR_INVALID_ARG;
    if (dtype != ADACODE_BF16 && dtype != ADACODE_FP16 && dtype != ADACODE_FP32) return ADACODE_ERR_INVALID_ARG;
    if (V > 1 << 30 || B > 1 << 27) return ADACODE_ERR_TOO_LARGE;
    if (B == 0) return ADACODE_OK;
    const int size = dtype == ADACODE_FP32 ? 4 : 2;
    const bool wide = ((uintptr_t)logits & 15) == 0 && (row_stride * size) % 16 == 0;
    const SampleArgs a{logits, row_stride, V, wide, uniforms, temperature, top_p, min_p, top_k, tokens, temperature_all, top_p_all, min_p_all, top_k_all};
    // CTAs per row: up to four, as long as all rows' make no more than three for each of 148 SMs (two fit at a time; more rounds than that only add
    // the rows' ends) and every warp has a step of the vocabulary; eight if every CTA then has an SM of its own and every warp two steps.  192 rows of
    // 151936: 218 us with one, 159 with two, 193 with four (then; 150 with two now); 64 rows of 128256: 34, 22, 21.5 and 37 with eight; one row of
    // 32000: 16, 12.6, 11 and 11.2; one row of 262144 with top_p 54 with four and 39 with eight, 32 rows of 32000 with top_k 11 and 16.5.
    int ctas = 1;
    while (ctas < kMostCtas && (int64_t)B * ctas * 2 <= (ctas < 4 ? 3 * 148 : 148) && V > ctas * kWarps * kStep * (ctas < 4 ? 1 : 2)) ctas *= 2;
    cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = dtype == ADACODE_BF16 ? launch<__nv_bfloat16>(a, B, ctas, st)
                          : dtype == ADACODE_FP16 ? launch<__half>(a, B, ctas, st)
                                                  : launch<float>(a, B, ctas, st);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return ADACODE_ERR_CUDA;
    }
    return ADACODE_OK;
}
