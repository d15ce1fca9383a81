// One token per row of logits: temperature, top-k, top-p, min-p and the draw from a given uniform number.
//
// Logits become 32-bit keys whose order is the logits' order.  Every cut (the top_k first, the nucleus) is a prefix of the
// order (descending logit, ascending token) and is kept as a key and the number of that key's tokens that are inside.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "adacode.h"

namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr int kThreads = 1024;

struct SampleArgs {
    const void *logits;
    long long row_stride;
    int V;
    const float *uniforms, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int64_t *tokens;
};

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen(float v) { return v; }
template <>
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// NaN and minus infinity have key 0 (never drawn), plus infinity that of the largest finite number, both zeros one key.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0;
    x = fminf(x, FLT_MAX) + 0.f;
    const uint32_t u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key); }

template <typename R, typename Op>
__device__ R block_reduce(R v, Op op, R *shared) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = op(v, __shfl_xor_sync(kFull, v, d));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    R r = shared[0];
    for (int w = 1; w < kThreads / 32; ++w) r = op(r, shared[w]);
    return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample(const SampleArgs a) {
    __shared__ double s_d[32];
    __shared__ unsigned long long s_u[32];
    __shared__ double s_line[kThreads];
    __shared__ int s_ties[kThreads];
    const int row = blockIdx.x, tid = threadIdx.x, V = a.V;
    const T *x = reinterpret_cast<const T *>(a.logits) + row * a.row_stride;
    const auto plus = [](auto p, auto q) { return p + q; };
    const auto most = [](auto p, auto q) { return p > q ? p : q; };
    // largest key, and the first token that has it
    unsigned long long best = 0;
    for (int i = tid; i < V; i += kThreads) best = most(best, (unsigned long long)key_of(widen(x[i])) << 32 | (0xFFFFFFFFu - (uint32_t)i));
    best = block_reduce(best, most, s_u);
    const uint32_t top = (uint32_t)(best >> 32);
    const float t = a.temperature[row];
    if (top == 0 || !(t > 0.f)) {
        if (tid == 0) a.tokens[row] = top == 0 ? -1 : (int64_t)(0xFFFFFFFFu - (uint32_t)best);
        return;
    }
    const double largest = value_of(top), temperature = t;
    const auto weight = [&](uint32_t key) { return key == 0 ? 0.0 : exp(((double)value_of(key) - largest) / temperature); };
    // the cut: tokens of keys above `cut`, and the first `ties` tokens of key `cut`
    uint32_t cut = 1;
    long long ties = V;
    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < V) {
        // the largest key that at least k tokens reach
        uint32_t lo = 1, hi = top;
        long long above = 0;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            unsigned long long n = 0;
            for (int i = tid; i < V; i += kThreads) n += key_of(widen(x[i])) >= mid;
            n = block_reduce(n, plus, s_u);
            if ((long long)n >= k) lo = mid;
            else hi = mid - 1, above = (long long)n;
        }
        cut = lo;
        ties = k - above;
    }
    const float p = a.top_p ? a.top_p[row] : 1.f;
    if (p < 1.f) {
        const auto total = [&](uint32_t from) {           // weight of the tokens of keys from `from` on, inside the cut
            double w = 0.0;
            for (int i = tid; i < V; i += kThreads) {
                const uint32_t key = key_of(widen(x[i]));
                if (key >= from && key > cut) w += weight(key);
            }
            w = block_reduce(w, plus, s_d);
            if (from <= cut) {
                unsigned long long n = 0;
                for (int i = tid; i < V; i += kThreads) n += key_of(widen(x[i])) == cut;
                n = block_reduce(n, plus, s_u);
                if (n > 0) w += (double)((long long)n < ties ? (long long)n : ties) * weight(cut);   // (no token has a NaN's key)
            }
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
    const double least = a.min_p ? (double)a.min_p[row] : 0.0;
    // runs of consecutive tokens per thread: ties before it, weight before it, the token
    const int per = (V + kThreads - 1) / kThreads, i0 = min(tid * per, V), i1 = min(i0 + per, V);
    int same = 0;
    for (int i = i0; i < i1; ++i) same += key_of(widen(x[i])) == cut;
    s_ties[tid] = same;
    __syncthreads();
    long long before = 0;
    for (int j = 0; j < tid; ++j) before += s_ties[j];
    const auto walk = [&](double from, double aim, int &found) {
        long long n = before;
        for (int i = i0; i < i1; ++i) {
            const uint32_t key = key_of(widen(x[i]));
            if (key == 0 || key < cut || (key == cut && n++ >= ties)) continue;
            const double w = weight(key);
            if (w < least || w == 0.0) continue;
            from += w;
            if (from > aim) {
                found = i;
                return from;
            }
        }
        return from;
    };
    int found = -1;
    s_line[tid] = walk(0.0, INFINITY, found);
    __syncthreads();
    double from = 0.0, all = 0.0;
    for (int j = 0; j < kThreads; ++j) {
        if (j == tid) from = all;
        all += s_line[j];
    }
    const double aim = (double)a.uniforms[row] * all;
    if (s_line[tid] > 0.0 && from <= aim && from + s_line[tid] > aim) {
        walk(from, aim, found);
        if (found >= 0) a.tokens[row] = found;
    }
}

}  // namespace

extern "C" int adacode_sample_tokens(const void *logits, int64_t row_stride, int dtype, int B, int V, const float *uniforms,
                                     const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                                     int64_t *tokens, void *stream) {
    if (B < 0 || V <= 0 || (B > 0 && (!logits || !uniforms || !temperature || !tokens))) return ADACODE_ERR_INVALID_ARG;
    if (B == 0) return ADACODE_OK;
    const SampleArgs a{logits, row_stride, V, uniforms, temperature, top_p, min_p, top_k, tokens};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == ADACODE_BF16) k_sample<__nv_bfloat16><<<B, kThreads, 0, st>>>(a);
    else if (dtype == ADACODE_FP16) k_sample<__half><<<B, kThreads, 0, st>>>(a);
    else if (dtype == ADACODE_FP32) k_sample<float><<<B, kThreads, 0, st>>>(a);
    else return ADACODE_ERR_INVALID_ARG;
    return cudaGetLastError() == cudaSuccess ? ADACODE_OK : ADACODE_ERR_CUDA;
}
