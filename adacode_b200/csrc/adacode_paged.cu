// New tokens of a serving step on their way into a paged cache: rotation and append.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "adacode.h"

namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;

#include "adacode_pages.cuh"

// ---------------------------------------------------------------------------------------
// rotation and append
// ---------------------------------------------------------------------------------------

struct AppendArgs {
    adacode_paged_cache cache;
    adacode_rotary rotary;
    const void *query, *key, *value;
    void *query_out;
    long long q_n, q_h, o_n, o_h, k_n, k_h, v_n, v_h;
    int Hq;
    int32_t *status;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Chunk {
    T v[V];
};

// A CTA has one token; a thread one pair of V-column chunks of every so manieth head, whose angles it keeps: bound by memory, and by
// latency where tokens are few.  The chunks of a pair are rotated against each other (half-split), lie side by side (interleaved), or
// are copied (columns that are not rotated, and values).
template <typename T, typename A, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(256) k_append_rotary(const __grid_constant__ AppendArgs a) {
    const adacode_paged_cache &c = a.cache;
    const adacode_rotary &r = a.rotary;
    const int i = blockIdx.x, pairs = c.D / (2 * V), pair = threadIdx.x % pairs, first = threadIdx.x / pairs, step = blockDim.x / pairs;
    int end = 0, slot = 0;
    const int b = sequence_of(c, i, end);
    if (b >= c.B) return;
    const int at = c.seq_lens[b] - end + i, page = page_of(c, b, at, slot);
    if (page < 0 && threadIdx.x == 0) atomicOr(a.status, ADACODE_STATUS_BAD_PAGE);
    const bool turned = pair * V < r.half;
    const int lo = INTERLEAVED || !turned ? pair * 2 * V : pair * V;
    const int hi = INTERLEAVED || !turned ? lo + V : r.half + pair * V;
    float cs[V], sn[V];
#pragma unroll
    for (int j = 0; j < V; ++j) cs[j] = 1.f, sn[j] = 0.f;
    if (turned) {
        const A *cos = reinterpret_cast<const A *>(r.cos) + i * r.token_stride, *sin = reinterpret_cast<const A *>(r.sin) + i * r.token_stride;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int f = pair * V + j;
            int axis = 0, upto = r.section[0];
            while (axis + 1 < r.axes && f >= upto) upto += r.section[++axis];
            cs[j] = widen(cos[axis * r.axis_stride + f]), sn[j] = widen(sin[axis * r.axis_stride + f]);
        }
    }
    const int rotated = a.Hq + c.Hkv, heads = rotated + c.Hkv;
    for (int h = first; h < heads; h += step) {
        const T *src;
        T *dst;
        if (h < a.Hq) {
            src = reinterpret_cast<const T *>(a.query) + i * a.q_n + h * a.q_h;
            dst = reinterpret_cast<T *>(a.query_out) + i * a.o_n + h * a.o_h;
        } else if (page < 0) {
            break;
        } else if (h < rotated) {
            src = reinterpret_cast<const T *>(a.key) + i * a.k_n + (h - a.Hq) * a.k_h;
            dst = reinterpret_cast<T *>(c.key_pages) + page * c.key_page + (h - a.Hq) * c.key_head + slot * c.key_slot;
        } else {
            src = reinterpret_cast<const T *>(a.value) + i * a.v_n + (h - rotated) * a.v_h;
            dst = reinterpret_cast<T *>(c.value_pages) + page * c.value_page + (h - rotated) * c.value_head + slot * c.value_slot;
        }
        const Chunk<T, V> x = *reinterpret_cast<const Chunk<T, V> *>(src + lo), y = *reinterpret_cast<const Chunk<T, V> *>(src + hi);
        Chunk<T, V> u = x, v = y;
        if (turned && h < rotated) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (INTERLEAVED) {
                    const T *from = 2 * j < V ? x.v : y.v;
                    T *to = 2 * j < V ? u.v : v.v;
                    const int e = 2 * j % V;
                    if constexpr (V > 1) {
                        const float p = widen(from[e]), q = widen(from[e + 1]);
                        to[e] = narrow<T>(p * cs[j] - q * sn[j]), to[e + 1] = narrow<T>(q * cs[j] + p * sn[j]);
                    } else {
                        const float p = widen(x.v[0]), q = widen(y.v[0]);
                        u.v[0] = narrow<T>(p * cs[0] - q * sn[0]), v.v[0] = narrow<T>(q * cs[0] + p * sn[0]);
                    }
                } else {
                    const float p = widen(x.v[j]), q = widen(y.v[j]);
                    u.v[j] = narrow<T>(p * cs[j] - q * sn[j]), v.v[j] = narrow<T>(q * cs[j] + p * sn[j]);
                }
            }
        }
        *reinterpret_cast<Chunk<T, V> *>(dst + lo) = u;
        *reinterpret_cast<Chunk<T, V> *>(dst + hi) = v;
    }
}

template <typename T, typename A, int V>
void launch_append(const AppendArgs &a, cudaStream_t st) {
    const int pairs = a.cache.D / (2 * V);
    const int threads = pairs * (pairs < 256 ? 256 / pairs : 1);
    if (a.rotary.interleaved) k_append_rotary<T, A, V, true><<<a.cache.N, threads, 0, st>>>(a);
    else k_append_rotary<T, A, V, false><<<a.cache.N, threads, 0, st>>>(a);
}

template <typename T, typename A>
void launch_append(const AppendArgs &a, bool wide, cudaStream_t st) {
    if (wide) launch_append<T, A, 8>(a, st);
    else launch_append<T, A, 1>(a, st);
}

template <typename T>
void launch_append(const AppendArgs &a, bool wide, cudaStream_t st) {
    if (a.rotary.dtype == ADACODE_FP32) launch_append<T, float>(a, wide, st);
    else launch_append<T, T>(a, wide, st);
}

}  // namespace

extern "C" {

int adacode_append_rotary(const adacode_paged_cache *cache, const adacode_rotary *rotary, const void *query, int64_t query_token,
                          int64_t query_head, int Hq, void *query_out, int64_t out_token, int64_t out_head, const void *key,
                          int64_t key_token, int64_t key_head, const void *value, int64_t value_token, int64_t value_head,
                          int32_t *status, void *stream) {
    if (!valid(cache) || !rotary || !status || !key || !value || Hq < 0 || (Hq > 0 && (!query || !query_out))) return ADACODE_ERR_INVALID_ARG;
    const adacode_rotary &r = *rotary;
    if (cache->D <= 0 || cache->D % 2 != 0 || cache->D > 512 || r.half < 0 || 2 * r.half > cache->D || r.axes < 1 || r.axes > 4)
        return ADACODE_ERR_INVALID_ARG;
    if (r.half > 0 && (!r.cos || !r.sin)) return ADACODE_ERR_INVALID_ARG;
    if (r.dtype != ADACODE_FP32 && r.dtype != cache->dtype) return ADACODE_ERR_INVALID_ARG;
    int columns = 0;
    for (int x = 0; x < r.axes; ++x) {
        if (r.section[x] < 0) return ADACODE_ERR_INVALID_ARG;
        columns += r.section[x];
    }
    if (columns != r.half) return ADACODE_ERR_INVALID_ARG;
    if (cache->N == 0) return ADACODE_OK;
    const AppendArgs a{*cache,    r,       query,    key,       value,   query_out, query_token, query_head,
                       out_token, out_head, key_token, key_head, value_token, value_head, Hq,        status};
    // sixteen bytes at a time where everything allows it
    const uintptr_t pointers = (uintptr_t)query | (uintptr_t)query_out | (uintptr_t)key | (uintptr_t)value | (uintptr_t)cache->key_pages |
                               (uintptr_t)cache->value_pages;
    const int64_t strides = query_token | query_head | out_token | out_head | key_token | key_head | value_token | value_head | cache->key_page |
                            cache->key_head | cache->key_slot | cache->value_page | cache->value_head | cache->value_slot;
    const bool wide = (pointers & 15) == 0 && (strides & 7) == 0 && cache->D % 16 == 0 && r.half % 8 == 0;
    if (cache->dtype == ADACODE_BF16) launch_append<__nv_bfloat16>(a, wide, (cudaStream_t)stream);
    else launch_append<__half>(a, wide, (cudaStream_t)stream);
    return cudaGetLastError() == cudaSuccess ? ADACODE_OK : ADACODE_ERR_CUDA;
}

}  // extern "C"
