// New tokens of a serving step and their paged cache: rotation and append, attention over the pages.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "adacode.h"

namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }

// Sequence of new token i (B if it is behind the last), found by the whole warp, and the tokens of the call up to its end.
__device__ __forceinline__ int sequence_of(const adacode_paged_cache &c, int i, int &end) {
    if (!c.cu_seqlens) {
        const int each = c.N / c.B, b = i / each;
        end = (b + 1) * each;
        return b;
    }
    const int lane = threadIdx.x & 31;
    int b = 0;
    for (int k = 0; k < c.B; k += 32) {
        const int e = k + lane < c.B ? c.cu_seqlens[k + lane + 1] : INT32_MAX;
        const unsigned before = __ballot_sync(kFull, e <= i);
        b += __popc(before);
        if (before != kFull) {
            end = __shfl_sync(kFull, e, __popc(before));
            break;
        }
    }
    return b;
}

// The page of position `at` of sequence b, or -1.
__device__ __forceinline__ int page_of(const adacode_paged_cache &c, int b, int at, int &slot) {
    const int n = at / c.page_size;
    slot = at - n * c.page_size;
    if (at < 0 || n >= c.table_width) return -1;
    const int page = c.block_table[b * c.table_stride + n];
    return page >= 0 && page < c.n_pages ? page : -1;
}

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

bool valid(const adacode_paged_cache *c) {
    return c && c->key_pages && c->value_pages && c->block_table && c->seq_lens && c->B > 0 && c->n_pages > 0 && c->page_size > 0 &&
           c->table_width > 0 && c->Hkv > 0 && c->N >= 0 && (c->dtype == ADACODE_BF16 || c->dtype == ADACODE_FP16) &&
           (c->cu_seqlens || c->N % c->B == 0);
}

// ---------------------------------------------------------------------------------------
// attention over pages
// ---------------------------------------------------------------------------------------

constexpr float kLog2e = 1.4426950408889634f;

struct PagedArgs {
    adacode_paged_cache cache;
    const void *query;
    void *out;
    long long q_n, q_h, o_n, o_h;
    const int32_t *starts;
    int Hq, G, causal, window;
    float scale;              // times log2 e
    int32_t *status;
};

// One warp per token and head, one cached token after the other.  A value whose weight is 0 has no influence.
template <typename T, int D>
__global__ void __launch_bounds__(128) k_paged_rows(const __grid_constant__ PagedArgs a) {
    constexpr int E = D / 32;
    const adacode_paged_cache &c = a.cache;
    const int lane = threadIdx.x & 31;
    const long long w = blockIdx.x * 4ll + threadIdx.x / 32;
    const int i = (int)(w / a.Hq), h = (int)(w - (long long)i * a.Hq);
    if (i >= c.N) return;
    int end = 0;
    const int b = sequence_of(c, i, end);
    if (b >= c.B) return;
    const int len = c.seq_lens[b], at = len - end + i;
    int lo = a.starts ? a.starts[b] : 0, hi = a.causal && at + 1 < len ? at + 1 : len;
    if (a.window > 0 && lo < at - a.window + 1) lo = at - a.window + 1;
    if (lo < 0) lo = 0;
    const T *q = reinterpret_cast<const T *>(a.query) + i * a.q_n + h * a.q_h + lane * E;
    float x[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = widen(q[e]) * a.scale, acc[e] = 0.f;
    // twice over the tokens: the weights' sum first, so that values are added up with weights below 1 and large ones do not overflow
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        const float base = m == -INFINITY ? 0.f : m, share = pass ? 1.f / l : 0.f;
        for (int j = lo; j < hi; ++j) {
            int slot;
            const int page = page_of(c, b, j, slot);
            if (page < 0) {
                if (lane == 0) atomicOr(a.status, ADACODE_STATUS_BAD_PAGE);
                continue;
            }
            const T *k = reinterpret_cast<const T *>(c.key_pages) + page * c.key_page + (h / a.G) * c.key_head + slot * c.key_slot + lane * E;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) s = fmaf(x[e], widen(k[e]), s);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(kFull, s, d);
            if (pass == 0) {
                const float top = fmaxf(m, s), from = top == -INFINITY ? 0.f : top;
                l = l * exp2f(m - from) + exp2f(s - from);
                m = top;
                continue;
            }
            const float p = exp2f(s - base) * share;
            if (p == 0.f) continue;
            const T *v = reinterpret_cast<const T *>(c.value_pages) + page * c.value_page + (h / a.G) * c.value_head + slot * c.value_slot + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(p, widen(v[e]), acc[e]);
        }
        if (l == 0.f) break;
    }
    T *out = reinterpret_cast<T *>(a.out) + i * a.o_n + h * a.o_h + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = narrow<T>(l == 0.f ? 0.f : acc[e]);
}

template <typename T>
void launch_paged(const PagedArgs &a, cudaStream_t st) {
    const unsigned grid = (unsigned)(((long long)a.cache.N * a.Hq + 3) / 4);
    if (a.cache.D == 128) k_paged_rows<T, 128><<<grid, 128, 0, st>>>(a);
    else k_paged_rows<T, 64><<<grid, 128, 0, st>>>(a);
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

size_t adacode_paged_attn_workspace_bytes(int D) { return D > 0 ? 16 : 0; }

int adacode_paged_attn(const adacode_paged_cache *cache, const void *query, int64_t query_token, int64_t query_head, int Hq,
                       void *out, int64_t out_token, int64_t out_head, const int32_t *seq_starts, int max_query_len, float scale, int causal,
                       int window, void *workspace, size_t workspace_bytes, int32_t *status, void *stream) {
    if (!valid(cache) || !status || Hq <= 0 || Hq % cache->Hkv != 0 || window < 0 || max_query_len < 0) return ADACODE_ERR_INVALID_ARG;
    if (cache->D != 64 && cache->D != 128) return ADACODE_ERR_INVALID_ARG;
    if (cache->table_width > 1 && cache->page_size % 128 != 0 && cache->page_size != 16 && cache->page_size != 32 && cache->page_size != 64)
        return ADACODE_ERR_INVALID_ARG;
    if (cache->N == 0) return ADACODE_OK;
    if (!query || !out) return ADACODE_ERR_INVALID_ARG;
    const uintptr_t pointers = (uintptr_t)query | (uintptr_t)out | (uintptr_t)cache->key_pages | (uintptr_t)cache->value_pages;
    const int64_t strides = query_token | query_head | out_token | out_head | cache->key_page | cache->key_head | cache->key_slot |
                            cache->value_page | cache->value_head | cache->value_slot;
    if ((pointers & 15) != 0 || (strides & 7) != 0) return ADACODE_ERR_INVALID_ARG;
    const PagedArgs a{*cache, query, out, query_token, query_head, out_token, out_head, seq_starts, Hq, Hq / cache->Hkv, causal, window, scale * kLog2e, status};
    if (cache->dtype == ADACODE_BF16) launch_paged<__nv_bfloat16>(a, (cudaStream_t)stream);
    else launch_paged<__half>(a, (cudaStream_t)stream);
    return cudaGetLastError() == cudaSuccess ? ADACODE_OK : ADACODE_ERR_CUDA;
}

}  // extern "C"
