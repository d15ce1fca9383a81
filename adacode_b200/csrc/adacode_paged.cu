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
    bool whole_angles;        // of one axis, on 16-byte boundaries
    int group;
};

template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Chunk {
    T v[V];
};

// `group` threads (whole warps) have one token; a thread one pair of V-column chunks of every so manieth head, whose angles it keeps.  The chunks
// of a pair are rotated against each other (half-split), lie side by side (interleaved), or are copied (columns that are not rotated, and
// values).  Bound by memory where tokens are many (13 854 tokens of 48 heads of 128 move 348 MB in 60 us, 5.8 TB/s; that takes four CTAs on an
// SM, so 64 registers: with the next head's loads on their way early it is three and 68 us, with two more heads 82 to 159), by the
// latency of finding a token's page where they are few.
template <typename T, typename A, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 4) k_append_rotary(const __grid_constant__ AppendArgs a) {
    const adacode_paged_cache &c = a.cache;
    const adacode_rotary &r = a.rotary;
    const int tid = threadIdx.x % a.group, i = blockIdx.x * (blockDim.x / a.group) + threadIdx.x / a.group;
    const int pairs = c.D / (2 * V), pair = tid % pairs, first = tid / pairs, step = a.group / pairs;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (i >= c.N) return;
    const int rotated = a.Hq + c.Hkv, heads = first < step ? rotated + c.Hkv : 0;      // (threads behind the last whole set of pairs have none)
    const bool turned = pair * V < r.half;
    const int lo = INTERLEAVED || !turned ? pair * 2 * V : pair * V;
    const int hi = INTERLEAVED || !turned ? lo + V : r.half + pair * V;
    const auto load = [&](int h, Chunk<T, V> &x, Chunk<T, V> &y) {
        const T *src = h < a.Hq     ? reinterpret_cast<const T *>(a.query) + i * a.q_n + h * a.q_h
                       : h < rotated ? reinterpret_cast<const T *>(a.key) + i * a.k_n + (h - a.Hq) * a.k_h
                                     : reinterpret_cast<const T *>(a.value) + i * a.v_n + (h - rotated) * a.v_h;
        x = *reinterpret_cast<const Chunk<T, V> *>(src + lo), y = *reinterpret_cast<const Chunk<T, V> *>(src + hi);
    };
    Chunk<T, V> x, y;
    float cs[V], sn[V];
#pragma unroll
    for (int j = 0; j < V; ++j) cs[j] = 1.f, sn[j] = 0.f;
    if (turned && heads) {
        const A *cos = reinterpret_cast<const A *>(r.cos) + i * r.token_stride, *sin = reinterpret_cast<const A *>(r.sin) + i * r.token_stride;
        if (V > 1 && a.whole_angles) {
            const Chunk<A, V> p = *reinterpret_cast<const Chunk<A, V> *>(cos + pair * V), q = *reinterpret_cast<const Chunk<A, V> *>(sin + pair * V);
#pragma unroll
            for (int j = 0; j < V; ++j) cs[j] = widen(p.v[j]), sn[j] = widen(q.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int f = pair * V + j;
                int axis = 0, upto = r.section[0];
                while (axis + 1 < r.axes && f >= upto) upto += r.section[++axis];
                cs[j] = widen(cos[axis * r.axis_stride + f]), sn[j] = widen(sin[axis * r.axis_stride + f]);
            }
        }
    }
    int end = 0, slot = 0;
    const int b = sequence_of(c, i, end);
    if (b >= c.B) return;
    const int at = c.seq_lens[b] - end + i, page = page_of(c, b, at, slot);
    if (page < 0 && tid == 0) atomicOr(a.status, ADACODE_STATUS_BAD_PAGE);
    for (int h = first; h < heads; h += step) {
        load(h, x, y);
        Chunk<T, V> u = x, v = y;
        if (turned && h < rotated) {
            const Chunk<T, V> p = u, q = v;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // column j of the chunks, or columns 2 j and 2 j + 1 of the two together
                const float s = widen(INTERLEAVED && V > 1 ? (2 * j < V ? p : q).v[2 * j % V] : p.v[j]);
                const float t = widen(INTERLEAVED && V > 1 ? (2 * j < V ? p : q).v[(2 * j + 1) % V] : q.v[j]);
                const T first_of = narrow<T>(s * cs[j] - t * sn[j]), second_of = narrow<T>(t * cs[j] + s * sn[j]);
                if constexpr (INTERLEAVED && V > 1) {
                    (2 * j < V ? u : v).v[2 * j % V] = first_of;
                    (2 * j < V ? u : v).v[(2 * j + 1) % V] = second_of;
                } else {
                    u.v[j] = first_of, v.v[j] = second_of;
                }
            }
        }
        if (h >= a.Hq && page < 0) continue;
        T *dst = h < a.Hq     ? reinterpret_cast<T *>(a.query_out) + i * a.o_n + h * a.o_h
                 : h < rotated ? reinterpret_cast<T *>(c.key_pages) + page * c.key_page + (h - a.Hq) * c.key_head + slot * c.key_slot
                               : reinterpret_cast<T *>(c.value_pages) + page * c.value_page + (h - rotated) * c.value_head + slot * c.value_slot;
        *reinterpret_cast<Chunk<T, V> *>(dst + lo) = u;
        *reinterpret_cast<Chunk<T, V> *>(dst + hi) = v;
    }
}

template <typename T, typename A, int V>
cudaError_t launch_append(AppendArgs &a, cudaStream_t st) {
    // Threads per token: eight warps where tokens are few, down to one where they fill half of the GPU's threads that way.  32 tokens of 48 heads
    // of 128: 2.9 us with eight, 8.2 with one; 3090 tokens of 20 heads: 24.8 and 8.1; 13 854 tokens of 48 heads: 108 and 60.
    const int pairs = a.cache.D / (2 * V);
    a.group = 256;
    while (a.group > 32 && a.group / 2 >= pairs && (int64_t)a.cache.N * a.group > 148 * 1024) a.group /= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((int64_t)a.cache.N * a.group + 255) / 256)), cfg.blockDim = dim3(256), cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return a.rotary.interleaved ? cudaLaunchKernelEx(&cfg, k_append_rotary<T, A, V, true>, a) : cudaLaunchKernelEx(&cfg, k_append_rotary<T, A, V, false>, a);
}

template <typename T>
cudaError_t launch_append(AppendArgs &a, bool wide, cudaStream_t st) {
    if (a.rotary.dtype == ADACODE_FP32) return wide ? launch_append<T, float, 8>(a, st) : launch_append<T, float, 1>(a, st);
    return wide ? launch_append<T, T, 8>(a, st) : launch_append<T, T, 1>(a, st);
}

}  // namespace

extern "C" {

int adacode_append_rotary(const adacode_paged_cache *cache, const adacode_rotary *rotary, const void *query, int64_t query_token,
                          int64_t query_head, int Hq, void *query_out, int64_t out_token, int64_t out_head, const void *key,
                          int64_t key_token, int64_t key_head, const void *value, int64_t value_token, int64_t value_head,
                          int32_t *status, void *stream) {
    if (!valid(cache) || !rotary || !status || !key || !value || Hq < 0 || (Hq > 0 && (!query || !query_out))) return ADACODE_ERR_INVALID_ARG;
    const adacode_rotary &r = *rotary;
    const adacode_paged_cache given = used_strides(*cache);
    cache = &given;
    if (cache->N == 1) query_token = out_token = key_token = value_token = 0;
    if (Hq == 1) query_head = out_head = 0;
    if (cache->Hkv == 1) key_head = value_head = 0;
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
    const int size = r.dtype == ADACODE_FP32 ? 4 : 2;
    const bool whole_angles = r.axes == 1 && (((uintptr_t)r.cos | (uintptr_t)r.sin) & 15) == 0 && r.token_stride * size % 16 == 0;
    AppendArgs a{*cache,    r,        query,     key,      value,       query_out,  query_token, query_head,   out_token,
                 out_head,  key_token, key_head, value_token, value_head, Hq,       status,      whole_angles, 0};
    // sixteen bytes at a time where everything allows it
    const uintptr_t pointers = (uintptr_t)query | (uintptr_t)query_out | (uintptr_t)key | (uintptr_t)value | (uintptr_t)cache->key_pages |
                               (uintptr_t)cache->value_pages;
    const int64_t strides = query_token | query_head | out_token | out_head | key_token | key_head | value_token | value_head | cache->key_page |
                            cache->key_head | cache->key_slot | cache->value_page | cache->value_head | cache->value_slot;
    const bool wide = (pointers & 15) == 0 && (strides & 7) == 0 && cache->D % 16 == 0 && r.half % 8 == 0;
    const cudaError_t e = cache->dtype == ADACODE_BF16 ? launch_append<__nv_bfloat16>(a, wide, (cudaStream_t)stream)
                                                       : launch_append<__half>(a, wide, (cudaStream_t)stream);
    if (e == cudaSuccess) return ADACODE_OK;
    (void)cudaGetLastError();
    return ADACODE_ERR_CUDA;
}

}  // extern "C"
