// What the operators over a paged cache share.  Included inside an anonymous namespace by each .cu file.
#pragma once

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }

// Sequence of new token i (B if it is before the first or behind the last), found by the whole warp, and the tokens of the call up to its end.
__device__ __forceinline__ int sequence_of(const adacode_paged_cache &c, int i, int &end) {
    if (!c.cu_seqlens) {
        const int each = c.N / c.B, b = i / each;
        end = (b + 1) * each;
        return b;
    }
    const int lane = threadIdx.x & 31, first = c.cu_seqlens[0];
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
    return i < first ? c.B : b;
}

// The page of position `at` of sequence b, or -1.
__device__ __forceinline__ int page_of(const adacode_paged_cache &c, int b, int at, int &slot) {
    const int n = at / c.page_size;
    slot = at - n * c.page_size;
    if (at < 0 || n >= c.table_width) return -1;
    const int page = c.block_table[b * c.table_stride + n];
    return page >= 0 && page < c.n_pages ? page : -1;
}

bool valid(const adacode_paged_cache *c) {
    return c && c->key_pages && c->value_pages && c->block_table && c->seq_lens && c->B > 0 && c->n_pages > 0 && c->page_size > 0 &&
           c->table_width > 0 && c->Hkv > 0 && c->N >= 0 && (c->dtype == ADACODE_BF16 || c->dtype == ADACODE_FP16) &&
           (c->cu_seqlens || c->N % c->B == 0);
}

// A dimension of one entry may have any stride: none that alignment or a tensor map would stumble over.
adacode_paged_cache used_strides(adacode_paged_cache c) {
    if (c.n_pages == 1) c.key_page = c.value_page = 0;
    if (c.Hkv == 1) c.key_head = c.value_head = 0;
    if (c.page_size == 1) c.key_slot = c.value_slot = 0;
    return c;
}
