// Attention of new tokens over the pages of their sequences, on the tensor cores of sm_100a.
//
// Work.  A row is one query head of one new token; the G heads that share a cached head lie next to each other, so that the rows
// of (sequence, cached head) are n G consecutive ones, and a unit is 128 or 256 of them.  Its tiles are the runs of 128 cached
// positions that any of its rows sees.  The tiles of all units, one unit after the other, are cut evenly among the CTAs (one per SM), so a
// CTA has a run of tiles which may begin and end within a unit; what a CTA has of a unit is a piece.  A unit that is cut leaves
// partial results (numerator, maximum, sum per row) that a second kernel merges.  Lengths lie on the device: every
// CTA finds its run by itself.
//
// One CTA: warp 9 finds the pieces and loads the keys, warp 10 the values (one tensor copy per page and 64 columns), warp 8 issues the products
// of both streams (a warp for each made them interleave, and took a third longer), two warpgroups do the softmax, one row per thread.  S = Q K^T goes
// to TMEM, the weights go back to where S was, and O += P V takes them from there.  Two streams of S, P and O let one's softmax run while the other's products do:
//   PAIR  a unit has 256 rows, stream i the rows 128 i ..; every tile is used by both.
//   SOLO  a unit has 128 rows; stream i takes every second tile, and the two meet at the end of the piece.  For few rows, where
//         reading the cache is what takes time, with three instead of two tiles of keys and values on the way.
// Numerators are scaled by 2**-m for a maximum m that lags: it moves only when a row's maximum has grown by more
// than 2**8, which spares nearly all rescaling of O; weights stay below 2**8 and sums below 2**8 times the length.
//
// Measured (device time): a decode step of 64 sequences of up to 8192 tokens, 32 heads on 8 of 128, 220 us, 6.1 TB/s, bound by memory; two chunks of
// 2048 tokens behind 16384 644 us, 1103 TFLOP/s, and 509 tokens behind 20557 168 us, 1008 TFLOP/s, bound by the chain of one stream's tile (softmax
// 2300 cycles, products 1300; two streams take turns); one token behind 2050 12.5 us, bound by latency (finding the run some 3500 cycles, one
// tile 8000, the merge).
//
// Hidden positions get the score minus infinity; their values would still be multiplied by the weight 0.  Values that no row of the unit sees
// (behind its last token, before its first one's window, left padding, which a model may well leave full of NaN) are cleared in shared memory.
// Others, which some rows see, only matter if they are infinite or NaN: a row that ends with such a numerator but a finite sum is computed again by
// repair_row, which never looks at what is hidden.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "adacode.h"

#include <atomic>
#include <cmath>
#include <mutex>

namespace {

#include "adacode_device.cuh"
#define ADACODE_PIPELINE_UNPACK_ONLY
#include "adacode_pipeline.cuh"
#include "adacode_pages.cuh"

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 128;               // cached positions per tile, rows per stream
constexpr int kAttnThreads = 384;         // two warpgroups of softmax, one of which three warps work
// Registers per thread: 384 x 168 at the launch, which the softmax (whose rows are held whole) takes from the others.
constexpr int kRegsRows = 224, kRegsRest = 56;
static_assert(256 * kRegsRows + 128 * kRegsRest <= 384 * 168, "a split of what the launch has");
constexpr int kPieces = 4;               // pieces that the loading warps are ahead at most
constexpr float kLag = 8.f;              // how far (powers of two) a maximum may be behind

struct PagedArgs {
    adacode_paged_cache cache;
    const void *query;
    void *out;
    long long q_n, q_h, o_n, o_h;
    const int32_t *starts;
    int Hq, G, causal, window;
    float scale;              // times log2 e, positive (queries are negated where it is negative; 0 is the smallest there is: hidden
                              // scores are minus infinity, and that times 0 is no number)
    uint32_t negate;
    int box_shift;            // 2**box_shift rows per tensor copy
    int room;                 // positions that the table has
    Quotient by_page, by_group;
    float *part_o, *part_ml;  // [2 CTAs][rows][D], [2 CTAs][rows][2]
    struct Cut *cuts;         // [CTAs]
    int32_t *status;
};

// What a CTA has of a unit.
struct Piece {
    int n, j0;                // tiles, the first of them; n == 0: no more pieces
    int rows, row0;           // of the unit: how many, the first within the sequence's head
    int b, h, q0, fresh, len, start;
    int lo, hi;               // positions that any of the unit's rows sees: lo .. hi - 1
    int slot;                 // of the partial results, -1: the unit is whole
};

// A unit whose first piece is the CTA's, for the merging kernel (n == 0: none).
struct Cut {
    int n, rows, row0, b, h, q0, fresh, len, start;
};

// A wait of the whole warp, with one answer: lanes that give up and lanes that do not never part.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, int32_t *status) {
    return __all_sync(kFull, mbar_wait(bar, parity, status));
}

// ---------------------------------------------------------------------------------------
// tcgen05
// ---------------------------------------------------------------------------------------

__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// (the loaded registers pass through, so that nothing that uses them moves before the wait)
template <int N>
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[N][32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 32; ++e) asm volatile("" : "+r"(r[i][e]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_ld(uint32_t (&r)[32], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_st(const uint32_t (&r)[32], uint32_t at) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
        "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(const uint32_t (&r)[16], uint32_t at) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
        "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(at)
        : "memory");
}
// D[128 x N] (+)= A B, both operands in shared memory, or A (16-bit pairs along its columns) in TMEM.  Issued by one lane by a predicate, not
// in a branch: operands that a branch on the lane makes look different per lane are moved one by one before every product (100 cycles
// each; the product takes 64).
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
        : "memory");
}
// the barrier counts one arrival when all products issued so far are done
__device__ __forceinline__ void mma_commit(uint32_t leader, uint64_t *bar) {
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar)),
        "r"(leader)
        : "memory");
}
// Operands in shared memory are stacks of 8 rows of 128 bytes, their 16-byte pieces permuted by the row (128-byte swizzle); 64 columns
// of all rows come before the next 64.  Rows of queries and keys are the product's rows (its sum runs along the columns); rows of
// values are what the sum runs over, with `lead` bytes between one group of 64 columns and the next.
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t lead) {
    return (uint64_t)((at & 0x3FFFFu) >> 4) | (uint64_t)((lead >> 4) & 0x3FFFu) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
template <typename T>
__host__ __device__ constexpr uint32_t instruction(int n, bool b_by_rows) {
    return 1u << 4 | (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u << 7 | 1u << 10 : 0u) | (b_by_rows ? 1u << 16 : 0u) |
           (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack_two(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_two<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack_two<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two floats in one register pair, for the packed instructions.
using Two = unsigned long long;
__device__ __forceinline__ Two two(float lo, float hi) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void parts(Two v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ Two fma_two(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Two add_two(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float most_of(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The weights of 32 scores: summed up, rounded, stored to 16 columns of TMEM.  The special function unit takes eight cycles for a warp's
// powers of two, 1024 for a tile, as long as the tile's products.  (A polynomial of degree 3 on the FMA pipe for a quarter to a half of them
// made the two chunks of 2048 tokens behind 16384 slower, 652 us -> 674 and 694: what counts is a warp's own chain of
// instructions, while the unit is idle half of the time.)
template <typename T>
__device__ __forceinline__ void weigh(const uint32_t (&x)[32], Two c, Two base, Two (&sum)[2], uint32_t at) {
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const Two y = fma_two(two(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), c, base);
        float p0, p1;
        parts(y, p0, p1);
        p0 = exp2_fast(p0), p1 = exp2_fast(p1);
        sum[e & 1] = add_two(sum[e & 1], two(p0, p1));
        w[e] = pack_two<T>(p0, p1);
    }
    tmem_st16(w, at);
}

// ---------------------------------------------------------------------------------------
// units
// ---------------------------------------------------------------------------------------

// Positions that new token t (of `fresh`) of a sequence sees: lo .. hi - 1, of those that the table has.
__device__ __forceinline__ void seen_by(const PagedArgs &a, int t, int fresh, int len, int start, int &lo, int &hi) {
    const int at = len - fresh + t;
    lo = start > 0 ? start : 0;
    if (a.window > 0 && at >= 0 && at - lo >= a.window) lo = at - a.window + 1;
    hi = a.causal && at + 1 < len ? at + 1 : len;
    if (hi > a.room) hi = a.room;
}
// Those that any of rows row0 .. row1 - 1 sees.
__device__ __forceinline__ void seen_by_unit(const PagedArgs &a, int row0, int row1, int fresh, int len, int start, int &lo, int &hi) {
    int other;
    seen_by(a, (uint32_t)row0 / a.by_group, fresh, len, start, lo, other);
    seen_by(a, (uint32_t)(row1 - 1) / a.by_group, fresh, len, start, other, hi);
}
// Whether the last of them sees a position that the table does not have.
__device__ __forceinline__ bool beyond_table(const PagedArgs &a, const Piece &p) {
    if (p.len <= a.room) return false;
    const int t = (int)((uint32_t)(p.row0 + p.rows - 1) / a.by_group), at = p.len - p.fresh + t, to = a.causal && at + 1 < p.len ? at + 1 : p.len;
    return to > a.room && p.lo < to;
}
// The tiles of positions lo .. hi - 1 (one, of hidden positions, if there are none).
__device__ __forceinline__ int tiles_of(int lo, int hi, int &first) {
    first = lo / kTile;
    const int n = (hi > 0 ? (hi - 1) / kTile + 1 : 0) - first;
    if (n <= 0) first = 0;
    return n > 0 ? n : 1;
}
__device__ __forceinline__ int unit_tiles(const PagedArgs &a, int row0, int row1, int fresh, int len, int start, int &first) {
    int lo, hi;
    seen_by_unit(a, row0, row1, fresh, len, start, lo, hi);
    return tiles_of(lo, hi, first);
}
__device__ __forceinline__ void sequence(const PagedArgs &a, int b, int &q0, int &fresh, int &len, int &start) {
    if (a.cache.cu_seqlens) {
        q0 = a.cache.cu_seqlens[b];
        int q1 = a.cache.cu_seqlens[b + 1];
        if (q1 > a.cache.N) q1 = a.cache.N;
        fresh = q0 < 0 || q1 < q0 ? 0 : q1 - q0;
    } else {
        fresh = a.cache.N / a.cache.B;
        q0 = b * fresh;
    }
    len = a.cache.seq_lens[b] > 0 ? a.cache.seq_lens[b] : 0;
    start = a.starts ? a.starts[b] : 0;
}
// Tiles of all units of one head of a sequence.
template <int ROWS>
__device__ __forceinline__ uint32_t head_tiles(const PagedArgs &a, int fresh, int len, int start) {
    const int rows = fresh * a.G;
    uint32_t n = 0;
    int first;
    for (int r = 0; r < rows; r += ROWS) n += unit_tiles(a, r, r + ROWS < rows ? r + ROWS : rows, fresh, len, start, first);
    return n;
}
__device__ __forceinline__ uint32_t warp_scan(uint32_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t u = __shfl_up_sync(kFull, v, d);
        if (lane >= d) v += u;
    }
    return v;
}

// ---------------------------------------------------------------------------------------
// rows that hidden infinities have spoilt
// ---------------------------------------------------------------------------------------

// Columns c0 .. c1 - 1 of one row by the whole warp, in 32 bits, 32 positions at a time: first the weights' sum and then the values, of which hidden
// ones and those of weight 0 are not read.  A position without a page counts as zeros.
template <typename T, int D>
__device__ __noinline__ void repair_row(const PagedArgs &a, int b, int h, int q0, int fresh, int len, int start, int row, int c0, int c1) {
    constexpr int E = D / 32;
    const adacode_paged_cache &c = a.cache;
    const int lane = threadIdx.x & 31, t = (int)((uint32_t)row / a.by_group), head = h * a.G + row - t * a.G;
    int lo, hi;
    seen_by(a, t, fresh, len, start, lo, hi);
    const T *q = reinterpret_cast<const T *>(a.query) + (q0 + t) * a.q_n + head * a.q_h;
    const float scale = a.negate ? -a.scale : a.scale;
    float acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        const float base = m == -INFINITY ? 0.f : m, share = pass ? 1.f / l : 0.f;
#pragma unroll 1
        for (int j0 = lo; j0 < hi; j0 += 32) {
            // a position's score per lane
            int slot = 0;
            const int page = j0 + lane < hi ? page_of(c, b, j0 + lane, slot) : -1;
            float s = j0 + lane < hi ? 0.f : -INFINITY;
            if (page >= 0) {
                const T *k = reinterpret_cast<const T *>(c.key_pages) + page * c.key_page + h * c.key_head + slot * c.key_slot;
#pragma unroll 4
                for (int d = 0; d < D; d += 8) {
                    const uint4 kw = *reinterpret_cast<const uint4 *>(k + d), qw = *reinterpret_cast<const uint4 *>(q + d);
                    const T *ke = reinterpret_cast<const T *>(&kw), *qe = reinterpret_cast<const T *>(&qw);
#pragma unroll
                    for (int e = 0; e < 8; ++e) s = fmaf(widen(qe[e]), widen(ke[e]), s);
                }
                s *= scale;
            }
            if (pass == 0) {
                const float top = fmaxf(m, s), from = top == -INFINITY ? 0.f : top;
                l = l * exp2f(m - from) + exp2f(s - from);
                m = top;
                continue;
            }
            const float p = exp2f(s - base) * share;
            const long long at = page * c.value_page + slot * c.value_slot;
            unsigned seen = __ballot_sync(kFull, page >= 0 && p != 0.f);
            while (seen) {
                const int i = __ffs(seen) - 1;
                seen &= seen - 1;
                const float w = __shfl_sync(kFull, p, i);
                const T *v = reinterpret_cast<const T *>(c.value_pages) + __shfl_sync(kFull, at, i) + h * c.value_head + lane * E;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = fmaf(w, widen(v[e]), acc[e]);
            }
        }
        if (pass == 0) {
            // the lanes' maxima and sums put together
            float top = m;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
            l = m == -INFINITY ? l : l * exp2f(m - top);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(kFull, l, d);
            m = top;
            if (l == 0.f) break;
        }
    }
    T *out = reinterpret_cast<T *>(a.out) + (q0 + t) * a.o_n + head * a.o_h;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane * E + e >= c0 && lane * E + e < c1) out[lane * E + e] = narrow<T>(acc[e]);
}

// ---------------------------------------------------------------------------------------
// the kernel
// ---------------------------------------------------------------------------------------

template <int D, bool SOLO>
struct Shape {
    static constexpr int kRows = SOLO ? kTile : 2 * kTile;         // of a unit
    static constexpr int kHalf = kTile * 128;                      // bytes of 64 columns of a tile
    static constexpr int kBytes = kTile * D * 2;                   // of a tile
    static constexpr int kKeys = D == 128 ? 3 : 4, kValues = D == 128 ? (SOLO ? 3 : 2) : 4;  // stages
};

template <int D, bool SOLO>
struct Shared {
    using S = Shape<D, SOLO>;
    alignas(1024) uint8_t q[SOLO ? 1 : 2][S::kBytes];
    alignas(1024) uint8_t k[S::kKeys][S::kBytes];
    alignas(1024) uint8_t v[S::kValues][S::kBytes];
    alignas(8) uint64_t k_full[S::kKeys], k_empty[S::kKeys], v_full[S::kValues], v_empty[S::kValues];
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
    uint64_t piece_full[kPieces], piece_empty[kPieces], sums, read, done;   // (sums, read: SOLO)
    Piece piece[kPieces];
    float ml[2][kTile][2];
    uint32_t tmem;
};
static_assert(sizeof(Shared<128, true>) <= 227 * 1024 && sizeof(Shared<128, false>) <= 227 * 1024, "one CTA's shared memory");

// The k-th use of a ring of n stages.
struct Ring {
    int n, at = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ explicit Ring(int n) : n(n) {}
    __device__ __forceinline__ void next() {
        if (++at == n) at = 0, phase ^= 1;
    }
    __device__ __forceinline__ void back() {
        if (at == 0) at = n, phase ^= 1;
        --at;
    }
};

// a x / n, where a < n
__device__ __forceinline__ uint32_t share_of(uint32_t x, uint32_t a, uint32_t n) {
    return x < 1u << 22 && n < 1u << 10 ? x * a / n : (uint32_t)((uint64_t)x * a / n);
}

// Finds where the run of CTA `cta` begins: the unit (its row0, sequence and head in `p`) and how many of its tiles come before.  Returns the run's
// length; `ctas`: how many CTAs have runs (no CTA between two of a unit goes without a tile), `total`: all tiles.
template <int ROWS>
__device__ __forceinline__ int find_run(const PagedArgs &a, int cta, Piece &p, int &skipped, int &ctas, uint32_t &total) {
    const adacode_paged_cache &c = a.cache;
    const int lane = threadIdx.x & 31;
    int q0 = 0, fresh = 0, len = 0, start = 0;                 // of sequence b0 + lane
    uint32_t w = 0;
    const auto look_at = [&](int b) {
        fresh = 0;
        if (b < c.B) sequence(a, b, q0, fresh, len, start);
        w = head_tiles<ROWS>(a, fresh, len, start);
    };
    total = 0;
    for (int b0 = (c.B - 1) / 32 * 32; b0 >= 0; b0 -= 32) {    // (the first 32 last, whose numbers are kept)
        look_at(b0 + lane);
        total += w;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(kFull, total, d);
    total *= c.Hkv;
    ctas = total < gridDim.x ? (int)total : (int)gridDim.x;
    if (cta >= ctas) return 0;
    const uint32_t x = share_of(total, cta, ctas), end = share_of(total, cta + 1, ctas);
    uint32_t from = 0;
    int l = 0;
    for (int b0 = 0;; b0 += 32) {
        if (b0 > 0) look_at(b0 + lane);
        const uint32_t upto = from + warp_scan(w * c.Hkv);
        const unsigned later = __ballot_sync(kFull, upto > x);
        if (later || b0 + 32 >= c.B) {
            // (the bounds here and below only matter if lengths change while the kernel runs)
            l = later ? __ffs(later) - 1 : c.B - 1 - b0;
            p.b = b0 + l;
            from = __shfl_sync(kFull, upto, l);
            break;
        }
        from = __shfl_sync(kFull, upto, 31);
    }
    const uint32_t per_head = __shfl_sync(kFull, w, l);
    p.q0 = __shfl_sync(kFull, q0, l), p.fresh = __shfl_sync(kFull, fresh, l), p.len = __shfl_sync(kFull, len, l), p.start = __shfl_sync(kFull, start, l);
    if (per_head == 0 || p.fresh == 0) return 0;
    from -= per_head * c.Hkv;
    p.h = (int)((x - from) / per_head);
    if (p.h >= c.Hkv) p.h = c.Hkv - 1;
    from += p.h * per_head;
    for (p.row0 = 0;; p.row0 += ROWS) {
        p.rows = p.fresh * a.G - p.row0 < ROWS ? p.fresh * a.G - p.row0 : ROWS;
        const uint32_t n = unit_tiles(a, p.row0, p.row0 + p.rows, p.fresh, p.len, p.start, p.j0);
        skipped = x < from + n ? (int)(x - from) : (int)n - 1;
        if (x < from + n || p.row0 + ROWS >= p.fresh * a.G) break;
        from += n;
    }
    return (int)(end - x);
}

// Loads the keys or the values of a piece.  Lane i has the i-th page (or box of slots of one) of a tile; the table is read one tile ahead, so that
// its latency hides behind the copies.  Pages of which no row of the unit sees anything are neither looked up, they need not exist, nor copied.  A
// copy brings 64 columns of a page, issued by a lane of its own.  Keys and values have a warp each: with one for both, sixteen sequences of five
// tokens over pages of 16 took 62 us instead of 48.
template <int D, int STAGES>
__device__ __forceinline__ bool load_tiles(const PagedArgs &a, const Piece &p, const CUtensorMap &map, Ring &r, uint8_t (*stage)[kTile * D * 2],
                                           uint64_t *full, uint64_t *empty) {
    const adacode_paged_cache &c = a.cache;
    const int lane = threadIdx.x & 31;
    const uint32_t leader = lane == 0;
    const int tiles = p.n, h = p.h, held = p.hi - p.j0 * kTile, at0 = p.j0 * kTile + (lane << a.box_shift);
    const int32_t *table = c.block_table + p.b * c.table_stride;
    const auto boxes_of = [&](int j) {                        // behind the last page of tile j that is seen
        const int valid = held - j * kTile;
        return j >= tiles || valid <= 0 ? 0 : valid >= kTile ? kTile >> a.box_shift : (valid + (1 << a.box_shift) - 1) >> a.box_shift;
    };
    int next_boxes = boxes_of(0), next_page = -1, next_slot = 0;
    int before = p.lo > p.j0 * kTile ? (p.lo - p.j0 * kTile) >> a.box_shift : 0;      // pages of the first tile that are not
    const auto look_up = [&](int j) {
        if (lane >= before && lane < next_boxes) {
            const int at = at0 + j * kTile, entry = (int)((uint32_t)at / a.by_page);
            next_slot = at - entry * c.page_size;
            next_page = entry < c.table_width ? table[entry] : -1;
        }
    };
    look_up(0);
    for (int j = 0; j < tiles; ++j) {
        const int boxes = next_boxes, hidden = before;
        int page = next_page, slot = next_slot;
        if (lane >= hidden && lane < boxes && (page < 0 || page >= c.n_pages)) {      // (a page behind the pool reads as zeros)
            page = c.n_pages, slot = 0;
            atomicOr(a.status, ADACODE_STATUS_BAD_PAGE);
        }
        before = 0;
        next_boxes = boxes_of(j + 1);
        look_up(j + 1);
        if (!warp_wait(&empty[r.at], r.phase ^ 1, a.status)) return false;
        const uint32_t bar = smem_u32(&full[r.at]), to = smem_u32(stage[r.at]);
        if (leader) {
            if (boxes > hidden) mbar_arrive_expect_tx(&full[r.at], (boxes - hidden) * (D * 2) << a.box_shift);
            else mbar_arrive(&full[r.at]);
        }
        __syncwarp();
        const int i = lane / (D / 64), half = lane % (D / 64);
        const int from = __shfl_sync(kFull, page, i), first = __shfl_sync(kFull, slot, i);
        if (i >= hidden && i < boxes)
            asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                             to + half * (kTile * 128) + (i * 128 << a.box_shift)),
                         "l"(&map), "r"(half * 64), "r"(first), "r"(h), "r"(from), "r"(bar)
                         : "memory");
        r.next();
    }
    return true;
}
// Given up: do not leave while a copy may be in flight.
template <int STAGES>
__device__ __forceinline__ void drain(Ring &r, uint64_t *full, int32_t *status) {
    for (int i = 0; i < STAGES; ++i) {
        r.back();
        mbar_wait(&full[r.at], r.phase, status, 1u << 16);
    }
}

// Finds the pieces and loads the keys.
template <int D, bool SOLO>
__device__ __forceinline__ void load_keys(const PagedArgs &a, Shared<D, SOLO> &s, const CUtensorMap &map) {
    using S = Shape<D, SOLO>;
    const adacode_paged_cache &c = a.cache;
    const int lane = threadIdx.x & 31;
    Ring r(S::kKeys), pr(kPieces);
    bool ok = true;
    Piece p;
    int skipped = 0, ctas;
    uint32_t total;
    int left = find_run<S::kRows>(a, blockIdx.x, p, skipped, ctas, total);
    bool is_cut = false;
    while (left > 0) {
        int first;
        seen_by_unit(a, p.row0, p.row0 + p.rows, p.fresh, p.len, p.start, p.lo, p.hi);
        const int all = tiles_of(p.lo, p.hi, first);
        const bool whole = all - skipped <= left;
        p.j0 = first + skipped;
        p.n = whole ? all - skipped : left;
        p.slot = skipped > 0 ? 2 * blockIdx.x : whole ? -1 : 2 * blockIdx.x + 1;
        ok = warp_wait(&s.piece_empty[pr.at], pr.phase ^ 1, a.status);
        if (!ok) break;
        if (lane == 0) {
            s.piece[pr.at] = p;
            mbar_arrive(&s.piece_full[pr.at]);
        }
        pr.next();
        ok = load_tiles<D, S::kKeys>(a, p, map, r, s.k, s.k_full, s.k_empty);
        if (!ok) break;
        if (beyond_table(a, p) && lane == 0) atomicOr(a.status, ADACODE_STATUS_BAD_PAGE);
        if (skipped == 0 && !whole) {
            // the unit goes on behind this run: its last tile is all - p.n tiles further on
            const uint32_t end = share_of(total, blockIdx.x + 1, ctas);
            // (no CTA is behind the last, even if lengths change while the kernel runs)
            const int last = (int)(((uint64_t)(end + (all - p.n)) * ctas - 1) / total);
            is_cut = true;
            if (lane == 0)
                a.cuts[blockIdx.x] = {(last < ctas ? last : ctas - 1) - (int)blockIdx.x + 1, p.rows, p.row0, p.b, p.h, p.q0, p.fresh, p.len, p.start};
        }
        left -= p.n;
        skipped = 0;
        if (left == 0) break;
        p.row0 += S::kRows;
        if (p.row0 >= p.fresh * a.G) {
            p.row0 = 0;
            if (++p.h == c.Hkv) {
                p.h = 0;
                if (p.b + 1 >= c.B) break;
                do sequence(a, ++p.b, p.q0, p.fresh, p.len, p.start);
                while (p.fresh == 0 && p.b + 1 < c.B);
                if (p.fresh == 0) break;
            }
        }
        p.rows = p.fresh * a.G - p.row0 < S::kRows ? p.fresh * a.G - p.row0 : S::kRows;
    }
    if (lane == 0 && (!is_cut || !ok)) a.cuts[blockIdx.x].n = 0;
    if (ok) ok = warp_wait(&s.piece_empty[pr.at], pr.phase ^ 1, a.status);
    if (ok && lane == 0) {
        s.piece[pr.at].n = 0;
        mbar_arrive(&s.piece_full[pr.at]);
    }
    if (!ok) drain<S::kKeys>(r, s.k_full, a.status);
}
template <int D, bool SOLO>
__device__ __forceinline__ void load_values(const PagedArgs &a, Shared<D, SOLO> &s, const CUtensorMap &map) {
    using S = Shape<D, SOLO>;
    Ring r(S::kValues), pr(kPieces);
    for (;;) {
        if (!warp_wait(&s.piece_full[pr.at], pr.phase, a.status)) break;
        if (s.piece[pr.at].n == 0) return;
        if (!load_tiles<D, S::kValues>(a, s.piece[pr.at], map, r, s.v, s.v_full, s.v_empty)) break;
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&s.piece_empty[pr.at]);
        pr.next();
    }
    drain<S::kValues>(r, s.v_full, a.status);
}

// Products.
template <typename T, int D, bool SOLO>
__device__ __forceinline__ bool multiply_pieces(const PagedArgs &a, Shared<D, SOLO> &s, uint32_t tmem) {
    using S = Shape<D, SOLO>;
    constexpr uint32_t kScores = instruction<T>(kTile, false), kOut = instruction<T>(D, true);
    const int lane = threadIdx.x & 31;
    const uint32_t leader = lane == 0;
    Ring kr(S::kKeys), vr(S::kValues), pr(kPieces);
    uint32_t q_phase = 0, p_phase = 0;       // (a bit per stream)
    const uint64_t q_at = operand(smem_u32(s.q), 16), k_at = operand(smem_u32(s.k), 16), v_at = operand(smem_u32(s.v), S::kHalf);
    const auto scores = [&](int i) {         // stream i's next tile of keys, which has arrived
        const uint64_t q = q_at + (SOLO ? 0 : i * (S::kBytes >> 4)), keys = k_at + kr.at * (S::kBytes >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = ((k / 4) * S::kHalf + (k % 4) * 32) >> 4;
            mma_ss(leader, tmem + i * 128, q + off, keys + off, kScores, k > 0);
        }
        mma_commit(leader, &s.s_full[i]);
    };
    const auto output = [&](int i, bool add) {
        const uint64_t values = v_at + vr.at * (S::kBytes >> 4);
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
            mma_ts(leader, tmem + 256 + i * D, tmem + i * 128 + k * 8, values + k * (2048 >> 4), kOut, k > 0 ? 1u : (uint32_t)add);
    };
    const auto release = [&](uint64_t *bar) { mma_commit(leader, bar); };
    for (;;) {
        if (!warp_wait(&s.piece_full[pr.at], pr.phase, a.status)) return false;
        const int tiles = s.piece[pr.at].n, rows = s.piece[pr.at].rows, j0 = s.piece[pr.at].j0 * kTile, lo = s.piece[pr.at].lo - j0, hi = s.piece[pr.at].hi - j0;
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.piece_empty[pr.at]);
        pr.next();
        if (tiles == 0) return true;
        const int streams = SOLO ? (tiles > 1 ? 2 : 1) : (rows > kTile ? 2 : 1);
#pragma unroll 1
        for (int i = 0; i < (SOLO ? 1 : streams); ++i) {
            if (!warp_wait(&s.q_full[i], q_phase >> i & 1, a.status)) return false;
            q_phase ^= 1u << i;
        }
#pragma unroll 1
        for (int i = 0; i < streams; ++i) {
            if ((SOLO || i == 0) && !warp_wait(&s.k_full[kr.at], kr.phase, a.status)) return false;
            tmem_fence_after();
            scores(i);
            if (SOLO || i == streams - 1) release(&s.k_empty[kr.at]), kr.next();
        }
        for (int t = 0; t < tiles; ++t) {
            if (!warp_wait(&s.v_full[vr.at], vr.phase, a.status)) return false;
            const int from = lo - t * kTile, to = hi - t * kTile;
            if (from > 0 || to < kTile) {    // values that no row of the unit sees are cleared
                const auto clear = [&](int row0, int row1) {
                    for (int x = row0 * (D / 8) + lane; x < row1 * (D / 8); x += 32) {
                        const int row = x / (D / 8), col = x - row * (D / 8);
                        *reinterpret_cast<uint4 *>(s.v[vr.at] + (col / 8) * S::kHalf + row * 128 + (col % 8) * 16) = make_uint4(0, 0, 0, 0);
                    }
                };
                clear(0, from < kTile ? from : kTile);
                clear(to > 0 ? to : 0, kTile);
                fence_async_smem();
                __syncwarp();
            }
            const int last = t + (SOLO ? 2 : 1);          // the tile whose scores follow
            if (last < tiles && !warp_wait(&s.k_full[kr.at], kr.phase, a.status)) return false;
#pragma unroll 1
            for (int i = SOLO ? (t & 1) : 0; i < (SOLO ? (t & 1) + 1 : streams); ++i) {
                if (!warp_wait(&s.p_full[i], p_phase >> i & 1, a.status)) return false;
                p_phase ^= 1u << i;
                tmem_fence_after();
                output(i, t >= (SOLO ? 2 : 1));
                if (SOLO || i == streams - 1) release(&s.v_empty[vr.at]), vr.next();
                if (last < tiles) {
                    scores(i);
                    if (SOLO || i == streams - 1) release(&s.k_empty[kr.at]), kr.next();
                } else {
                    release(&s.o_full[i]);
                }
            }
        }
    }
}

// Softmax of stream `stream`, a row per thread.
template <typename T, int D, bool SOLO>
__device__ __forceinline__ bool soften_pieces(const PagedArgs &a, Shared<D, SOLO> &s, uint32_t tmem, int stream) {
    using S = Shape<D, SOLO>;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) & 3, r = warp * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)warp << 21), s_at = lanes + stream * 128, o_at = lanes + 256 + stream * D;
    const float c = a.scale;
    Ring pr(kPieces);
    uint32_t s_phase = 0, o_phase[2] = {0, 0}, ends = 0;
    for (;;) {
        if (!warp_wait(&s.piece_full[pr.at], pr.phase, a.status)) return false;
        const Piece p = s.piece[pr.at];
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.piece_empty[pr.at]);
        pr.next();
        if (p.n == 0) return true;
        const int row = (SOLO ? 0 : stream * kTile) + r;      // within the unit
        const bool mine = row < p.rows;
        if (!SOLO && p.rows <= stream * kTile) continue;
        const int t = (int)((uint32_t)(p.row0 + row) / a.by_group), head = p.h * a.G + p.row0 + row - t * a.G;
        int lo = 0, hi = INT32_MAX;
        if (mine) seen_by(a, t, p.fresh, p.len, p.start, lo, hi);
        // queries (of SOLO, half of the columns per warpgroup)
        {
            constexpr int kChunks = SOLO ? D / 16 : D / 8;
            const int c0 = SOLO ? stream * kChunks : 0;
            const uint4 *q = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.query) + (long long)(p.q0 + t) * a.q_n + head * a.q_h) + c0;
            uint4 x[kChunks];
#pragma unroll
            for (int k = 0; k < kChunks; ++k) x[k] = mine ? q[k] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < kChunks; ++k) {
                const int col = c0 + k;
                x[k].x ^= a.negate, x[k].y ^= a.negate, x[k].z ^= a.negate, x[k].w ^= a.negate;
                *reinterpret_cast<uint4 *>(s.q[SOLO ? 0 : stream] + (col / 8) * S::kHalf + r * 128 + (((col % 8) ^ (r & 7)) * 16)) = x[k];
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.q_full[SOLO ? 0 : stream]);
        }
        const bool idle = !__any_sync(kFull, mine);           // no row of this warp counts
        const int warp_lo = __reduce_max_sync(kFull, lo), warp_hi = __reduce_min_sync(kFull, hi);
        float m = -INFINITY, l = 0.f;
        for (int n = SOLO ? stream : 0; n < p.n; n += SOLO ? 2 : 1) {
            if (!warp_wait(&s.s_full[stream], s_phase, a.status)) return false;
            s_phase ^= 1;
            tmem_fence_after();
            if (!idle) {
                const int j = (p.j0 + n) * kTile;
                uint32_t x[4][32];
#pragma unroll
                for (int k = 0; k < 4; ++k) tmem_ld(x[k], s_at + 32 * k);
                tmem_wait_ld(x);
                if (warp_lo > j || warp_hi < j + kTile) {
#pragma unroll
                    for (int k = 0; k < 128; ++k)
                        if (j + k < lo || j + k >= hi) x[k / 32][k % 32] = 0xFF800000u;
                }
                float top[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    top[k] = fmaxf(__uint_as_float(x[k][0]), __uint_as_float(x[k][1]));
#pragma unroll
                    for (int e = 2; e < 32; e += 2) top[k] = most_of(top[k], __uint_as_float(x[k][e]), __uint_as_float(x[k][e + 1]));
                }
                const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                if (n < (SOLO ? 2 : 1)) {
                    m = most;
                } else {
                    const bool grown = (most - m) * c > kLag || m == -INFINITY;
                    if (__any_sync(kFull, grown)) {
                        // (the product before this tile's scores is done: the barrier counts it too)
                        const float next = grown ? fmaxf(m, most) : m;
                        const float f = m == -INFINITY ? 0.f : exp2_fast((m - next) * c);
                        l *= f;
                        m = next;
#pragma unroll
                        for (int k = 0; k < D / 32; ++k) {
                            uint32_t o[1][32];
                            tmem_ld(o[0], o_at + 32 * k);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[0][e] = __float_as_uint(__uint_as_float(o[0][e]) * f);
                            tmem_st(o[0], o_at + 32 * k);
                        }
                    }
                }
                const float base = fmaxf(m * c, -FLT_MAX);        // (finite where all scaled scores are minus infinity, which then have no weight)
                const Two c2 = two(c, c), base2 = two(-base, -base);
                Two sum[2] = {two(0.f, 0.f), two(0.f, 0.f)};
#pragma unroll
                for (int k = 0; k < 4; ++k) weigh<T>(x[k], c2, base2, sum, s_at + 16 * k);
                float sums[4];
                parts(sum[0], sums[0], sums[1]), parts(sum[1], sums[2], sums[3]);
                l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
                tmem_wait_st();
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.p_full[stream]);
        }
        // (the largest score has weight 1 when it becomes the maximum, unless its product with the scale has passed 32 bits)
        if (l == 0.f && m * c > FLT_MAX) l = NAN;
        // the end of the piece; the streams of a SOLO unit are put together, half of the columns per warpgroup
        const int both = SOLO && p.n > 1;
        float f0 = 1.f, f1 = 0.f;
        if constexpr (SOLO) {
            s.ml[stream][r][0] = m, s.ml[stream][r][1] = l;
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.sums);
            if (!warp_wait(&s.sums, ends, a.status)) return false;
            const float m0 = s.ml[0][r][0], m1 = s.ml[1][r][0];
            m = fmaxf(m0, m1);
            f0 = m0 == -INFINITY ? 0.f : exp2_fast((m0 - m) * c), f1 = m1 == -INFINITY ? 0.f : exp2_fast((m1 - m) * c);
            l = s.ml[0][r][1] * f0 + s.ml[1][r][1] * f1;
            if (m0 == -INFINITY && s.ml[0][r][1] != 0.f) l = s.ml[0][r][1];       // (NaN scores)
            if (m1 == -INFINITY && s.ml[1][r][1] != 0.f) l = s.ml[1][r][1];
            for (int i = 0; i <= both; ++i) {
                if (!warp_wait(&s.o_full[i], o_phase[i], a.status)) return false;
                o_phase[i] ^= 1;
            }
        } else {
            if (!warp_wait(&s.o_full[stream], o_phase[stream], a.status)) return false;
            o_phase[stream] ^= 1;
        }
        tmem_fence_after();
        constexpr int kCols = SOLO ? D / 2 : D;
        const int col0 = SOLO ? stream * kCols : 0;
        const uint32_t from = SOLO ? lanes + 256 + col0 : o_at;
        if (!idle) {
            bool odd = false;
            const float share = p.slot >= 0 ? 1.f : l == 0.f ? 0.f : 1.f / l;
            T *out = reinterpret_cast<T *>(a.out) + (long long)(p.q0 + t) * a.o_n + head * a.o_h + col0;
            float *part = a.part_o + ((long long)p.slot * S::kRows + row) * D + col0;
#pragma unroll
            for (int k = 0; k < kCols / 32; ++k) {
                uint32_t ld[SOLO ? 2 : 1][32];
                uint32_t (&o)[32] = ld[0];
                tmem_ld(o, from + 32 * k);
                if constexpr (SOLO) tmem_ld(ld[1], from + (both ? D : 0) + 32 * k);
                tmem_wait_ld(ld);
                if constexpr (SOLO) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float v = __uint_as_float(o[e]) * f0;
                        o[e] = __float_as_uint(both ? fmaf(__uint_as_float(ld[1][e]), f1, v) : v);
                    }
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) odd |= !isfinite(__uint_as_float(o[e]));
                if (mine) {
                    if (p.slot >= 0) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<uint4 *>(part + 32 * k + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(l == 0.f ? 0.f : __uint_as_float(o[e]) * share);
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint4 w;
                            w.x = pack_two<T>(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), w.y = pack_two<T>(__uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                            w.z = pack_two<T>(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5])), w.w = pack_two<T>(__uint_as_float(o[e + 6]), __uint_as_float(o[e + 7]));
                            *reinterpret_cast<uint4 *>(out + 32 * k + e) = w;
                        }
                    }
                }
            }
            if (p.slot >= 0) {
                if (mine && (!SOLO || stream == 0)) {
                    float *ml = a.part_ml + ((long long)p.slot * S::kRows + row) * 2;
                    ml[0] = m, ml[1] = l;
                }
            } else {
                unsigned again = __ballot_sync(kFull, mine && odd && isfinite(l));
                while (again) {
                    const int who = __ffs(again) - 1;
                    again &= again - 1;
                    repair_row<T, D>(a, p.b, p.h, p.q0, p.fresh, p.len, p.start, p.row0 + __shfl_sync(kFull, row, who), col0, col0 + kCols);
                }
            }
        }
        tmem_fence_before();
        if constexpr (SOLO) {                                 // both streams' numerators have been read
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.read);
            if (!warp_wait(&s.read, ends, a.status)) return false;
            ends ^= 1;
        }
    }
}

template <typename T, int D, bool SOLO>
__global__ void __launch_bounds__(kAttnThreads, 1) k_paged_attn(const __grid_constant__ PagedArgs a, const __grid_constant__ CUtensorMap keys,
                                                                const __grid_constant__ CUtensorMap values) {
    using S = Shape<D, SOLO>;
    extern __shared__ __align__(1024) uint8_t raw[];
    Shared<D, SOLO> &s = *reinterpret_cast<Shared<D, SOLO> *>(raw);
    const int warp = threadIdx.x >> 5;
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kKeys; ++i) mbar_init(&s.k_full[i], 1), mbar_init(&s.k_empty[i], 1);
        for (int i = 0; i < S::kValues; ++i) mbar_init(&s.v_full[i], 1), mbar_init(&s.v_empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&s.q_full[i], SOLO ? 8 : 4), mbar_init(&s.s_full[i], 1), mbar_init(&s.p_full[i], 4), mbar_init(&s.o_full[i], 1);
        for (int i = 0; i < kPieces; ++i) mbar_init(&s.piece_full[i], 1), mbar_init(&s.piece_empty[i], 8 + 2);
        mbar_init(&s.sums, 8), mbar_init(&s.read, 8), mbar_init(&s.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = __shfl_sync(kFull, s.tmem, 0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsRows));
        soften_pieces<T, D, SOLO>(a, s, tmem, warp >> 2);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
        if (warp == 9) {
            load_keys<D, SOLO>(a, s, keys);
        } else if (warp == 10) {
            load_values<D, SOLO>(a, s, values);
        } else if (warp == 8 && !multiply_pieces<T, D, SOLO>(a, s, tmem)) {
            // (given up: products may still be running)
            mma_commit((threadIdx.x & 31) == 0, &s.done);
            mbar_wait(&s.done, 0, a.status, 1u << 16);
        }
    }
    // (not earlier: CTAs of the next kernel would take places on the SMs and wait there)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __syncwarp();
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Puts the pieces of a unit together, a row per warp: the first piece is CTA c's, the others those of the CTAs behind it.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) k_paged_merge(const __grid_constant__ PagedArgs a) {
    constexpr int E = D / 32;
    // Numerators on their way before their weights are known: eight pieces' where few rows are cut into many pieces (one token behind 2050:
    // 12.5 us for both kernels, 13.7 with one piece after the other), two where rows are many and threads have to be.
    constexpr int kAhead = ROWS == kTile ? 8 : 2;
    const int c = blockIdx.x, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Cut cut = a.cuts[c];
    if (cut.n == 0) return;
    for (int row = blockIdx.y * 8 + threadIdx.x / 32; row < cut.rows; row += gridDim.y * 8) {
        const auto piece = [&](int i) { return (long long)(i ? 2 * (c + i) : 2 * c + 1) * ROWS + row; };
        float v[kAhead][E];
        const auto look = [&](int i0) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (i0 + u < cut.n) {
                    const float *src = a.part_o + piece(i0 + u) * D + lane * E;
                    if constexpr (E == 4) {
                        const float4 x = *reinterpret_cast<const float4 *>(src);
                        v[u][0] = x.x, v[u][1] = x.y, v[u][2] = x.z, v[u][3] = x.w;
                    } else {
                        const float2 x = *reinterpret_cast<const float2 *>(src);
                        v[u][0] = x.x, v[u][1] = x.y;
                    }
                }
        };
        look(0);
        // a piece per lane: maximum and sum
        float2 ml = make_float2(-INFINITY, 0.f);
        float m = -INFINITY;
        for (int i = lane; i < cut.n; i += 32) {
            ml = *reinterpret_cast<const float2 *>(a.part_ml + piece(i) * 2);
            m = fmaxf(m, ml.x);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, d));
        float l = 0.f, f = 0.f, o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
        for (int i0 = 0; i0 < cut.n; i0 += kAhead) {
            if (i0 % 32 == 0) {
                if (cut.n > 32) ml = i0 + lane < cut.n ? *reinterpret_cast<const float2 *>(a.part_ml + piece(i0 + lane) * 2) : make_float2(-INFINITY, 0.f);
                // (without a maximum the sum is 0, or NaN as the scores are; the numerator is not looked at)
                f = ml.x == -INFINITY ? -1.f : exp2_fast((ml.x - m) * a.scale);
                l += ml.x == -INFINITY ? ml.y : ml.y * f;
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const float w = __shfl_sync(kFull, f, (i0 + u) % 32);
                if (i0 + u < cut.n && !(w < 0.f)) {
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = fmaf(v[u][e], w, o[e]);
                }
            }
            look(i0 + kAhead);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(kFull, l, d);
        bool odd = false;
#pragma unroll
        for (int e = 0; e < E; ++e) odd |= !isfinite(o[e]);
        if (__any_sync(kFull, odd) && isfinite(l)) {
            repair_row<T, D>(a, cut.b, cut.h, cut.q0, cut.fresh, cut.len, cut.start, cut.row0 + row, 0, D);
            continue;
        }
        const int t = (int)((uint32_t)(cut.row0 + row) / a.by_group), head = cut.h * a.G + cut.row0 + row - t * a.G;
        T *out = reinterpret_cast<T *>(a.out) + (long long)(cut.q0 + t) * a.o_n + head * a.o_h + lane * E;
        const float share = l == 0.f ? 0.f : 1.f / l;
        uint32_t w[E / 2];
#pragma unroll
        for (int e = 0; e < E; e += 2) w[e / 2] = l == 0.f ? 0u : pack_two<T>(o[e] * share, o[e + 1] * share);
        if constexpr (E == 4) *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t *>(out) = w[0];
    }
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------

int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

size_t workspace_bytes_of(bool solo, int D) {
    const size_t slots = 2 * (size_t)sm_count(), rows = slots * (solo ? kTile : 2 * kTile);
    return rows * (D + 2) * sizeof(float) + sm_count() * sizeof(Cut);
}
// One unit of 128 rows suffices: the rows of a sequence's head are few, and the two streams take every second tile each.
bool is_solo(long long max_query_len, int G) { return max_query_len * G <= kTile; }

// Keys or values as the copies see them: (column, slot, head, page), boxes of 64 columns of the slots of one page and head.
bool map_pages(CUtensorMap &map, void *pages, const adacode_paged_cache &c, int64_t page, int64_t head, int64_t slot, int box_rows) {
    static const auto encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            f = nullptr;
        }
        return (decltype(&cuTensorMapEncodeTiled))f;
    }();
    // (a dimension of one entry may have any stride)
    if (c.page_size == 1) slot = c.D;
    if (c.Hkv == 1) head = c.D;
    if (c.n_pages == 1) page = c.D;
    constexpr int64_t kMost = 1ll << 38;
    if (!encode || slot <= 0 || head <= 0 || page <= 0 || slot >= kMost || head >= kMost || page >= kMost) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c.D, (cuuint64_t)c.page_size, (cuuint64_t)c.Hkv, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)slot * 2, (cuuint64_t)head * 2, (cuuint64_t)page * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, step[4] = {1, 1, 1, 1};
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, pages, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Two launches hand partial results on in the workspace: threads that share a stream and a workspace must not come between them, whichever
// kernels their calls are for.
std::mutex &lock_of(const void *workspace) {
    static std::mutex locks[64];
    return locks[((uintptr_t)workspace >> 9) * 0x9E3779B97F4A7C15ull >> 58];
}

template <typename T, int D, bool SOLO>
int launch_paged(const PagedArgs &a, const CUtensorMap &keys, const CUtensorMap &values, int ctas, int max_query_len, cudaStream_t st) {
    // the kernel's limit of dynamic shared memory is raised once per device
    static std::atomic<bool> done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ADACODE_ERR_CUDA;
    constexpr int bytes = (int)sizeof(Shared<D, SOLO>);
    if (dev < 0 || dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(k_paged_attn<T, D, SOLO>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return ADACODE_ERR_CUDA;
        if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
    }
    constexpr int rows = Shape<D, SOLO>::kRows;
    const std::lock_guard<std::mutex> both(lock_of(a.part_o));
    if (launch_dependent(k_paged_attn<T, D, SOLO>, dim3(ctas), kAttnThreads, bytes, st, a, keys, values) != cudaSuccess) return ADACODE_ERR_CUDA;
    // (a warp for four rows, or one where a unit has few by max_query_len: 256 rows of 148 units by a warp each took the chunk of 509 tokens
    // behind 20557 170.5 us instead of 168)
    const long long few = ((long long)max_query_len * a.G + 7) / 8, y = few < rows / 32 ? few : rows / 32;
    return launch_dependent(k_paged_merge<T, D, rows>, dim3(ctas, y < 1 ? 1 : (unsigned)y), 256, 0, st, a) == cudaSuccess ? ADACODE_OK : ADACODE_ERR_CUDA;
}

template <typename T>
int launch_paged(const PagedArgs &a, bool solo, const CUtensorMap &keys, const CUtensorMap &values, int ctas, int max_query_len, cudaStream_t st) {
    if (a.cache.D == 128) return solo ? launch_paged<T, 128, true>(a, keys, values, ctas, max_query_len, st) : launch_paged<T, 128, false>(a, keys, values, ctas, max_query_len, st);
    return solo ? launch_paged<T, 64, true>(a, keys, values, ctas, max_query_len, st) : launch_paged<T, 64, false>(a, keys, values, ctas, max_query_len, st);
}

}  // namespace

extern "C" {

size_t adacode_paged_attn_workspace_bytes(int max_query_len, int Hq, int Hkv, int D) {
    if (max_query_len < 0 || Hkv <= 0 || Hq <= 0 || D <= 0) return 0;
    return workspace_bytes_of(is_solo(max_query_len, Hq / Hkv), D);
}

int adacode_paged_attn(const adacode_paged_cache *cache, const void *query, int64_t query_token, int64_t query_head, int Hq,
                       void *out, int64_t out_token, int64_t out_head, const int32_t *seq_starts, int max_query_len, float scale, int causal,
                       int window, void *workspace, size_t workspace_bytes, int32_t *status, void *stream) {
    if (!valid(cache) || !status || Hq <= 0 || Hq % cache->Hkv != 0 || window < 0 || max_query_len < 0 || !std::isfinite(scale)) return ADACODE_ERR_INVALID_ARG;
    const adacode_paged_cache given = used_strides(*cache);
    cache = &given;
    if (cache->N == 1) query_token = out_token = 0;
    if (Hq == 1) query_head = out_head = 0;
    const int D = cache->D;
    if (D != 64 && D != 128) return ADACODE_ERR_INVALID_ARG;
    const bool one_page = cache->table_width == 1;
    if (!one_page && cache->page_size % 128 != 0 && cache->page_size != 16 && cache->page_size != 32 && cache->page_size != 64)
        return ADACODE_ERR_INVALID_ARG;
    const uintptr_t pointers = (uintptr_t)query | (uintptr_t)out | (uintptr_t)cache->key_pages | (uintptr_t)cache->value_pages | (uintptr_t)workspace;
    const int64_t strides = query_token | query_head | out_token | out_head | cache->key_page | cache->key_head | cache->key_slot |
                            cache->value_page | cache->value_head | cache->value_slot;
    if ((pointers & 15) != 0 || (strides & 7) != 0) return ADACODE_ERR_INVALID_ARG;
    if (cache->N == 0) return ADACODE_OK;
    if (!query || !out || query == out || !workspace || (long long)cache->N * (Hq / cache->Hkv) >= 1ll << 31 || cache->n_pages == INT32_MAX) return ADACODE_ERR_INVALID_ARG;
    const int G = Hq / cache->Hkv, ctas = sm_count();
    const bool solo = is_solo(max_query_len, G);
    if (workspace_bytes < workspace_bytes_of(solo, D)) return ADACODE_ERR_WORKSPACE;
    PagedArgs a;
    a.cache = *cache;
    a.query = query, a.out = out, a.q_n = query_token, a.q_h = query_head, a.o_n = out_token, a.o_h = out_head, a.starts = seq_starts;
    a.Hq = Hq, a.G = G, a.causal = causal, a.window = window;
    a.scale = fmaxf(fabsf(scale) * kLog2e, 1.4e-45f), a.negate = scale < 0 ? 0x80008000u : 0u;
    const int box_rows = one_page || cache->page_size > kTile ? kTile : cache->page_size;         // (16, 32, 64 or 128)
    for (a.box_shift = 0; 1 << a.box_shift < box_rows; ++a.box_shift) {}
    const size_t rows = 2 * (size_t)ctas * (solo ? kTile : 2 * kTile);
    a.part_o = (float *)workspace, a.part_ml = a.part_o + rows * D, a.cuts = (Cut *)(a.part_ml + rows * 2);
    const long long room = (long long)cache->table_width * cache->page_size;
    a.room = room < 1 << 30 ? (int)room : 1 << 30;
    a.by_page = quotient_by(cache->page_size), a.by_group = quotient_by(G);
    a.status = status;
    CUtensorMap keys, values;
    if (!map_pages(keys, cache->key_pages, *cache, cache->key_page, cache->key_head, cache->key_slot, box_rows) ||
        !map_pages(values, cache->value_pages, *cache, cache->value_page, cache->value_head, cache->value_slot, box_rows))
        return ADACODE_ERR_INVALID_ARG;
    const cudaStream_t st = (cudaStream_t)stream;
    const int rc = cache->dtype == ADACODE_BF16 ? launch_paged<__nv_bfloat16>(a, solo, keys, values, ctas, max_query_len, st)
                                                : launch_paged<__half>(a, solo, keys, values, ctas, max_query_len, st);
    if (rc != ADACODE_OK) (void)cudaGetLastError();
    return rc;
}

}  // extern "C"
