// Attention of many query rows (whole prompts, chunks) over the paged cache on
// the tensor cores (tcgen05.mma, accumulators in TMEM).
//
// out = softmax(q K^T / sqrt(D)) V per row, one pass over the keys: with m the
// running maximum of the scores x (in powers of two), weights w = 2^(x - m), l =
// sum w and acc = sum w V, a larger maximum rescales l and acc by 2^(m_old -
// m_new), and out = acc / l at the end.  Query rows of one kv head are packed as
// (token, head of the group), so that a group shares every K and V tile.
//
// Precision.  Rows are f32, and one 16-bit operand would round q and the
// weights to 2^-9 or 2^-11.  Both go in as two fp16 halves (x = hi + lo to
// 2^-22; fp16 carries three bits more than bf16, so two halves do what takes
// bf16 three), which doubles the MMA work instead of tripling it.  Both operands
// of an MMA are then fp16, so the CTA's loader turns page rows into fp16: every
// tile of K or V is multiplied by the power of two that brings its largest
// magnitude to [2^13, 2^14), which keeps bf16 values exact down to 2^-31 of the
// tile's largest, and f32 values (as two halves, three products) to 2^-22 of
// their own or 2^-39 of the tile's largest, whichever is more; query rows
// likewise, row by row.  The scales return as one factor of the scores and one of
// the tile's sum.  Weights are taken relative to the largest of their row and tile,
// not of the row so far, and the difference joins the tile's scale: values far
// larger in another tile count with weights far smaller.
//
// What the halves cannot carry is found here and attended again by attend_rows in
// f32, row by row, each over the keys it sees alone (20 to 65 times as long):
// - Scores.  What an element loses beside its row's or its tile's largest is
//   bounded by the two largest, whether or not they meet in a score that counts:
//   less than 2^-18 of a score while their product stays below 2^14 (heads of 128;
//   2^15 for 64).  Rows beyond go again.
// - Values.  The tile's largest may stand in a row that is masked or has no weight,
//   or in another column.  Where some group of neighbours of a row or of a column
//   lies more than 2^16 below it and is not zero, the rows that see some of the tile
//   go again: no value is off by more than 2^-23 of the largest of its neighbours.
// - Weights.  Where the largest weight's own value is zero, or next to it, all that
//   is left may lie below 2^-39: rows whose sums end that far below the tiles'
//   scales go again.
// - Infinities in the tile or in the query, and results that are not finite, unless
//   the sum of weights is NaN: that takes a NaN score the row does see, and the row
//   is NaN.  (NaN stays out of the tiles' largest.)
// The marks travel with the tiles' scales (a negative scale of V, an infinite one
// of K), so that they reach the same rows every time, however far ahead the loader
// is.
//
// The tensor cores add into an f32 accumulator with truncation: measured
// relative error 1.1e-9 per K (9e-6 at K = 8192, always toward zero), so
// a tile's sum of V is taken out of TMEM after every 64 or 128 keys and added in
// registers with rounding, and the products of the second halves, small ones, come
// first.
//
// One CTA: 256 query rows as two M = 128 tiles, so that the softmax of one runs
// under the MMAs of the other.  Warps 0-3 and 4-7: a thread per row of the two
// tiles (scores from TMEM, weights back over them in place, acc in registers).
// Warps 8-11: the loader, global memory to swizzled shared tiles through
// registers, a ring of tiles K0 K1 V0 K2 V1 ..  Warp 12: one thread issues the MMAs.
// Every wait is bounded: one that runs out sets ERR_TIMEOUT and the roles stop.
//
// Measured (causal, bf16 pages, 8 kv heads, 8192 tokens, back to back): 24 heads of
// 64 503 us, 16 heads of 128 490 us (561 TFLOP/s without counting the halves
// twice); f32 pages, 32 heads of 64, 4096 tokens: 250 us; the checks of what the
// halves carry cost 1 to 3 % of it.  No pipe is near full (at
// 4096 of the first: tensor 34 %, exponentials 35 %, issue slots 53 %): the latency
// of a row's chain from scores to weights to sums bounds it, two warps a scheduler.
// Not kept at an earlier step of the first: exponentials by polynomial on the FMA
// units for half or a quarter of them (545, 501 us against 488), in turns (541
// against 498).
#include <cmath>
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "paged.cuh"
#include "paged_dev.cuh"
#include "tcgen.cuh"

namespace krt {

namespace {

constexpr int kRows = kPromptRows;  // query rows of a CTA
constexpr int kPromptThreads = 512;
// Largest factor of the scores, times the head size, that the halves carry: an
// element far below its row's (its tile's) largest is off by up to 2^-25, times
// 2^14 at most and twice for q and K makes 2^-10 an element of the head before the
// factor, and 2^-18 (in powers of two) of the score with this one.
constexpr float kScoreTop = 0x1p-8f;
// A weight is off by up to 2^-25 (of at most 2^14) below 2^-3, so a tile's sums by
// 2^-11 a key and 2^-4 in all, times the scale: 2^-16 of a row whose largest sum
// is this many scales.  Ordinary values: 2^25 and more.
constexpr float kLost = 0x1p12f;
constexpr int kScaleRing = 16;  // tiles' scales; the loader is at most 4 tiles ahead

template <int D, bool F32>
struct Shape {
    static constexpr int Keys = F32 && D == 128 ? 64 : 128;  // keys of a tile
    static constexpr int Parts = F32 ? 2 : 1;                // fp16 halves of K and V
    static constexpr int Sub = Keys * 128;                   // bytes of a [Keys][64] fp16 sub-tile
    static constexpr int Slot = Parts * (D / 64) * Sub;
    static constexpr int Slots = D == 64 ? (F32 ? 4 : 6) : 3;
    static constexpr int QTile = 2 * (D / 64) * 128 * 128;  // both halves of 128 rows
    static constexpr size_t Smem = 2 * (size_t)QTile + (size_t)Slots * Slot + 1024;
    static constexpr int Step = 1024 / D;  // rows that the loader's threads take at once
    static constexpr int Wide = D == 64 ? 32 : 16;  // columns a softmax thread takes at a time
    // TMEM columns: three buffers of scores / weights, which the two query
    // tiles take in turn, and the sums of V of both tiles or, where they do not
    // fit, of one at a time
    static constexpr int Sums = 3 * Keys + 2 * D <= 512 ? 2 : 1;
    static constexpr int SumAt = 3 * Keys;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Instruction descriptor of kind::f16: D f32 (bits 4-5 = 1), A and B fp16 (bits
// 7-9, 10-12 = 0), A or B negated (bits 13, 14), A K-major, B K-major or (bit
// 16) MN-major, N / 8 at bits 17-22, M / 16 at bits 24-28.
template <int N, bool MnMajor>
__host__ __device__ constexpr uint32_t idesc(bool neg_a, bool neg_b) {
    return (1u << 4) | (neg_a ? 1u << 13 : 0u) | (neg_b ? 1u << 14 : 0u) | (MnMajor ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// Lower words of the descriptors of a 128-byte swizzled tile: K-major (the
// leading byte offset unused), and MN-major [K rows][64 of N per sub-tile] with
// 8-row groups of K 1 KB apart (the stride byte offset, as in K-major) and
// 64-wide groups of N `sub` bytes apart (leading byte offset).
__device__ __forceinline__ uint32_t k_desc(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t mn_desc(uint32_t saddr, uint32_t sub) { return (saddr >> 4) | ((sub >> 4) << 16); }

// The upper word of both descriptors; the lower one holds the address, in units
// of 16 bytes, to which offsets are added.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);

// D += A B with A from shared memory, or from TMEM.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t desc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(desc), "r"(accumulate), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t desc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(desc), "r"(accumulate), "r"(kDescHigh)
        : "memory");
}
// Keeps address arithmetic next to its use: hoisted out of the loop, the
// operands of every MMA would each hold a register.
__device__ __forceinline__ uint32_t here(uint32_t x) {
    asm volatile("" : "+r"(x));
    return x;
}

// W columns of this warp's lanes, one lane per thread.  A load is in flight until
// the wait, which v passes through, so that no use of it moves ahead.
template <int W>
struct Tmem;
template <>
struct Tmem<16> {
    using V = uint32_t[16];
    static __device__ __forceinline__ void load(uint32_t taddr, V &v) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
                       "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
                       "=r"(v[14]), "=r"(v[15])
                     : "r"(taddr));
    }
    static __device__ __forceinline__ void wait(V &v) {
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]),
                       "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]),
                       "+r"(v[14]), "+r"(v[15])::"memory");
    }
    static __device__ __forceinline__ void store(uint32_t taddr, const V &v) {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
                     "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                     "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
                     "r"(v[15])
                     : "memory");
    }
};
template <>
struct Tmem<32> {
    using V = uint32_t[32];
    static __device__ __forceinline__ void load(uint32_t taddr, V &v) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
                       "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
                       "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
                       "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]),
                       "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                     : "r"(taddr));
    }
    static __device__ __forceinline__ void wait(V &v) {
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]),
                       "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]),
                       "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]),
                       "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]),
                       "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])::"memory");
    }
    static __device__ __forceinline__ void store(uint32_t taddr, const V &v) {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
                     "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                     "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
                     "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
                     "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
                     "r"(v[29]), "r"(v[30]), "r"(v[31])
                     : "memory");
    }
};

// Calls use(c, v) for columns c .. c + W - 1 of N from taddr on, each load in
// flight while the columns before it are used.
template <int N, int W, class F>
__device__ __forceinline__ void tmem_each(uint32_t taddr, F &&use) {
    uint32_t v[2][W];
    Tmem<W>::load(taddr, v[0]);
#pragma unroll
    for (int c = 0; c < N; c += W) {
        uint32_t(&now)[W] = v[(c / W) & 1];
        Tmem<W>::wait(now);
        if (c + W < N) Tmem<W>::load(taddr + (uint32_t)(c + W), v[((c / W) & 1) ^ 1]);
        use(c, now);
    }
}

// Pairs at a time: sm_100 adds and multiplies two f32 in one instruction, and
// takes an fp16 half from an f32 in one.
struct F2 {
    float x, y;
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 d;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 d;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 d;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ F2 pair(uint32_t a, uint32_t b) { return {__uint_as_float(a), __uint_as_float(b)}; }
__device__ __forceinline__ F2 both(float a) { return {a, a}; }

__device__ __forceinline__ uint32_t pack_half(F2 a) {
    const __half2 v = __floats2half2_rn(a.x, a.y);
    return *reinterpret_cast<const uint32_t *>(&v);
}
// A pair as fp16: hi, and what hi has too much of it, -lo (the MMAs negate it).
__device__ __forceinline__ void split_half(F2 a, uint32_t &hi, uint32_t &neg_lo) {
    hi = pack_half(a);
    F2 d;
    asm("{\n\t.reg .f16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.f16 %0, l, %3;\n\tsub.rn.f32.f16 %1, h, %4;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "r"(hi), "f"(a.x), "f"(a.y));
    neg_lo = pack_half(d);
}
// The power of two that brings a magnitude with these bits to [2^13, 2^14), and
// its inverse (both normal: magnitudes below 2^-112 get 2^126).
__device__ __forceinline__ float up_scale(uint32_t bits) {
    const int e = (int)(bits >> 23);
    return e == 255 ? 1.0f : __uint_as_float((uint32_t)(267 - e < 253 ? 267 - e : 253) << 23);
}
__device__ __forceinline__ float down_scale(float up) { return __uint_as_float((254u << 23) - __float_as_uint(up)); }

// The bits of the largest magnitude of eight f32 (NaN left out).
__device__ __forceinline__ uint32_t most_of(const float4 &a, const float4 &b) {
    const float x = fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w)));
    const float y = fmaxf(fmaxf(fabsf(b.x), fabsf(b.y)), fmaxf(fabsf(b.z), fabsf(b.w)));
    return __float_as_uint(fmaxf(fmaxf(x, y), 0.0f));
}

// Byte offset of 16-byte chunk c of row r in a 128-byte swizzled sub-tile.
__device__ __forceinline__ uint32_t swizzled(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ void store_shared(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Eight f32 values times s as fp16 halves hi and -lo.
__device__ __forceinline__ void halves(const float4 &a, const float4 &b, float s, uint4 &hi, uint4 &lo) {
    split_half(mul2({a.x, a.y}, both(s)), hi.x, lo.x);
    split_half(mul2({a.z, a.w}, both(s)), hi.y, lo.y);
    split_half(mul2({b.x, b.y}, both(s)), hi.z, lo.z);
    split_half(mul2({b.z, b.w}, both(s)), hi.w, lo.w);
}
// A pair of bf16 times a power of two (exact) as fp16.
__device__ __forceinline__ uint32_t to_half(uint32_t u, __nv_bfloat162 s) {
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&u), s);
    u = *reinterpret_cast<const uint32_t *>(&v);
    return pack_half(pair(u << 16, u & 0xffff0000u));
}
// The larger magnitudes of two pairs, with signs of no meaning (NaN is left out).
__device__ __forceinline__ uint32_t max_abs_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// How far values may spread, in powers of two: the largest of a few neighbours
// below their tile's largest.  The neighbours are eight elements of a row (of bf16
// the four even or the four odd ones), and a thread's N rows of a column.  (Of a
// single row an element is no group: an ordinary one is small now and then.
// Sequences too short for two rows a thread have a check of their own, short_wide.)
constexpr int kSpread = 16;
// The largest magnitude (as f32 bits) of a thread's share of a tile, eight elements
// of each of N rows, and the least of its rows' largest, less one step of their
// bits, so that zeros come out above all others.
template <bool F32, int N>
__device__ __forceinline__ void rows_spread(const uint4 (&v)[N * (F32 ? 2 : 1)], uint32_t &most, uint32_t &least) {
    if constexpr (F32) {
        most = 0, least = 0xffffffffu;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t m = most_of(*reinterpret_cast<const float4 *>(&v[2 * k]),
                                       *reinterpret_cast<const float4 *>(&v[2 * k + 1]));
            most = max(most, m);
            least = min(least, m - 1);
        }
    } else {  // two bf16 a register
        uint32_t hi = 0, lo = 0xffffffffu;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t m = max_abs_bf16x2(max_abs_bf16x2(v[k].x, v[k].y), max_abs_bf16x2(v[k].z, v[k].w)) & 0x7fff7fffu;
            hi = max_abs_bf16x2(hi, m);
            lo = min_u16x2(lo, __vsub2(m, 0x00010001u));
        }
        most = max(hi << 16, hi & 0xffff0000u);
        least = min(lo << 16, lo & 0xffff0000u);
    }
}
// The same least of its columns.
template <bool F32, int N>
__device__ __forceinline__ uint32_t columns_spread(const uint4 (&v)[N * (F32 ? 2 : 1)]) {
    if constexpr (F32) {
        uint32_t least = 0xffffffffu;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            float m = 0.0f;
#pragma unroll
            for (int k = 0; k < N; ++k) m = fmaxf(m, fabsf((&reinterpret_cast<const float4 *>(&v[2 * k + x / 4])->x)[x % 4]));
            least = min(least, __float_as_uint(m) - 1);
        }
        return least;
    } else {
        uint32_t m[4] = {0, 0, 0, 0}, lo = 0xffffffffu;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            m[0] = max_abs_bf16x2(m[0], v[k].x), m[1] = max_abs_bf16x2(m[1], v[k].y);
            m[2] = max_abs_bf16x2(m[2], v[k].z), m[3] = max_abs_bf16x2(m[3], v[k].w);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) lo = min_u16x2(lo, __vsub2(m[x] & 0x7fff7fffu, 0x00010001u));
        return min(lo << 16, lo & 0xffff0000u);
    }
}
template <bool F32>
__device__ __forceinline__ bool too_wide(uint32_t most, uint32_t least) {
    constexpr uint32_t step = F32 ? 1 : 0x10000;
    return least < 0x80000000u && (int)(most >> 23) - (int)((least + step) >> 23) > kSpread;
}

// Barrier of the loader's 128 threads that also says whether any of them has p.
__device__ __forceinline__ bool loader_or(bool p) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
        : "=r"(r)
        : "r"((uint32_t)p)
        : "memory");
    return r != 0;
}

// Whether the columns of the values of a sequence of `n` keys, at most 32, spread
// too far, by a whole warp.
template <bool F32>
__device__ __forceinline__ bool short_wide_of(const PagesView &p, int layer, int j, const int32_t *table, int n) {
    const int page_mask = (1 << p.page_shift) - 1;
    const size_t first = page_elem(p, layer, 1, table[0], j);
    const size_t second = n > page_mask + 1 ? page_elem(p, layer, 1, table[1], j) : first;
    uint32_t most = 0, least = 0xffffffffu;
    for (int d = threadIdx.x & 31; d < p.head; d += 32) {
        float m = 0.0f;
#pragma unroll 8
        for (int t = 0; t < n; ++t) {
            const size_t e = (t > page_mask ? second : first) + (size_t)(t & page_mask) * p.head + d;
            if constexpr (F32) m = fmaxf(m, fabsf(static_cast<const float *>(p.kv)[e]));
            else m = fmaxf(m, fabsf(__bfloat162float(static_cast<const __nv_bfloat16 *>(p.kv)[e])));
        }
        most = max(most, __float_as_uint(m));
        least = min(least, __float_as_uint(m) - 1);
    }
    return too_wide<true>(__reduce_max_sync(0xffffffffu, most), __reduce_min_sync(0xffffffffu, least));
}
__device__ __noinline__ bool short_wide(const PagesView &p, int layer, int j, const int32_t *table, int n) {
    return p.f32 ? short_wide_of<true>(p, layer, j, table, n) : short_wide_of<false>(p, layer, j, table, n);
}

// The rows of a warp whose bits are in `rest` attended again, four at a time: a
// lane's row has its query at q + at and its values at o + to, the result or, with
// ml, a part's.
__device__ __noinline__ void attend_again(const PagesView &p, int layer, int j, const int32_t *table, const float *q,
                                          float *o, float2 *ml, size_t at, size_t to, int lo, int limit, unsigned rest) {
    constexpr int R = 4;
    const int lane = threadIdx.x & 31;
    while (rest) {
        const float *qs[R];
        int his[R], of[R];
#pragma unroll
        for (int x = 0; x < R; ++x) {  // (the last again where there are fewer)
            of[x] = rest ? __ffs((int)rest) - 1 : of[x - 1];
            rest &= rest - 1;
            qs[x] = q + __shfl_sync(0xffffffffu, at, of[x]);
            his[x] = __shfl_sync(0xffffffffu, limit, of[x]);
        }
        RowAcc a[R];
        attend_rows<R>(p, layer, j, table, qs, lo, his, a);
#pragma unroll
        for (int x = 0; x < R; ++x) {
            float *dst = o + __shfl_sync(0xffffffffu, to, of[x]);
            const float l = ml ? 1.0f : a[x].l;
#pragma unroll
            for (int i = 0; i < kHeadMax / 32; ++i)
                if (lane + 32 * i < p.head) dst[lane + 32 * i] = a[x].o[i] / l;
            if (ml && lane == of[x]) *ml = make_float2(a[x].m, a[x].l);
        }
    }
}

template <int T>
struct Tile {  // a number known at compile time
    __device__ __forceinline__ constexpr operator int() const { return T; }
};

template <int D, bool F32>
__global__ void __launch_bounds__(kPromptThreads, 1)
    k_pages_prompt(PagesView p, int layer, const StepSeq *__restrict__ seqs, const AttnItem *__restrict__ items,
                   AttnScratch scratch, const float *__restrict__ q, float *__restrict__ out, int *err, float scale,
                   float top) {
    using S = Shape<D, F32>;
    constexpr int Keys = S::Keys, W = S::Wide;
    extern __shared__ unsigned char raw_smem[];
    __shared__ uint64_t slot_full[S::Slots], slot_empty[S::Slots], s_full[3], p_full[2], o_full[2], o_free, q_full, done;
    __shared__ uint32_t s_tmem, s_red[2][4][2];
    __shared__ float s_kscale[kScaleRing], s_vscale[kScaleRing];
    __shared__ int s_abort;
    const uint32_t base = (smem_addr(raw_smem) + 1023u) & ~1023u;
    const uint32_t slots = base + 2 * S::QTile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort_flag = &s_abort;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::Slots; ++i) {
            mbar_init(&slot_full[i], 4);
            mbar_init(&slot_empty[i], 1);
        }
        for (int b = 0; b < 3; ++b) mbar_init(&s_full[b], 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&p_full[t], 4);
            mbar_init(&o_full[t], 1);
        }
        mbar_init(&o_free, 4);
        mbar_init(&q_full, 8);
        mbar_init(&done, 1);
        s_abort = 0;
        mbar_fence_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    const int item = (int)(blockIdx.x / (unsigned)p.kv_heads), j = (int)(blockIdx.x % (unsigned)p.kv_heads);
    const AttnItem it = items[item];
    const StepSeq sq = seqs[it.seq];
    const int32_t *table = p.table + (size_t)sq.slot * p.max_pages;
    // key tiles of a query tile: up to the last position any of its rows sees
    const auto tiles_of = [&](int t) {
        const int last = min(it.rows, 128 * (t + 1)) - 1;
        const int seen = min(it.hi, sq.ctx + (it.row + last) / p.group + 1) - it.lo;
        return last < 128 * t || seen <= 0 ? 0 : (seen + Keys - 1) / Keys;
    };
    // (rows ascend, so n0 <= n1 unless there is no second tile)
    const int n0 = tiles_of(0), n1 = tiles_of(1), n = max(n0, n1);
    wait_before();
    // The order of the work on (key tile i, query tile t): the s-th takes score
    // buffer s % 3.
    //   s = 2 i + t while both tiles have keys, then n0 + i; n1 = 0: s = i

    const auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return true;
        const uint32_t t0 = (uint32_t)clock();
        while (!mbar_try_wait(bar, parity)) {
            if (*abort_flag) return false;
            if ((uint32_t)clock() - t0 > 1u << 31) {  // about a second
                if (err) atomicOr(err, ERR_TIMEOUT);
                *abort_flag = 1;
                return false;
            }
        }
        return true;
    };

    if (warp < 8) {
        // ---- a thread per query row -----------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int t = warp >> 2, r = threadIdx.x;  // r = 128 t + row of the tile
        const bool live = r < it.rows;
        const int m_row = it.row + (live ? r : 0), token = m_row / p.group;
        const size_t at =
            ((size_t)(sq.row0 + token) * p.heads + (size_t)j * p.group + (m_row - token * p.group)) * p.head;
        const int limit = live ? min(it.hi, sq.ctx + token + 1) : it.lo;
        float down;  // the scale of the row's halves, taken back
        {  // the row's halves, scaled to its largest element
            const int chunks = p.head >> 3;
            const float4 *src = reinterpret_cast<const float4 *>(q + at);
            float4 x[D / 4];  // (the registers of acc)
#pragma unroll
            for (int c = 0; c < D / 4; ++c)
                x[c] = live && c < 2 * chunks ? __ldg(src + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            uint32_t most = 0;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) most = max(most, most_of(x[2 * c], x[2 * c + 1]));
            const float up = up_scale(most);
            down = most == 0x7f800000u ? INFINITY : down_scale(up);
            const uint32_t tile = base + (uint32_t)t * S::QTile;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                uint4 hi, lo;
                halves(x[2 * c], x[2 * c + 1], up, hi, lo);
                const uint32_t o = tile + (uint32_t)(c >> 3) * 16384 + swizzled(r & 127, c & 7);
                store_shared(o, hi);
                store_shared(o + (D / 64) * 16384, lo);
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
        }

        F2 acc[D / 2];
#pragma unroll
        for (int d = 0; d < D / 2; ++d) acc[d] = both(0.0f);
        float m = -INFINITY, l = 0.0f;
        float f = 0.0f;      // the weights' own scale in the last tile, 2^(its maximum - m)
        float e = 0.0f;      // what acc may be off by, less kLost
        // the row is attended again in f32
        bool again = it.lo == 0 && it.hi < 2 * S::Step && short_wide(p, layer, j, table, it.hi);
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t o_at = tmem + lanes + (uint32_t)(S::SumAt + (S::Sums == 2 ? t * D : 0));
        // the sum of V over a key tile, once it is there, into the registers
        const auto flush = [&](int tile) {
            if (!__all_sync(0xffffffffu, wait(&o_full[t], (uint32_t)tile & 1u))) return false;
            tc_fence_after();
            const float mark = s_vscale[tile & (kScaleRing - 1)], vs = f * fabsf(mark);
            e += vs;
            again = again || (mark < 0.0f && limit > it.lo + tile * Keys);
            tmem_each<D, W>(o_at, [&](int c, uint32_t(&v)[W]) {
#pragma unroll
                for (int i = 0; i < W / 2; ++i)
                    acc[c / 2 + i] = fma2(pair(v[2 * i], v[2 * i + 1]), both(vs), acc[c / 2 + i]);
            });
            if constexpr (S::Sums == 1) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&o_free);
            }
            return true;
        };
        bool ok = true;
        const int mine = t ? n1 : n0;
        int buf = t && n0 > 0;  // s = t, or 0 where tile 1 is alone
        uint32_t round = 0;
        for (int tile = 0; ok && tile < mine; ++tile) {
            ok = __all_sync(0xffffffffu, wait(&s_full[buf], round));
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_at = tmem + lanes + (uint32_t)(buf * Keys);
            buf += n1 > 0 && tile + 1 < (t ? n0 : mine) ? 2 : 1;
            if (buf >= 3) buf -= 3, round ^= 1;
            const int rem = limit - (it.lo + tile * Keys);  // the tile's keys this row sees
            const bool masked = __any_sync(0xffffffffu, rem < Keys);
            // (the powers of two first: their product is exact, or far out of use)
            const float ks = scale * (down * s_kscale[tile & (kScaleRing - 1)]);
            again = again || (rem > 0 && ks > top);
            float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            // (rolled loops: the roles' code competes for the instruction caches)
#pragma unroll 1
            for (int c = 0; c < Keys; c += 32) {
                uint32_t v[32];
                Tmem<32>::load(s_at + (uint32_t)c, v);
                Tmem<32>::wait(v);
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c + i >= rem) v[i] = 0xff800000u;  // -inf
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) part[i & 3] = fmaxf(part[i & 3], __uint_as_float(v[i]));
            }
            const float mx = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
            if (S::Sums == 2 && tile && !(ok = flush(tile - 1))) break;
            const float mt = mx * ks, mn = fmaxf(m, mt);
            if (tile && __any_sync(0xffffffffu, mn > m)) {
                const float keep = mn == -INFINITY ? 0.0f : ex2(m - mn);
                l *= keep;
                e *= keep;
#pragma unroll
                for (int d = 0; d < D / 2; ++d) acc[d] = mul2(acc[d], both(keep));
            }
            m = mn;
            // weights relative to the tile's own largest, times 2^14: the halves of
            // small ones stay normal numbers (mt: -inf or NaN where the row sees no
            // finite score)
            const bool some = mt > -INFINITY;
            const float bias = 14.0f - (some ? mt : 0.0f);
            F2 sum[2] = {both(0.0f), both(0.0f)};
            const auto weights = [&](auto some_masked) {
#pragma unroll 1
                for (int c = 0; c < Keys; c += W) {
                    uint32_t v[W], h[W];
                    Tmem<W>::load(s_at + (uint32_t)c, v);
                    Tmem<W>::wait(v);
                    // in place: W / 2 columns of the halves hi, W / 2 of -lo
#pragma unroll
                    for (int i = 0; i < W / 2; ++i) {
                        const F2 x = fma2(pair(v[2 * i], v[2 * i + 1]), both(ks), both(bias));
                        F2 w{ex2(x.x), ex2(x.y)};
                        if (some_masked) {
                            if (c + 2 * i >= rem) w.x = 0.0f;
                            if (c + 2 * i + 1 >= rem) w.y = 0.0f;
                        }
                        sum[i & 1] = add2(sum[i & 1], w);
                        split_half(w, h[i], h[W / 2 + i]);
                    }
                    Tmem<W>::store(s_at + (uint32_t)c, h);
                }
            };
            if (masked) weights(Tile<1>{});
            else weights(Tile<0>{});
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t]);
            f = some ? ex2(mt - m) : 0.0f;
            l = __fmaf_rn((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y), f, l);
            if (S::Sums == 1) ok = flush(tile);
        }
        if (S::Sums == 2 && ok && mine) ok = flush(mine - 1);
        if (ok) {
            bool fine = isfinite(l);
            float most = 0.0f;
#pragma unroll
            for (int d = 0; d < D / 2; ++d) {
                fine = fine && isfinite(acc[d].x) && isfinite(acc[d].y);
                most = fmaxf(most, fmaxf(fabsf(acc[d].x), fabsf(acc[d].y)));
            }
            fine = fine && most >= e * kLost;
            fine = fine || l != l;  // (a NaN score among the row's own: dividing by l says so)
            fine = fine && !again;
            const size_t part = ((size_t)item * p.kv_heads + j) * kRows + r;
            if (live && fine) {
                const float f = it.n_parts == 1 ? 1.0f / l : 0x1p-14f;
                float4 *dst = reinterpret_cast<float4 *>(it.n_parts == 1 ? out + at : scratch.o + part * p.head);
#pragma unroll
                for (int d = 0; d < D / 2; d += 2)
                    if (2 * d < p.head)
                        dst[d / 2] = make_float4(acc[d].x * f, acc[d].y * f, acc[d + 1].x * f, acc[d + 1].y * f);
                if (it.n_parts > 1) scratch.ml[part] = make_float2(m, l * 0x1p-14f);
            }
            const unsigned rest = __ballot_sync(0xffffffffu, live && !fine);
            if (rest) {
                const bool whole = it.n_parts == 1;
                attend_again(p, layer, j, table, q, whole ? out : scratch.o, whole ? nullptr : scratch.ml + part, at,
                             whole ? at : part * p.head, it.lo, limit, rest);
            }
        }
    } else if (warp < 12) {
        // ---- the loader: tiles K0 K1 V0 K2 V1 .. V(n-1) ---------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        constexpr int PerRow = D / 8, Step = S::Step;  // eight-element chunks of a row, rows of a step
        constexpr int Loads = Keys / Step;
        const int tid = threadIdx.x - 256, chunk = tid % PerRow, row = tid / PerRow;
        constexpr uint32_t Size = F32 ? 4 : 2;
        const int page_mask = (1 << p.page_shift) - 1;
        const uint32_t row_bytes = (uint32_t)p.head * Size;
        const size_t page_bytes = (size_t)p.kv_heads * ((size_t)row_bytes << p.page_shift);
        const char *k_src = static_cast<const char *>(p.kv) + (page_elem(p, layer, 0, 0, j) + 8 * chunk) * Size +
                            (size_t)row * row_bytes;
        const char *v_src = k_src + (page_elem(p, layer, 1, 0, j) - page_elem(p, layer, 0, 0, j)) * Size;
        // lane i: where positions 16 i .. of a tile lie
        const auto places = [&](int tile) {
            const int pos = it.lo + tile * Keys + 16 * lane;
            if (lane >= Keys / 16 || pos >= it.hi) return (size_t)0;
            return (size_t)__ldg(table + (pos >> p.page_shift)) * page_bytes + (size_t)(pos & page_mask) * row_bytes;
        };
        // rows of a tile that this thread's row 0 is in front of the end by
        const auto room_of = [&](int tile) { return chunk < (p.head >> 3) ? it.hi - (it.lo + tile * Keys) - row : 0; };
        const auto is_v = [&](int i) { return i == 2 * n - 1 || (i > 0 && !(i & 1)); };
        const auto tile_of = [&](int i) { return i == 2 * n - 1 ? n - 1 : is_v(i) ? i / 2 - 1 : (i + 1) / 2; };
        size_t place = places(tile_of(1));  // of the tile after the one in registers
        uint4 v[Loads * (F32 ? 2 : 1)];
        const auto load = [&](int k, const char *src, size_t at, int room) {
            const uint4 *from = reinterpret_cast<const uint4 *>(src + __shfl_sync(0xffffffffu, at, k * Step / 16) +
                                                                (k * Step % 16) * row_bytes);
            const uint4 zero = make_uint4(0, 0, 0, 0);
            const bool in = k * Step < room;
            if constexpr (F32) {
                v[2 * k] = in ? __ldg(from) : zero;
                v[2 * k + 1] = in ? __ldg(from + 1) : zero;
            } else {
                v[k] = in ? __ldg(from) : zero;
            }
        };
        if (n > 0) {
            const size_t first = places(0);
#pragma unroll
            for (int k = 0; k < Loads; ++k) load(k, k_src, first, room_of(0));
        }
        int slot = 0;
        uint32_t freed = 1;  // parity of the slot's last use; the first round finds every slot free
        for (int i = 0; i < 2 * n; ++i) {
            const int next = min(i + 1, 2 * n - 1);
            const size_t place_next = places(tile_of(min(i + 2, 2 * n - 1)));
            // the tile's largest magnitude and, of V, the smallest of its groups'
            // (columns where this thread has rows, not one)
            uint32_t most, least;
            rows_spread<F32, Loads>(v, most, least);
            if (is_v(i)) {
                if (room_of(tile_of(i)) > Step) least = min(least, columns_spread<F32, Loads>(v));
                least = __reduce_min_sync(0xffffffffu, least);
            }
            most = __reduce_max_sync(0xffffffffu, most);
            uint32_t(&red)[4][2] = s_red[i & 1];
            if (lane == 0) {
                red[warp - 8][0] = most;
                red[warp - 8][1] = least;
            }
            const bool ok = wait(&slot_empty[slot], freed);
            if (loader_or(!ok)) break;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                most = max(most, red[w][0]);
                least = min(least, red[w][1]);
            }
            const float up = up_scale(most);
            if (tid == 0) {
                const bool inf = most == 0x7f800000u;
                const bool mark = inf || too_wide<F32>(most, least);
                const float down = down_scale(up);
                if (is_v(i)) s_vscale[tile_of(i) & (kScaleRing - 1)] = mark ? -down : most ? down : 0.0f;
                else s_kscale[tile_of(i) & (kScaleRing - 1)] = inf ? INFINITY : down;
            }
            const uint32_t dst =
                slots + (uint32_t)slot * S::Slot + (uint32_t)(chunk >> 3) * S::Sub + swizzled(row, chunk & 7);
            // a chunk's registers take the next tile's as soon as it is stored
            // (the last tile's load again)
            const char *src = is_v(next) ? v_src : k_src;
            const int room = room_of(tile_of(next));
            const __nv_bfloat162 up2 = __float2bfloat162_rn(up);
#pragma unroll
            for (int k = 0; k < Loads; ++k) {
                uint4 hi, lo;
                if constexpr (F32) {
                    halves(*reinterpret_cast<const float4 *>(&v[2 * k]), *reinterpret_cast<const float4 *>(&v[2 * k + 1]),
                           up, hi, lo);
                } else {
                    hi = make_uint4(to_half(v[k].x, up2), to_half(v[k].y, up2), to_half(v[k].z, up2),
                                    to_half(v[k].w, up2));
                }
                // (row + k Step) & 7 = row & 7: the swizzle is the row's
                store_shared(dst + k * Step * 128, hi);
                if (F32) store_shared(dst + k * Step * 128 + (D / 64) * S::Sub, lo);
                load(k, src, place, room);
            }
            place = place_next;
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&slot_full[slot]);
            if (++slot == S::Slots) slot = 0, freed ^= 1;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
        if (warp == 12) {
            // ---- the MMAs: the warp waits as one, one lane issues ---------------------------------------------------------
            const auto scores = [&](auto t, int slot, int buf) {  // S = (q_hi + q_lo) K^T
                if (!elect_one()) return;
                const uint32_t a = here(k_desc(base + t * S::QTile)), k = here(k_desc(slots + slot * S::Slot));
                const uint32_t d_at = here(tmem + buf * Keys);
#pragma unroll 1
                for (int y = 0; y < S::Parts + 1; ++y) {  // q_lo K_hi, q_hi K_lo, q_hi K_hi
                    const int x = y < S::Parts ? y + 1 : 0;
                    const int qo = x == 1 ? (D / 64) * 16384 : 0, ko = x == 2 ? (D / 64) * S::Sub : 0;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d)
                        mma_ss(d_at, a + ((qo + (d >> 2) * 16384 + (d & 3) * 32) >> 4),
                               k + ((ko + (d >> 2) * S::Sub + (d & 3) * 32) >> 4), idesc<Keys, false>(x == 1, x == 2),
                               y | d);
                }
            };
            const auto values = [&](auto t, int slot, int buf) {  // O = (w_hi + w_lo) V
                if (!elect_one()) return;
                const uint32_t v = here(mn_desc(slots + slot * S::Slot, S::Sub)), w = here(tmem + buf * Keys);
                const uint32_t d_at = here(tmem + S::SumAt + (S::Sums == 2 ? t * D : 0));
#pragma unroll 1
                for (int y = 0; y < S::Parts + 1; ++y) {  // w_lo V_hi, w_hi V_lo, w_hi V_hi
                    const int x = y < S::Parts ? y + 1 : 0;
                    const int vo = x == 2 ? (D / 64) * S::Sub : 0;
#pragma unroll
                    for (int k = 0; k < Keys / 16; ++k)
                        mma_ts(d_at, w + k * 16 / W * W + k * 16 % W / 2 + (x == 1 ? W / 2 : 0), v + ((vo + k * 2048) >> 4),
                               idesc<D, true>(x == 1, x == 2), y | k);
                }
            };
            const auto commit = [&](uint64_t *bar) {
                if (elect_one()) mma_commit(bar);
            };
            const auto wait_all = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
            struct Ring {  // a place in a ring of N, and the parity of its round
                int at;
                uint32_t parity;
                __device__ __forceinline__ void advance(int by, int n) {
                    at += by;
                    if (at >= n) at -= n, parity ^= 1;
                }
            };
            // Tiles of K come at 0, 1, 3, 5 .. of the slots' order, of V at 2, 4
            // .. 2 n - 2 and 2 n - 1.
            Ring kp{0, 0}, vp{n > 1 ? 2 : 1, 0};
            int sb = 0, pb = 0;  // score buffers of the next scores and values
            uint32_t freed = 1;  // parity for o_free: the first sum finds its place free
            bool ok = wait_all(&q_full, 0);
            const auto next_scores = [&](auto t, int tile, bool last_use) {
                if (!wait_all(&slot_full[kp.at], kp.parity)) return false;
                tc_fence_after();
                scores(t, kp.at, sb);
                commit(&s_full[sb]);
                sb = sb == 2 ? 0 : sb + 1;
                if (last_use) {  // by the last query tile that reads it
                    commit(&slot_empty[kp.at]);
                    kp.advance(tile ? 2 : 1, S::Slots);
                }
                return true;
            };
            const auto next_values = [&](auto t, int tile, bool last_use) {
                if (!wait_all(&slot_full[vp.at], vp.parity) || !wait_all(&p_full[t], (uint32_t)tile & 1u)) return false;
                if (S::Sums == 1) {
                    if (!wait_all(&o_free, freed)) return false;
                    freed ^= 1;
                }
                tc_fence_after();
                values(t, vp.at, pb);
                commit(&o_full[t]);
                pb = pb == 2 ? 0 : pb + 1;
                if (last_use) {
                    commit(&slot_empty[vp.at]);
                    vp.advance(tile + 2 < n ? 2 : 1, S::Slots);
                }
                return true;
            };
            // The scores run three pieces of work ahead of the values.
            Tile<0> first;
            Tile<1> second;
            int st = n0 > 0 ? 0 : 1, si = 0;  // the next scores' query and key tile
            const auto advance_scores = [&]() {
                if (si >= n) return true;
                const bool both_have = n1 > 0 && si < n0;
                const bool fine = st ? next_scores(second, si, true) : next_scores(first, si, !both_have);
                if (st == 0 && both_have) st = 1;
                else ++si, st = n0 > si ? 0 : 1;
                return fine;
            };
            for (int k = 0; ok && k < 3; ++k) ok = advance_scores();
            for (int tile = 0; ok && tile < n; ++tile) {
                if (tile < n0) ok = next_values(first, tile, n1 == 0) && advance_scores();
                if (ok && tile < n1) ok = next_values(second, tile, true) && advance_scores();
            }
            commit(&done);  // every MMA issued, finished loop or not
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        mbar_wait_bounded(&done, 0);  // before the TMEM goes
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Joins the pieces of split rows, in the order of the pieces: a warp per row.
__global__ void __launch_bounds__(128) k_pages_join(PagesView p, const StepSeq *__restrict__ seqs,
                                                    const AttnItem *__restrict__ items, AttnScratch scratch,
                                                    float *__restrict__ out) {
    const int item = (int)(blockIdx.x / (unsigned)p.kv_heads), j = (int)(blockIdx.x % (unsigned)p.kv_heads);
    const AttnItem it = items[item];
    if (it.n_parts == 1 || it.first != item) return;
    const StepSeq sq = seqs[it.seq];
    const int lane = threadIdx.x & 31;
    for (int r = 4 * blockIdx.y + (threadIdx.x >> 5); r < it.rows; r += 4 * gridDim.y) {
        const size_t first = ((size_t)it.first * p.kv_heads + j) * kRows + r, step = (size_t)p.kv_heads * kRows;
        float M = -INFINITY;
        for (int i = 0; i < it.n_parts; ++i) M = fmaxf(M, scratch.ml[first + i * step].x);
        float L = 0.0f, acc[kHeadMax / 32] = {};
#pragma unroll 4
        for (int i = 0; i < it.n_parts; ++i) {
            const size_t w = first + i * step;
            const float2 ml = scratch.ml[w];
            const float k = M == -INFINITY ? 0.0f : ex2(ml.x - M);
            L = __fmaf_rn(ml.y, k, L);
#pragma unroll
            for (int x = 0; x < kHeadMax / 32; ++x)
                if (lane + 32 * x < p.head) acc[x] = __fmaf_rn(scratch.o[w * p.head + lane + 32 * x], k, acc[x]);
        }
        const int mr = it.row + r, tok = mr / p.group;
        const size_t at = ((size_t)(sq.row0 + tok) * p.heads + (size_t)j * p.group + (mr - tok * p.group)) * p.head;
#pragma unroll
        for (int x = 0; x < kHeadMax / 32; ++x)
            if (lane + 32 * x < p.head) out[at + lane + 32 * x] = acc[x] / L;
    }
}

template <int D, bool F32>
cudaError_t launch(const PagesView &p, int layer, const StepSeq *seqs, const AttnItem *items, int n_items,
                   const AttnScratch &scratch, const float *q, float *out, int *err, cudaStream_t s) {
    static bool attr_done[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (!attr_done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(k_pages_prompt<D, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)Shape<D, F32>::Smem);
        if (e != cudaSuccess) return e;
        attr_done[dev] = true;
    }
    const cudaError_t e = launch_after(k_pages_prompt<D, F32>, dim3((unsigned)p.kv_heads * (unsigned)n_items),
                                       kPromptThreads, Shape<D, F32>::Smem, s, p, layer, seqs, items, scratch, q, out, err,
                                       kLog2e / std::sqrt((float)p.head), kScoreTop / (float)p.head);
    if (e != cudaSuccess) return e;
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_pages_prompt(const PagesView &p, int layer, const StepSeq *seqs, const AttnItem *items, int n_items,
                                bool split, const AttnScratch &scratch, const float *q, float *out, int *err,
                                cudaStream_t s) {
    if (n_items == 0) return cudaSuccess;
    const cudaError_t e =
        p.head <= 64 ? (p.f32 ? launch<64, true>(p, layer, seqs, items, n_items, scratch, q, out, err, s)
                              : launch<64, false>(p, layer, seqs, items, n_items, scratch, q, out, err, s))
                     : (p.f32 ? launch<128, true>(p, layer, seqs, items, n_items, scratch, q, out, err, s)
                              : launch<128, false>(p, layer, seqs, items, n_items, scratch, q, out, err, s));
    if (e != cudaSuccess || !split) return e;
    k_pages_join<<<dim3((unsigned)p.kv_heads * (unsigned)n_items, 8), 128, 0, s>>>(p, seqs, items, scratch, out);
    count_launch();
    return cudaGetLastError();
}

}  // namespace krt
