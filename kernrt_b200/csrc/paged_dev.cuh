// Device helpers shared by the paged cache's kernels.
#pragma once

#include <cuda_bf16.h>

#include "paged.cuh"

namespace krt {

// A kernel launched by launch_after may start while the kernel before it on the
// stream still runs, once all its CTAs have called let_next_start (or ended);
// behind wait_before, everything that kernel and those before it did is there.
// What lies before wait_before touches only what older work made (a step's
// descriptors, pieces and tables: pages_write starts after them and is the only
// kernel that lets the next one start).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, A... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// The sequence of the step that holds row r: the last with row0 <= r (row0
// ascends, empty sequences repeat their successor's row0).
__device__ __forceinline__ int step_seq_of(const StepSeq *seqs, int n, int r) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(&seqs[mid].row0) <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// First element of (layer, K or V, page, kv head).
__device__ __forceinline__ size_t page_elem(const PagesView &p, int layer, int kv, int page, int j) {
    return ((((size_t)layer * 2 + kv) * p.n_pages + page) * p.kv_heads + j) * ((size_t)p.head << p.page_shift);
}

constexpr int kHeadMax = 128;  // largest head size
constexpr float kLog2e = 1.4426950408889634f;

// Eight elements from e on (16 or 32 bytes aligned).
template <bool F32>
__device__ __forceinline__ void load_kv8(const PagesView &p, size_t e, float (&x)[8]) {
    if constexpr (F32) {
        const float4 *at = reinterpret_cast<const float4 *>(static_cast<const float *>(p.kv) + e);
        const float4 a = at[0], b = at[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(p.kv) + e);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// R query rows against positions lo .. hi - 1 (a row's own hi) of one kv head, by a
// whole warp in f32: running maximum m of the scaled scores (in powers of two), sum
// l of the weights and weighted values o (lane: elements lane + 32 i).  A weight
// 2^(x - m) with m = -inf (every score so far -inf) counts as 0, so that a
// later finite score takes over; a row with no finite score ends with l = 0 and
// 0 / 0, one with a NaN score is NaN.  What lies in a row's masked places (NaN,
// infinities) cannot reach it.  A lane has one of 32 positions' scores at a time,
// whose loads the R rows share.  Bound by latency: a warp works alone on its rows.
// Measured, every row of a prompt of 2048 tokens, 24 heads of 64: 27.1 ms with a
// row and an element at a time, 1.6 ms with R = 4 and 16 bytes a load.
struct RowAcc {
    float m, l;
    float o[kHeadMax / 32];
};
template <int R, bool F32>
__device__ __forceinline__ void attend_rows_of(const PagesView &view, int layer, int j, const int32_t *table,
                                            const float *const (&q)[R], int lo, const int (&hi)[R], RowAcc (&a)[R]) {
    const PagesView p = view;
    const int lane = threadIdx.x & 31;
    const int mask = (1 << p.page_shift) - 1;
    const float scale = kLog2e * rsqrtf((float)p.head);
    const size_t k_base = page_elem(p, layer, 0, 0, j), to_v = page_elem(p, layer, 1, 0, j) - k_base;
    const size_t page_stride = (size_t)p.kv_heads * ((size_t)p.head << p.page_shift);
    int last = hi[0];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        last = max(last, hi[r]);
        a[r].m = -INFINITY;
        a[r].l = 0.0f;
#pragma unroll
        for (int i = 0; i < kHeadMax / 32; ++i) a[r].o[i] = 0.0f;
    }
    for (int t0 = lo; t0 < last; t0 += 32) {
        // lane: the scores of position t0 + lane
        const int t = t0 + lane;
        const size_t e = t < last ? k_base + (size_t)table[t >> p.page_shift] * page_stride + (size_t)(t & mask) * p.head : 0;
        float w[R];
#pragma unroll
        for (int r = 0; r < R; ++r) w[r] = 0.0f;
        if (t < last) {
#pragma unroll 4
            for (int d = 0; d < p.head; d += 8) {
                float k[8];
                load_kv8<F32>(p, e + d, k);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float4 x = __ldg(reinterpret_cast<const float4 *>(q[r] + d));
                    const float4 y = __ldg(reinterpret_cast<const float4 *>(q[r] + d) + 1);
                    w[r] = __fmaf_rn(x.x, k[0], w[r]), w[r] = __fmaf_rn(x.y, k[1], w[r]);
                    w[r] = __fmaf_rn(x.z, k[2], w[r]), w[r] = __fmaf_rn(x.w, k[3], w[r]);
                    w[r] = __fmaf_rn(y.x, k[4], w[r]), w[r] = __fmaf_rn(y.y, k[5], w[r]);
                    w[r] = __fmaf_rn(y.z, k[6], w[r]), w[r] = __fmaf_rn(y.w, k[7], w[r]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float x = t < hi[r] ? w[r] * scale : -INFINITY;
            float m = x;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            m = fmaxf(m, a[r].m);
            const float keep = m == -INFINITY ? 0.0f : exp2f(a[r].m - m);
            w[r] = t < hi[r] && m != -INFINITY ? exp2f(x - m) : 0.0f;
            if (x != x) w[r] = x;
            float sum = w[r];
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            a[r].m = m;
            a[r].l = __fmaf_rn(a[r].l, keep, sum);
#pragma unroll
            for (int i = 0; i < kHeadMax / 32; ++i) a[r].o[i] *= keep;
        }
        // (four keys' loads first: the branches around the sums would part them)
        const int n = min(32, last - t0);
        for (int s0 = 0; s0 < n; s0 += 4) {
            float v[4][kHeadMax / 32];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const size_t ev = __shfl_sync(0xffffffffu, e, min(s0 + s, n - 1)) + to_v + lane;
#pragma unroll
                for (int i = 0; i < kHeadMax / 32; ++i) {
                    v[s][i] = 0.0f;
                    if (lane + 32 * i >= p.head) continue;
                    if constexpr (F32) v[s][i] = static_cast<const float *>(p.kv)[ev + 32 * i];
                    else v[s][i] = __bfloat162float(static_cast<const __nv_bfloat16 *>(p.kv)[ev + 32 * i]);
                }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float ws = __shfl_sync(0xffffffffu, w[r], s0 + s);
                    if (t0 + s0 + s < hi[r])
#pragma unroll
                        for (int i = 0; i < kHeadMax / 32; ++i) a[r].o[i] = __fmaf_rn(ws, v[s][i], a[r].o[i]);
                }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (a[r].l != a[r].l)  // a NaN score: the whole row is NaN
#pragma unroll
            for (int i = 0; i < kHeadMax / 32; ++i) a[r].o[i] = a[r].l;
}
template <int R>
__device__ __forceinline__ void attend_rows(const PagesView &p, int layer, int j, const int32_t *table,
                                            const float *const (&q)[R], int lo, const int (&hi)[R], RowAcc (&a)[R]) {
    if (p.f32) attend_rows_of<R, true>(p, layer, j, table, q, lo, hi, a);
    else attend_rows_of<R, false>(p, layer, j, table, q, lo, hi, a);
}
static __device__ __noinline__ RowAcc attend_row(const PagesView &p, int layer, int j, const int32_t *table, const float *q,
                                    int lo, int hi) {
    const float *const qs[1] = {q};
    const int his[1] = {hi};
    RowAcc a[1];
    attend_rows<1>(p, layer, j, table, qs, lo, his, a);
    return a[0];
}

}  // namespace krt
