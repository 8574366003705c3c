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

__device__ __forceinline__ float load_kv(const PagesView &p, size_t e) {
    return p.f32 ? static_cast<const float *>(p.kv)[e] : __bfloat162float(static_cast<const __nv_bfloat16 *>(p.kv)[e]);
}

constexpr int kHeadMax = 128;  // largest head size
constexpr float kLog2e = 1.4426950408889634f;

// One query row against positions [lo, hi) of one kv head, by a whole warp in
// f32: running maximum m of the scaled scores (in powers of two), sum l of the
// weights and weighted values o (lane: elements lane + 32 i).  A weight
// 2^(x - m) with m = -inf (every score so far -inf) counts as 0, so that a
// later finite score takes over; a row with no finite score ends with l = 0 and
// 0 / 0.  Only positions of the range are read: what lies in masked places
// (NaN, infinities) cannot reach the row.
struct RowAcc {
    float m, l;
    float o[kHeadMax / 32];
};
static __device__ __noinline__ RowAcc attend_row(const PagesView &p, int layer, int j, const int32_t *table, const float *q, int lo,
                                    int hi) {
    const int lane = threadIdx.x & 31;
    const int mask = (1 << p.page_shift) - 1;
    const float scale = kLog2e * rsqrtf((float)p.head);
    RowAcc a;
    a.m = -INFINITY;
    a.l = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeadMax / 32; ++i) a.o[i] = 0.0f;
    for (int t0 = lo; t0 < hi; t0 += 32) {
        // lane: the score of position t0 + lane
        const int t = t0 + lane;
        float x = -INFINITY;
        if (t < hi) {
            const size_t e = page_elem(p, layer, 0, table[t >> p.page_shift], j) + (size_t)(t & mask) * p.head;
            float dot = 0.0f;
            for (int d = 0; d < p.head; ++d) dot = __fmaf_rn(__ldg(q + d), load_kv(p, e + d), dot);
            x = dot * scale;
        }
        float m = x;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        m = fmaxf(m, a.m);
        const float keep = m == -INFINITY ? 0.0f : exp2f(a.m - m);
        const float w = t < hi && m != -INFINITY ? exp2f(x - m) : 0.0f;
        float sum = w;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        a.m = m;
        a.l = __fmaf_rn(a.l, keep, sum);
#pragma unroll
        for (int i = 0; i < kHeadMax / 32; ++i) a.o[i] *= keep;
        if (a.l != a.l) {  // a NaN score: the whole row is NaN
#pragma unroll
            for (int i = 0; i < kHeadMax / 32; ++i) a.o[i] = a.l;
            break;
        }
        const int n = min(32, hi - t0);
        for (int s = 0; s < n; ++s) {
            const float ws = __shfl_sync(0xffffffffu, w, s);
            const int ts = t0 + s;
            const size_t e = page_elem(p, layer, 1, table[ts >> p.page_shift], j) + (size_t)(ts & mask) * p.head;
#pragma unroll
            for (int i = 0; i < kHeadMax / 32; ++i)
                if (lane + 32 * i < p.head) a.o[i] = __fmaf_rn(ws, load_kv(p, e + lane + 32 * i), a.o[i]);
        }
    }
    return a;
}

}  // namespace krt
