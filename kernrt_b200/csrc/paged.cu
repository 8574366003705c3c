// The paged key/value cache on the device: the step's descriptors and page
// tables, the write of new rows, page copies, and attention over the pages.
#include "kernels.cuh"
#include "paged.cuh"
#include "paged_dev.cuh"

namespace krt {

namespace {

cudaError_t launched() {
    count_launch();
    return cudaGetLastError();
}

// One CTA per sequence: its descriptor, and the table entries that changed.
__global__ void __launch_bounds__(128) k_pages_step(const StepSeq *__restrict__ staged, StepSeq *__restrict__ seqs,
                                                    int32_t *__restrict__ table, int max_pages) {
    const StepSeq q = staged[blockIdx.x];
    const int32_t *delta = reinterpret_cast<const int32_t *>(staged + gridDim.x) + q.delta;
    if (threadIdx.x == 0) seqs[blockIdx.x] = q;
    for (int i = threadIdx.x; i < q.n_dirty; i += blockDim.x)
        table[(size_t)q.slot * max_pages + q.dirty + i] = delta[i];
}

// Eight elements of a k or v row per thread; the row's page comes from the
// sequence's table.
__global__ void __launch_bounds__(256) k_pages_write(PagesView p, int layer, const StepSeq *__restrict__ seqs, int n,
                                                     int rows, const float4 *__restrict__ k,
                                                     const float4 *__restrict__ v) {
    const int row_chunks = p.kv_heads * p.head / 8, head_chunks = p.head / 8;
    const size_t total = (size_t)rows * 2 * row_chunks;
    for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        const int c = (int)(i % row_chunks);
        const size_t rk = i / row_chunks;
        const int kv = (int)(rk & 1), r = (int)(rk >> 1);
        const StepSeq &q = seqs[step_seq_of(seqs, n, r)];
        const int t = q.ctx + (r - q.row0);
        const int page = p.table[(size_t)q.slot * p.max_pages + (t >> p.page_shift)];
        const int j = c / head_chunks;
        const size_t e = page_elem(p, layer, kv, page, j) + (size_t)(t & ((1 << p.page_shift) - 1)) * p.head +
                         (size_t)(c - j * head_chunks) * 8;
        const float4 *src = (kv ? v : k) + ((size_t)r * row_chunks + c) * 2;
        const float4 a = __ldg(src), b = __ldg(src + 1);
        if (p.f32) {
            float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(p.kv) + e);
            dst[0] = a;
            dst[1] = b;
        } else {  // round to nearest even, the cache's own precision
            __nv_bfloat162 w[4] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(a.z, a.w),
                                   __floats2bfloat162_rn(b.x, b.y), __floats2bfloat162_rn(b.z, b.w)};
            *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.kv) + e) = *reinterpret_cast<const uint4 *>(w);
        }
    }
}

// One warp per (copy, layer, K or V, kv head): the used rows of a page are
// contiguous there.
__global__ void __launch_bounds__(256) k_pages_copy(PagesView p, const CopyItem *__restrict__ items, size_t units) {
    const int lane = threadIdx.x & 31;
    const int per_copy = p.n_layers * 2 * p.kv_heads;
    const size_t size = p.f32 ? 4 : 2;
    for (size_t u = blockIdx.x * (size_t)(blockDim.x / 32) + (threadIdx.x >> 5); u < units;
         u += (size_t)gridDim.x * (blockDim.x / 32)) {
        const CopyItem c = items[u / per_copy];
        const int rest = (int)(u % per_copy), j = rest % p.kv_heads, lk = rest / p.kv_heads;
        const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const char *>(p.kv) +
                                                           page_elem(p, lk >> 1, lk & 1, c.src, j) * size);
        uint4 *dst =
            reinterpret_cast<uint4 *>(static_cast<char *>(p.kv) + page_elem(p, lk >> 1, lk & 1, c.dst, j) * size);
        const int n = (int)((size_t)c.rows * p.head * size / 16);
#pragma unroll 4
        for (int i = lane; i < n; i += 32) dst[i] = src[i];
    }
}

// One warp per (row, head).
__global__ void __launch_bounds__(128) k_pages_attention_rows(PagesView p, int layer, const StepSeq *__restrict__ seqs,
                                                              int n, int rows, const float *__restrict__ q,
                                                              float *__restrict__ out) {
    const int lane = threadIdx.x & 31;
    const size_t w = blockIdx.x * (size_t)(blockDim.x / 32) + (threadIdx.x >> 5);
    if (w >= (size_t)rows * p.heads) return;
    const int r = (int)(w / p.heads), h = (int)(w % p.heads);
    const StepSeq s = seqs[step_seq_of(seqs, n, r)];
    const size_t at = ((size_t)r * p.heads + h) * p.head;
    const RowAcc a = attend_row(p, layer, h / p.group, p.table + (size_t)s.slot * p.max_pages, q + at, 0,
                                s.ctx + (r - s.row0) + 1);
#pragma unroll
    for (int i = 0; i < kHeadMax / 32; ++i)
        if (lane + 32 * i < p.head) out[at + lane + 32 * i] = a.o[i] / a.l;
}

}  // namespace

cudaError_t launch_pages_step(const StepSeq *staged, int n, StepSeq *seqs, int32_t *table, int max_pages,
                              cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    k_pages_step<<<(unsigned)n, 128, 0, s>>>(staged, seqs, table, max_pages);
    return launched();
}

cudaError_t launch_pages_write(const PagesView &p, int layer, const StepSeq *seqs, int n, int rows, const float *k,
                               const float *v, cudaStream_t s) {
    if (rows == 0) return cudaSuccess;
    const size_t total = (size_t)rows * 2 * (p.kv_heads * p.head / 8), cap = (size_t)device_sms() * 8;
    const size_t grid = (total + 255) / 256;
    k_pages_write<<<(unsigned)(grid < cap ? grid : cap), 256, 0, s>>>(
        p, layer, seqs, n, rows, reinterpret_cast<const float4 *>(k), reinterpret_cast<const float4 *>(v));
    return launched();
}

cudaError_t launch_pages_copy(const PagesView &p, const CopyItem *items, int n, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    const size_t units = (size_t)n * p.n_layers * 2 * p.kv_heads, cap = (size_t)device_sms() * 8;
    const size_t grid = (units + 7) / 8;
    k_pages_copy<<<(unsigned)(grid < cap ? grid : cap), 256, 0, s>>>(p, items, units);
    return launched();
}

cudaError_t launch_pages_attention_rows(const PagesView &p, int layer, const StepSeq *seqs, int n, int rows,
                                        const float *q, float *out, cudaStream_t s) {
    if (rows == 0) return cudaSuccess;
    const size_t warps = (size_t)rows * p.heads;
    k_pages_attention_rows<<<(unsigned)((warps + 3) / 4), 128, 0, s>>>(p, layer, seqs, n, rows, q, out);
    return launched();
}

}  // namespace krt
