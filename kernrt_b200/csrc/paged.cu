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

// One warp per 4 KB of (copy, layer, K or V, kv head), whose used rows are
// contiguous in a page: eight loads in flight a lane, and pieces small enough
// that the last wave is short (measured, 33 pages of 64 x 128 f32, 8 heads, 24
// layers, 830 MB moved: a warp per whole head and page 163 us, 4 KB pieces below).
constexpr int kCopyChunks = 256;  // of 16 bytes
__global__ void __launch_bounds__(256) k_pages_copy(PagesView p, const CopyItem *__restrict__ items, int pieces,
                                                    size_t units) {
    const int lane = threadIdx.x & 31;
    const size_t u = blockIdx.x * (size_t)(blockDim.x / 32) + (threadIdx.x >> 5);
    if (u >= units) return;
    const size_t size = p.f32 ? 4 : 2;
    const size_t head_unit = u / pieces;
    const int per_copy = p.n_layers * 2 * p.kv_heads, first = (int)(u - head_unit * pieces) * kCopyChunks;
    const CopyItem c = items[head_unit / per_copy];
    const int rest = (int)(head_unit % per_copy), j = rest % p.kv_heads, lk = rest / p.kv_heads;
    const int n = (int)((size_t)c.rows * p.head * size / 16) - first;
    const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const char *>(p.kv) +
                                                       page_elem(p, lk >> 1, lk & 1, c.src, j) * size) +
                       first;
    uint4 *dst = reinterpret_cast<uint4 *>(static_cast<char *>(p.kv) + page_elem(p, lk >> 1, lk & 1, c.dst, j) * size) +
                 first;
    uint4 v[kCopyChunks / 32];
#pragma unroll
    for (int i = 0; i < kCopyChunks / 32; ++i)
        if (lane + 32 * i < n) v[i] = src[lane + 32 * i];
#pragma unroll
    for (int i = 0; i < kCopyChunks / 32; ++i)
        if (lane + 32 * i < n) dst[lane + 32 * i] = v[i];
}

// ---- single tokens: attention split over the length ------------------------------
//
// One warp takes 16 positions at a time against 8 query rows with m16n8k16 MMAs
// whose operands it loads straight into registers.  A product over k or over
// the keys may take its terms in any order, so each thread reads 16 contiguous
// bytes and the fragments follow from that: for scores, thread (g, t) = (lane /
// 4, lane % 4) holds elements 32 b + 8 t .. + 7 of key g; for values, elements 64
// b + 8 g .. + 7 of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9.
//
// Precision: f32 queries and weights go in as three bf16 parts (24 bits: x = x1
// + x2 + x3 with each part the rounding of what is left), which a bf16 cache
// multiplies exactly.  The MMA has 16 rows and there are 8 query rows, so parts 1
// and 2 share one MMA (rows 0-7 and 8-15) and part 3 takes a second into the
// accumulator of part 1; a thread then finds the parts of one score in its own
// registers.  An f32 cache is split the same way, and the products down to
// 2^-24 are kept: (x1 + x2) k1, x3 k1, (x1 + x2) k2, x1 k3.
template <int NB>
struct QFrag {  // [block of 32][half of it]: A of parts 1 and 2, and of part 3
    uint32_t a[NB][2][4], c[NB][2][2];
};

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
// The three parts of a pair, and what is left of it after each.
__device__ __forceinline__ void split3(float x, float y, uint32_t &p1, uint32_t &p2, uint32_t &p3) {
    p1 = pack_bf16(x, y);
    x -= __uint_as_float(p1 << 16);
    y -= __uint_as_float(p1 & 0xffff0000u);
    p2 = pack_bf16(x, y);
    x -= __uint_as_float(p2 << 16);
    y -= __uint_as_float(p2 & 0xffff0000u);
    p3 = pack_bf16(x, y);
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Eight elements of a page row: raw bf16 pairs, or f32.
template <bool F32>
struct Chunk;
template <>
struct Chunk<false> {
    uint4 v;
    __device__ __forceinline__ void load(const void *kv, size_t e, bool ok) {
        v = ok ? __ldg(reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(kv) + e)) : make_uint4(0, 0, 0, 0);
    }
};
template <>
struct Chunk<true> {
    float4 v[2];
    __device__ __forceinline__ void load(const void *kv, size_t e, bool ok) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(kv) + e);
        const float4 z = make_float4(0, 0, 0, 0);
        v[0] = ok ? __ldg(p) : z;
        v[1] = ok ? __ldg(p + 1) : z;
    }
};

constexpr int kDecodeWarps = 4;

template <int NB, bool F32>
__global__ void __launch_bounds__(32 * kDecodeWarps)
    k_pages_decode(PagesView p, int layer, const StepSeq *__restrict__ seqs, const AttnItem *__restrict__ items,
                   AttnScratch scratch, const float *__restrict__ q, float *__restrict__ out) {
    constexpr int NV = (NB + 1) / 2;  // blocks of 64 of the values
    constexpr int R = kDecodeRows;
    __shared__ float s_o[kDecodeWarps][R][32 * NB + 4];
    __shared__ float s_m[kDecodeWarps][R], s_l[kDecodeWarps][R];
    __shared__ int s_last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const AttnItem it = items[blockIdx.x];
    const int j = blockIdx.y;
    const StepSeq sq = seqs[it.seq];
    const int32_t *table = p.table + (size_t)sq.slot * p.max_pages;
    const int head = p.head, chunks = head >> 3, page_mask = (1 << p.page_shift) - 1;
    const size_t page_stride = (size_t)p.kv_heads * ((size_t)head << p.page_shift);  // of one page, all heads
    const size_t k_base = page_elem(p, layer, 0, 0, j), v_base = page_elem(p, layer, 1, 0, j);
    // row g: token and head of the group; it sees positions below `limit`
    const int m_row = it.row + g;
    const int token = m_row / p.group;
    const bool live = g < it.rows;
    const int limit = live ? min(it.hi, sq.ctx + token + 1) : 0;
    const size_t q_at = ((size_t)(sq.row0 + token) * p.heads + (size_t)j * p.group + (m_row - token * p.group)) * head;

    QFrag<NB> qf;
    const float scale = kLog2e * rsqrtf((float)head);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int c = 4 * b + t;
        float4 x0 = make_float4(0, 0, 0, 0), x1 = x0;
        if (live && c < chunks) {
            x0 = __ldg(reinterpret_cast<const float4 *>(q + q_at) + 2 * c);
            x1 = __ldg(reinterpret_cast<const float4 *>(q + q_at) + 2 * c + 1);
        }
        split3(x0.x, x0.y, qf.a[b][0][0], qf.a[b][0][1], qf.c[b][0][0]);
        split3(x0.z, x0.w, qf.a[b][0][2], qf.a[b][0][3], qf.c[b][0][1]);
        split3(x1.x, x1.y, qf.a[b][1][0], qf.a[b][1][1], qf.c[b][1][0]);
        split3(x1.z, x1.w, qf.a[b][1][2], qf.a[b][1][3], qf.c[b][1][1]);
    }

    float o[NV][8][4];
#pragma unroll
    for (int b = 0; b < NV; ++b)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[b][i][x] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // this warp's tiles: 16 positions at lo + 16 warp, step 64; a tile never
    // leaves its page
    const int t0 = it.lo + 16 * warp;
    const int n_tiles = it.hi > t0 ? (it.hi - t0 + kDecodeKeys - 1) / kDecodeKeys : 0;
    int pages = 0;  // lane i: the page of tile i of the current 32
    for (int tile = 0; tile < n_tiles; ++tile) {
        if ((tile & 31) == 0) {
            const int at = t0 + kDecodeKeys * (tile + lane);
            pages = at < it.hi ? __ldg(table + (at >> p.page_shift)) : 0;
        }
        const int pos = t0 + kDecodeKeys * tile;
        const size_t row0 = (size_t)__shfl_sync(0xffffffffu, pages, tile & 31) * page_stride +
                            (size_t)(pos & page_mask) * head;
        Chunk<F32> kc[2][NB], vc[NV][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int b = 0; b < NB; ++b)
                kc[u][b].load(p.kv, k_base + row0 + (size_t)(8 * u + g) * head + 8 * (4 * b + t),
                              4 * b + t < chunks && pos + 8 * u + g < it.hi);
#pragma unroll
        for (int b = 0; b < NV; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 2 * t + (i & 1) + 8 * (i >> 1);
                vc[b][i].load(p.kv, v_base + row0 + (size_t)key * head + 8 * (8 * b + g),
                              8 * b + g < chunks && pos + key < it.hi);
            }

        float s[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if constexpr (F32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t k1[2], k2[2], k3[2];
                        split3(kc[u][b].v[h].x, kc[u][b].v[h].y, k1[0], k2[0], k3[0]);
                        split3(kc[u][b].v[h].z, kc[u][b].v[h].w, k1[1], k2[1], k3[1]);
                        const uint32_t(&a)[4] = qf.a[b][h];
                        mma16816(c, a[0], a[1], a[2], a[3], k1[0], k1[1]);
                        mma16816(c, a[0], a[1], a[2], a[3], k2[0], k2[1]);
                        mma16816(c, a[0], 0, a[2], 0, k3[0], k3[1]);
                        mma16816(c, qf.c[b][h][0], 0, qf.c[b][h][1], 0, k1[0], k1[1]);
                    }
                } else {
                    const uint32_t k[4] = {kc[u][b].v.x, kc[u][b].v.y, kc[u][b].v.z, kc[u][b].v.w};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t(&a)[4] = qf.a[b][h];
                        mma16816(c, a[0], a[1], a[2], a[3], k[2 * h], k[2 * h + 1]);
                        mma16816(c, qf.c[b][h][0], 0, qf.c[b][h][1], 0, k[2 * h], k[2 * h + 1]);
                    }
                }
            }
            // rows 0-7 hold parts 1 and 3, rows 8-15 part 2 of the same score
            const int at = pos + 8 * u + 2 * t;
            s[u][0] = at < limit ? (c[0] + c[2]) * scale : -INFINITY;
            s[u][1] = at + 1 < limit ? (c[1] + c[3]) * scale : -INFINITY;
        }
        float mt = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        if (__any_sync(0xffffffffu, mt > m)) {
            const float mn = fmaxf(m, mt);
            const float keep = mn == -INFINITY ? 0.0f : ex2(m - mn);
            m = mn;
            l *= keep;
#pragma unroll
            for (int b = 0; b < NV; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[b][i][x] *= keep;
        }
        // a row that has seen only -inf keeps weights of 0
        const float mb = m == -INFINITY ? 0.0f : m;
        uint32_t pa[4], pc[2];
        {
            const float w0 = ex2(s[0][0] - mb), w1 = ex2(s[0][1] - mb), w2 = ex2(s[1][0] - mb), w3 = ex2(s[1][1] - mb);
            l += (w0 + w1) + (w2 + w3);
            split3(w0, w1, pa[0], pa[1], pc[0]);
            split3(w2, w3, pa[2], pa[3], pc[1]);
        }
#pragma unroll
        for (int b = 0; b < NV; ++b) {
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float e[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) e[x] = (&vc[b][x].v[i >> 2].x)[i & 3];
                    uint32_t v1[2], v2[2], v3[2];
                    split3(e[0], e[1], v1[0], v2[0], v3[0]);
                    split3(e[2], e[3], v1[1], v2[1], v3[1]);
                    mma16816(o[b][i], pa[0], pa[1], pa[2], pa[3], v1[0], v1[1]);
                    mma16816(o[b][i], pa[0], pa[1], pa[2], pa[3], v2[0], v2[1]);
                    mma16816(o[b][i], pa[0], 0, pa[2], 0, v3[0], v3[1]);
                    mma16816(o[b][i], pc[0], 0, pc[1], 0, v1[0], v1[1]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
                    const uint32_t b0 = __byte_perm((&vc[b][0].v.x)[i >> 1], (&vc[b][1].v.x)[i >> 1], sel);
                    const uint32_t b1 = __byte_perm((&vc[b][2].v.x)[i >> 1], (&vc[b][3].v.x)[i >> 1], sel);
                    mma16816(o[b][i], pa[0], pa[1], pa[2], pa[3], b0, b1);
                    mma16816(o[b][i], pc[0], 0, pc[1], 0, b0, b1);
                }
            }
        }
    }

    // the CTA's warps meet in shared memory
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
        s_m[warp][g] = m;
        s_l[warp][g] = l;
    }
#pragma unroll
    for (int b = 0; b < NV; ++b)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int d = 64 * b + 8 * (2 * t + x) + i;
                if (d < 32 * NB) s_o[warp][g][d] = o[b][i][x] + o[b][i][2 + x];
            }
    __syncthreads();
    const size_t piece = (size_t)blockIdx.x * p.kv_heads + j;
    // warp w: rows w, w + 4; lane: elements lane + 32 i
    for (int r = warp; r < it.rows; r += kDecodeWarps) {
        float M = s_m[0][r];
#pragma unroll
        for (int w = 1; w < kDecodeWarps; ++w) M = fmaxf(M, s_m[w][r]);
        RowAcc a;
        a.m = M;
        a.l = 0.0f;
#pragma unroll
        for (int i = 0; i < kHeadMax / 32; ++i) a.o[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) {
            const float k = M == -INFINITY ? 0.0f : ex2(s_m[w][r] - M);
            a.l = __fmaf_rn(s_l[w][r], k, a.l);
#pragma unroll
            for (int i = 0; i < NB; ++i) a.o[i] = __fmaf_rn(s_o[w][r][lane + 32 * i], k, a.o[i]);
        }
        // A masked key's NaN or infinity has weight 0 and still makes NaN, and
        // parts of an infinity are no parts: such a row is attended again in
        // f32, over its own positions only.
        bool fine = isfinite(a.l);
#pragma unroll
        for (int i = 0; i < NB; ++i) fine = fine && isfinite(a.o[i]);
        const int mr = it.row + r, tok = mr / p.group;
        const size_t at = ((size_t)(sq.row0 + tok) * p.heads + (size_t)j * p.group + (mr - tok * p.group)) * head;
        if (!__all_sync(0xffffffffu, fine))
            a = attend_row(p, layer, j, table, q + at, it.lo, min(it.hi, sq.ctx + tok + 1));
        if (it.n_parts == 1) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (lane + 32 * i < head) out[at + lane + 32 * i] = a.o[i] / a.l;
        } else {
            const size_t w = piece * R + r;
            if (lane == 0) scratch.ml[w] = make_float2(a.m, a.l);
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (lane + 32 * i < head) scratch.o[w * head + lane + 32 * i] = a.o[i];
        }
    }
    if (it.n_parts == 1) return;

    // The piece that arrives last joins all, in the order of the pieces.
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned *count = scratch.count + (size_t)it.join * p.kv_heads + j;
        s_last = atomicAdd(count, 1u) == (unsigned)it.n_parts - 1;
        if (s_last) *count = 0;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    for (int r = warp; r < it.rows; r += kDecodeWarps) {
        const size_t first = ((size_t)it.first * p.kv_heads + j) * R + r, step = (size_t)p.kv_heads * R;
        float M = -INFINITY;
        for (int i = lane; i < it.n_parts; i += 32) M = fmaxf(M, __ldcg(&scratch.ml[first + i * step]).x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
        float L = 0.0f, acc[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = 0.0f;
#pragma unroll 4
        for (int i = 0; i < it.n_parts; ++i) {
            const size_t w = first + i * step;
            const float2 ml = __ldcg(&scratch.ml[w]);
            const float k = M == -INFINITY ? 0.0f : ex2(ml.x - M);
            L = __fmaf_rn(ml.y, k, L);
#pragma unroll
            for (int x = 0; x < NB; ++x)
                if (lane + 32 * x < head) acc[x] = __fmaf_rn(__ldcg(&scratch.o[w * head + lane + 32 * x]), k, acc[x]);
        }
        const int mr = it.row + r, tok = mr / p.group;
        const size_t at = ((size_t)(sq.row0 + tok) * p.heads + (size_t)j * p.group + (mr - tok * p.group)) * head;
#pragma unroll
        for (int x = 0; x < NB; ++x)
            if (lane + 32 * x < head) out[at + lane + 32 * x] = acc[x] / L;
    }
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
    const int chunks = (int)(((size_t)p.head << p.page_shift) * (p.f32 ? 4 : 2) / 16);
    const int pieces = (chunks + kCopyChunks - 1) / kCopyChunks;
    const size_t units = (size_t)n * p.n_layers * 2 * p.kv_heads * pieces;
    if ((units + 7) / 8 > (size_t)INT32_MAX) return cudaErrorInvalidValue;
    k_pages_copy<<<(unsigned)((units + 7) / 8), 256, 0, s>>>(p, items, pieces, units);
    return launched();
}

cudaError_t launch_pages_decode(const PagesView &p, int layer, const StepSeq *seqs, const AttnItem *items, int n_items,
                                const AttnScratch &scratch, const float *q, float *out, cudaStream_t s) {
    if (n_items == 0) return cudaSuccess;
    const dim3 grid((unsigned)n_items, (unsigned)p.kv_heads);
    const auto go = [&](auto kernel) { kernel<<<grid, 32 * kDecodeWarps, 0, s>>>(p, layer, seqs, items, scratch, q, out); };
    const int nb = (p.head + 31) / 32;
    if (p.f32) {
        if (nb == 1) go(k_pages_decode<1, true>);
        else if (nb == 2) go(k_pages_decode<2, true>);
        else if (nb == 3) go(k_pages_decode<3, true>);
        else go(k_pages_decode<4, true>);
    } else {
        if (nb == 1) go(k_pages_decode<1, false>);
        else if (nb == 2) go(k_pages_decode<2, false>);
        else if (nb == 3) go(k_pages_decode<3, false>);
        else go(k_pages_decode<4, false>);
    }
    return launched();
}

}  // namespace krt
