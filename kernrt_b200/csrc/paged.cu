// The paged key/value cache on the device: the step's descriptors and page
// tables, the write of new rows, page copies, and attention over the pages.
#include "kernels.cuh"
#include "paged.cuh"
#include "paged_dev.cuh"

#include <type_traits>

namespace krt {

namespace {

cudaError_t launched() {
    count_launch();
    return cudaGetLastError();
}

// Eight elements of a k or v row per thread; the row's page comes from the
// sequence's table.
__global__ void __launch_bounds__(256) k_pages_write(PagesView p, int layer, const StepSeq *__restrict__ seqs, int n,
                                                     int rows, const float4 *__restrict__ k,
                                                     const float4 *__restrict__ v) {
    let_next_start();
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
// layers, 830 MB moved: a warp per whole head and page 163 us, 4 KB pieces 138).
constexpr int kCopyChunks = 256;  // of 16 bytes
struct Copies {
    const CopyItem *items;
    int pieces;    // of a head's part of a page
    size_t units;  // pieces in all
};
__device__ __forceinline__ void copy_piece(const PagesView &p, const Copies &copies, size_t u) {
    if (u >= copies.units) return;
    const int lane = threadIdx.x & 31;
    const size_t size = p.f32 ? 4 : 2;
    const size_t head_unit = u / copies.pieces;
    const int per_copy = p.n_layers * 2 * p.kv_heads, first = (int)(u - head_unit * copies.pieces) * kCopyChunks;
    const CopyItem c = copies.items[head_unit / per_copy];
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

__global__ void __launch_bounds__(256) k_pages_copy(PagesView p, Copies copies) {
    copy_piece(p, copies, blockIdx.x * (size_t)8 + (threadIdx.x >> 5));
}

Copies copies_of(const PagesView &p, const CopyItem *items, int n) {
    Copies c{items, 0, 0};
    const int chunks = (int)(((size_t)p.head << p.page_shift) * (p.f32 ? 4 : 2) / 16);
    c.pieces = (chunks + kCopyChunks - 1) / kCopyChunks;
    c.units = (size_t)n * p.n_layers * 2 * p.kv_heads * c.pieces;
    return c;
}

// A step's first n CTAs bring a sequence's descriptor and the table entries
// that changed; the others copy the shared pages that sequences grow into.
__global__ void __launch_bounds__(256) k_pages_step(PagesView p, const StepSeq *__restrict__ staged, int n,
                                                    StepSeq *__restrict__ seqs, int32_t *__restrict__ table,
                                                    Copies copies) {
    if (blockIdx.x >= (unsigned)n) {
        copy_piece(p, copies, (blockIdx.x - (unsigned)n) * (size_t)8 + (threadIdx.x >> 5));
        return;
    }
    const StepSeq q = staged[blockIdx.x];
    const int32_t *delta = reinterpret_cast<const int32_t *>(staged + n) + q.delta;
    if (threadIdx.x == 0) seqs[blockIdx.x] = q;
    for (int i = threadIdx.x; i < q.n_dirty; i += blockDim.x)
        table[(size_t)q.slot * p.max_pages + q.dirty + i] = delta[i];
}

// ---- single tokens: attention split over the length ------------------------------
//
// One warp takes 16 positions at a time against 8 query rows with m16n8k16 MMAs.
// Its tiles come through a ring in shared memory of its own (cp.async, no
// barrier beyond the warp's), so that several are in flight while one is used.
// A product over k or over the keys may take its terms in any order, so each
// thread reads 16 contiguous bytes (32 of f32) and the fragments follow from
// that: for scores, thread (g, t) = (lane / 4, lane % 4) holds elements 32 b + 8 t ..
// + 7 of column g, which is key 8 u + 4 (g % 2) + g / 2 of the tile; for values,
// elements 64 b + 8 g .. + 7 of keys t, t + 4, t + 8, t + 12, the ones whose weights
// are in its registers.  A row's 16-byte chunks are swizzled (swap) so that the
// eight lanes of a shared-memory access reach all banks.
//
// Precision: f32 queries and weights go in as three bf16 parts (24 bits: x = x1
// + x2 + x3 with each part the rounding of what is left), which a bf16 cache
// multiplies exactly.  The MMA has 16 rows and there are 8 query rows, so parts 1
// and 2 share one MMA (rows 0-7 and 8-15) and part 3 takes a second into the
// accumulator of part 1; a thread then finds the parts of one score in its own
// registers.  An f32 cache is split the same way, and the products down to
// 2^-24 are kept: (x1 + x2) k1, x3 k1, (x1 + x2) k2, x1 k3.  The MMAs add with
// truncation, so the small products are summed apart from the large ones, and
// after every 16 tiles (4 for wide f32 heads) the sums go to shared memory, where
// they are added with rounding (added in registers after every tile, one token of
// 64 sequences of 100 to 8000 keys, 16 heads of 128, took 207 us instead of 177).
// Bound by HBM: 131072 keys of 8 kv heads of 128 in bf16 take 91.5 us, 5.9 TB/s.
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
    __device__ __forceinline__ void load(const unsigned char *row, int c, int swap) {
        v = *reinterpret_cast<const uint4 *>(row + ((c ^ swap) << 4));
    }
};
template <>
struct Chunk<true> {
    float4 v[2];
    __device__ __forceinline__ void load(const unsigned char *row, int c, int swap) {
        v[0] = *reinterpret_cast<const float4 *>(row + (((2 * c) ^ swap) << 4));
        v[1] = *reinterpret_cast<const float4 *>(row + (((2 * c + 1) ^ swap) << 4));
    }
};
template <bool F32>
__device__ __forceinline__ int k_swap(int row) { return F32 ? row >> 2 & 1 : row & 7; }
template <bool F32>
__device__ __forceinline__ int v_swap(int row) { return F32 ? (row & 1) | (row & 2) << 1 : (row & 3) << 1; }

// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

template <int NB, bool F32>
struct Ring {
    static constexpr int Row = F32 ? 128 * NB : 128 * ((NB + 1) / 2);  // bytes of a row
    static constexpr int Tile = 16 * Row;                              // of K or V
    static constexpr int Stages = Tile <= 2048 ? 4 : 3;
    static constexpr int Bytes = Stages * 2 * Tile;                    // of a warp
};

constexpr int kDecodeWarps = 4;

template <int NB, bool F32>
__global__ void __launch_bounds__(32 * kDecodeWarps)
    k_pages_decode(PagesView p, int layer, const StepSeq *__restrict__ seqs, const AttnItem *__restrict__ items,
                   AttnScratch scratch, const float *__restrict__ q, float *__restrict__ out) {
    constexpr int NV = (NB + 1) / 2;  // blocks of 64 of the values
    constexpr int R = kDecodeRows;
    // f32 heads of more than 64 have no registers to sum their small products
    // apart, and put their sums out more often instead (131,072 x 8 heads of 128:
    // 217 us, spilling for it 239)
    constexpr bool kApart = NB <= 2;
    constexpr int kRun = F32 && !kApart ? 4 : 16;  // tiles between put_out
    using G = Ring<NB, F32>;
    extern __shared__ __align__(128) unsigned char ring[];
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

    wait_before();

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
    // the sums so far to shared memory, relative to the maximum m_out (a thread's
    // elements are its own there)
    float m_out = -INFINITY;
    const auto put_out = [&]() {
        const float keep = m_out == -INFINITY ? 0.0f : ex2(m_out - m);
#pragma unroll
        for (int b = 0; b < NV; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int d = 64 * b + 8 * (2 * t + x) + i;
                    if (d >= 32 * NB) continue;
                    const float v = o[b][i][x] + o[b][i][2 + x];
                    s_o[warp][g][d] = m_out == -INFINITY ? v : __fmaf_rn(s_o[warp][g][d], keep, v);
                    o[b][i][x] = o[b][i][2 + x] = 0.0f;
                }
        m_out = m;
    };

    // this warp's tiles: 16 positions at lo + 16 warp, step 64; a tile never
    // leaves its page
    const int t0 = it.lo + 16 * warp;
    const int n_tiles = it.hi > t0 ? (it.hi - t0 + kDecodeKeys - 1) / kDecodeKeys : 0;
    unsigned char *const mine = ring + warp * G::Bytes;
    const uint32_t mine_at = (uint32_t)__cvta_generic_to_shared(mine);
    int pages = 0;  // lane i: the page of tile i of the current 32
    const char *const kv = static_cast<const char *>(p.kv);
    constexpr int Size = F32 ? 4 : 2, PerRow = G::Row / 16;  // chunks of a row in shared memory
    const int have = head * Size / 16;                       // of them in a page
    const auto fetch = [&](int tile) {
        if (tile < n_tiles) {
            if ((tile & 31) == 0) {
                const int at = t0 + kDecodeKeys * (tile + lane);
                pages = at < it.hi ? __ldg(table + (at >> p.page_shift)) : 0;
            }
            const int pos = t0 + kDecodeKeys * tile;
            const size_t row0 = (size_t)__shfl_sync(0xffffffffu, pages, tile & 31) * page_stride +
                                (size_t)(pos & page_mask) * head;
            const uint32_t to = mine_at + (uint32_t)(tile % G::Stages) * (2 * G::Tile);
            const char *const k_src = kv + (k_base + row0) * Size, *const v_src = kv + (v_base + row0) * Size;
#pragma unroll
            for (int i = 0; i < PerRow / 2; ++i) {  // 16 rows of PerRow chunks
                const int at = lane + 32 * i, r = at / PerRow, c = at % PerRow;
                const bool in = c < have && pos + r < it.hi;
                const size_t off = in ? (size_t)r * head * Size + 16 * c : 0;
                copy16(to + r * G::Row + ((c ^ k_swap<F32>(r)) << 4), k_src + off, in);
                copy16(to + G::Tile + r * G::Row + ((c ^ v_swap<F32>(r)) << 4), v_src + off, in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < G::Stages - 1; ++i) fetch(i);
    for (int tile = 0; tile < n_tiles; ++tile) {
        const int pos = t0 + kDecodeKeys * tile;
        asm volatile("cp.async.wait_group %0;" ::"n"(G::Stages - 2) : "memory");
        __syncwarp();
        fetch(tile + G::Stages - 1);  // into the place of the tile used last
        const unsigned char *const k_tile = mine + (tile % G::Stages) * (2 * G::Tile), *const v_tile = k_tile + G::Tile;

        float s[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            // the products of the first parts, and all the smaller ones
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f}, e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const int key = 8 * u + 4 * (g & 1) + (g >> 1);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                Chunk<F32> kc;
                kc.load(k_tile + key * G::Row, 4 * b + t, k_swap<F32>(key));
                if constexpr (F32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t k1[2], k2[2], k3[2];
                        split3(kc.v[h].x, kc.v[h].y, k1[0], k2[0], k3[0]);
                        split3(kc.v[h].z, kc.v[h].w, k1[1], k2[1], k3[1]);
                        const uint32_t(&a)[4] = qf.a[b][h];
                        mma16816(c, a[0], a[1], a[2], a[3], k1[0], k1[1]);
                        mma16816(e, a[0], a[1], a[2], a[3], k2[0], k2[1]);
                        mma16816(e, a[0], 0, a[2], 0, k3[0], k3[1]);
                        mma16816(e, qf.c[b][h][0], 0, qf.c[b][h][1], 0, k1[0], k1[1]);
                    }
                } else {
                    const uint32_t k[4] = {kc.v.x, kc.v.y, kc.v.z, kc.v.w};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t(&a)[4] = qf.a[b][h];
                        mma16816(c, a[0], a[1], a[2], a[3], k[2 * h], k[2 * h + 1]);
                        mma16816(e, qf.c[b][h][0], 0, qf.c[b][h][1], 0, k[2 * h], k[2 * h + 1]);
                    }
                }
            }
            // rows 0-7 hold part 1 (and 3), rows 8-15 part 2 of the same score;
            // columns 2 t and 2 t + 1 are keys 8 u + t and 8 u + 4 + t
            const int at = pos + 8 * u + t;
            s[u][0] = at < limit ? (c[0] + (c[2] + (e[0] + e[2]))) * scale : -INFINITY;
            s[u][1] = at + 4 < limit ? (c[1] + (c[3] + (e[1] + e[3]))) * scale : -INFINITY;
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
            Chunk<F32> vc[4];  // (blocks past the row are not read)
            if (F32 && 64 * b + 32 >= 32 * NB) {  // the row ends inside the block
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (g < 4) vc[x].load(v_tile + (4 * x + t) * G::Row, 8 * b + g, v_swap<F32>(t));
                    else vc[x] = Chunk<F32>{};
            } else {
#pragma unroll
                for (int x = 0; x < 4; ++x) vc[x].load(v_tile + (4 * x + t) * G::Row, 8 * b + g, v_swap<F32>(t));
            }
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float e[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) e[x] = (&vc[x].v[i >> 2].x)[i & 3];
                    uint32_t v1[2], v2[2], v3[2];
                    split3(e[0], e[1], v1[0], v2[0], v3[0]);
                    split3(e[2], e[3], v1[1], v2[1], v3[1]);
                    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    float(&small)[4] = kApart ? c : o[b][i];
                    mma16816(small, pa[0], pa[1], pa[2], pa[3], v2[0], v2[1]);
                    mma16816(small, pa[0], 0, pa[2], 0, v3[0], v3[1]);
                    mma16816(small, pc[0], 0, pc[1], 0, v1[0], v1[1]);
                    mma16816(o[b][i], pa[0], pa[1], pa[2], pa[3], v1[0], v1[1]);
                    if (kApart)
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[b][i][x] += c[x];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
                    const uint32_t b0 = __byte_perm((&vc[0].v.x)[i >> 1], (&vc[1].v.x)[i >> 1], sel);
                    const uint32_t b1 = __byte_perm((&vc[2].v.x)[i >> 1], (&vc[3].v.x)[i >> 1], sel);
                    mma16816(o[b][i], pa[0], pa[1], pa[2], pa[3], b0, b1);
                    mma16816(o[b][i], pc[0], 0, pc[1], 0, b0, b1);
                }
            }
        }
        if (tile % kRun == kRun - 1) put_out();
    }

    // the CTA's warps meet in shared memory
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
        s_m[warp][g] = m;
        s_l[warp][g] = l;
    }
    put_out();
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
    // The ring's memory is free: the pieces' weights 2^(m_i - M), Batch of each row
    // at a time, and the sums of the threads that share four elements.
    constexpr int Batch = 512, Threads = 32 * kDecodeWarps;
    float *const weight = reinterpret_cast<float *>(ring);                 // [R][Batch]
    float4 *const sums = reinterpret_cast<float4 *>(weight + R * Batch);   // [units]
    const size_t first = ((size_t)it.first * p.kv_heads + j) * R, step = (size_t)p.kv_heads * R;
    for (int r = warp; r < it.rows; r += kDecodeWarps) {
        float M = -INFINITY;
#pragma unroll 4
        for (int i = lane; i < it.n_parts; i += 32) M = fmaxf(M, __ldcg(&scratch.ml[first + r + i * step]).x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
        if (lane == 0) s_m[0][r] = M, s_l[0][r] = 0.0f;
    }
    __syncwarp();
    const int quads = head >> 2, groups = it.rows * quads, shares = max(1, Threads / groups);
    constexpr int Units = R * kHeadMax / 4 / Threads;  // at most, of a thread
    float4 acc[Units];
#pragma unroll
    for (int x = 0; x < Units; ++x) acc[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int base = 0; base < it.n_parts; base += Batch) {
        const int n = min(Batch, it.n_parts - base);
        for (int r = warp; r < it.rows; r += kDecodeWarps) {
            const float M = s_m[0][r];
            float L = 0.0f;
            for (int i = lane; i < n; i += 32) {
                const float2 ml = __ldcg(&scratch.ml[first + r + (base + i) * step]);
                const float k = M == -INFINITY ? 0.0f : ex2(ml.x - M);
                weight[r * Batch + i] = k;
                L = __fmaf_rn(ml.y, k, L);
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
            if (lane == 0) s_l[0][r] += L;
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < Units; ++x) {
            const int u = threadIdx.x + x * Threads, group = u % groups, r = group / quads;
            if (u >= groups * shares) break;
            const float4 *src = reinterpret_cast<const float4 *>(scratch.o + (first + r + base * step) * head) + group % quads;
#pragma unroll 8
            for (int i = u / groups; i < n; i += shares) {
                const float4 v = __ldcg(src + i * step * quads);
                const float k = weight[r * Batch + i];
                acc[x] = make_float4(__fmaf_rn(v.x, k, acc[x].x), __fmaf_rn(v.y, k, acc[x].y),
                                     __fmaf_rn(v.z, k, acc[x].z), __fmaf_rn(v.w, k, acc[x].w));
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < Units; ++x)
        if (threadIdx.x + x * Threads < groups * shares) sums[threadIdx.x + x * Threads] = acc[x];
    __syncthreads();
    for (int group = threadIdx.x; group < groups; group += Threads) {
        const int r = group / quads;
        float4 v = sums[group];
        for (int i = 1; i < shares; ++i) {
            const float4 w = sums[group + i * groups];
            v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
        }
        const float L = s_l[0][r];
        const int mr = it.row + r, tok = mr / p.group;
        const size_t at = ((size_t)(sq.row0 + tok) * p.heads + (size_t)j * p.group + (mr - tok * p.group)) * head;
        reinterpret_cast<float4 *>(out + at)[group % quads] = make_float4(v.x / L, v.y / L, v.z / L, v.w / L);
    }
}

}  // namespace

cudaError_t launch_pages_step(const PagesView &p, const StepSeq *staged, int n, StepSeq *seqs, int32_t *table,
                              const CopyItem *items, int n_items, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    const Copies c = copies_of(p, items, n_items);
    const size_t grid = (size_t)n + (c.units + 7) / 8;
    if (grid > (size_t)INT32_MAX) return cudaErrorInvalidValue;
    k_pages_step<<<(unsigned)grid, 256, 0, s>>>(p, staged, n, seqs, table, c);
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
    const Copies c = copies_of(p, items, n);
    if ((c.units + 7) / 8 > (size_t)INT32_MAX) return cudaErrorInvalidValue;
    k_pages_copy<<<(unsigned)((c.units + 7) / 8), 256, 0, s>>>(p, c);
    return launched();
}

namespace {

// Calls f(NB, F32) with the cache's head blocks and kind as types.
template <class F>
auto by_shape(const PagesView &p, F &&f) {
    const auto by_head = [&](auto f32) {
        switch ((p.head + 31) / 32) {
        case 1: return f(std::integral_constant<int, 1>{}, f32);
        case 2: return f(std::integral_constant<int, 2>{}, f32);
        case 3: return f(std::integral_constant<int, 3>{}, f32);
        default: return f(std::integral_constant<int, 4>{}, f32);
        }
    };
    return p.f32 ? by_head(std::true_type{}) : by_head(std::false_type{});
}

// Opts k_pages_decode into its shared memory on the current device; returns its
// CTAs per SM in *ctas.
template <int NB, bool F32>
cudaError_t decode_ready(int *ctas) {
    static int known[64] = {0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (known[dev] == 0) {
        constexpr int smem = kDecodeWarps * Ring<NB, F32>::Bytes;
        cudaError_t e = cudaFuncSetAttribute(k_pages_decode<NB, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        int n = 0;
        if (e == cudaSuccess)
            e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_pages_decode<NB, F32>, 32 * kDecodeWarps, smem);
        if (e != cudaSuccess) return e;
        known[dev] = n > 0 ? n : 1;
    }
    *ctas = known[dev];
    return cudaSuccess;
}

}  // namespace

int pages_decode_ctas(const PagesView &p) {
    int n = 1;
    by_shape(p, [&](auto nb, auto f32) { return decode_ready<decltype(nb)::value, decltype(f32)::value>(&n); });
    return n;
}

cudaError_t launch_pages_decode(const PagesView &p, int layer, const StepSeq *seqs, const AttnItem *items, int n_items,
                                const AttnScratch &scratch, const float *q, float *out, cudaStream_t s) {
    if (n_items == 0) return cudaSuccess;
    const dim3 grid((unsigned)n_items, (unsigned)p.kv_heads);
    return by_shape(p, [&](auto nb, auto f32) {
        constexpr int NB = decltype(nb)::value;
        constexpr bool F32 = decltype(f32)::value;
        int n = 0;
        const cudaError_t e = decode_ready<NB, F32>(&n);
        if (e != cudaSuccess) return e;
        const cudaError_t l = launch_after(k_pages_decode<NB, F32>, grid, 32 * kDecodeWarps,
                                           kDecodeWarps * Ring<NB, F32>::Bytes, s, p, layer, seqs, items, scratch, q, out);
        if (l != cudaSuccess) return l;
        return launched();
    });
}

}  // namespace krt
