// Log probabilities of given tokens: per row of logits, with m the largest and
// L = m + log sum exp(x - m), the target's x_t - L, the entropy
// L - sum p x with p = exp(x - L), and the largest logits less L.
//
// Logits of -inf are tokens that cannot be drawn: probability 0, nothing to
// the entropy.  A row that holds NaN or +inf, or nothing above -inf, has no
// distribution: its log probabilities and entropy are NaN.  The order of the
// top entries is by value, NaN above +inf, ids ascending among equals (-0 and
// +0 are equal).
//
// One read of the logits.  Measured: 1024 rows of 49152, 201 MB, 37.4 us without
// top entries (5.4 TB/s), 52.1 us with 5; one row of 151936, 7.5 us and, with 20,
// 12.7 us.
#include "kernels.cuh"
#include "paged.cuh"

namespace krt {

namespace {

// Ascending unsigned keys in the order of the values.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// Larger is better: the value's key, then the lower id.
__device__ __forceinline__ unsigned long long rank_of(float x, int id) {
    return ((unsigned long long)order_key(x) << 32) | (uint32_t)~id;
}

// A row is cut into chunks of some tiles of 256 x 16 elements, one CTA each, so
// that a few rows still fill the SMs and many keep HBM busy.  A tile is in
// registers, the next one in flight, and the row is read once: each thread keeps
// a running maximum m of its own with s = sum e and d = sum e (x - m), e = exp(x -
// m), which meet at the end of the chunk, and the row's last CTA joins the chunks
// in their order.
//
// The chunk's top entries: in the first tile each thread has its best element,
// and a bound that at least `top` of these 256 reach keeps every element of the
// top; only elements of those threads can reach it.  A warp finds such a bound
// by bisection over (value, id), stopping as soon as few enough reach it; ties
// (whole rows of equal values) end in the ids and never overflow.  In later
// tiles a thread only compares its maximum with that bound.
constexpr int kThreads = 256;
constexpr int kEach = 16;                               // elements of a thread in a tile
constexpr int kReach = kTopMost + kTopMost / 4 + 4;     // threads that reach a bound
constexpr int kNew = kReach * kEach;                // elements of a tile that can
constexpr int kRoom = 10 * kThreads;                    // candidates: those, and more from other tiles
static_assert(kRoom >= kNew + 1024, "room for a tile beside the candidates so far");
using u64 = unsigned long long;

struct Part {
    float m, s, d, bad;
};

__device__ __forceinline__ float exp_of(float d) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * 1.4426950408889634f));
    return y;
}

// The candidates in order, the first `top` of them to `to`: each counts
// those above it.
template <class F>
__device__ __forceinline__ void take_top(const u64 *cand, int n, int top, F &&to) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 r = cand[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += cand[j] > r;
        if (above < top) to(above, r);
    }
}

// A bound that at least `top` of the block's best[] reach and not many more (0 if
// fewer than `top` are above 0): one warp bisects, the values first and, where
// too many are equal, their ids.
template <class T>
__device__ __forceinline__ bool bisect(const T (&b)[kThreads / 32], T &lo, T hi, int top) {
    while (lo < hi) {  // at least `top` reach lo, fewer reach hi + 1
        const T mid = lo + (hi - lo) / 2 + 1;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) n += b[i] >= mid;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n < top) {
            hi = mid - 1;
        } else {
            lo = mid;
            if (n <= top + top / 4 + 4) return true;
        }
    }
    return false;
}
__device__ __forceinline__ u64 bound_of(const u64 *best, int top) {
    const int lane = threadIdx.x & 31;
    uint32_t b[kThreads / 32];
    uint32_t lo = ~0u, hi = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
        b[i] = (uint32_t)(best[lane + 32 * i] >> 32);
        lo = min(lo, b[i]);
        hi = max(hi, b[i]);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    if (bisect(b, lo, __reduce_max_sync(0xffffffffu, hi), top)) return (u64)lo << 32;
    u64 c[kThreads / 32], low = (u64)lo << 32;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) c[i] = best[lane + 32 * i];
    bisect(c, low, low | 0xffffffffull, top);
    return low;
}

// (m, s, d) joined with another of maximum m2: sums over elements less m, the
// larger of both; exp(x - m) (x - m) with x - m = (x - m_i) + (m_i - m).
__device__ __forceinline__ void join(float &m, float &s, float &d, float m2, float s2, float d2) {
    const float mn = fmaxf(m, m2);
    // (nothing but -inf on a side: its sums are 0, or NaN, which stays)
    const float t = fmaxf(m - mn, -1e30f), t2 = fmaxf(m2 - mn, -1e30f), w = exp_of(t), w2 = exp_of(t2);
    d = __fmaf_rn(w, __fmaf_rn(s, t, d), w2 * __fmaf_rn(s2, t2, d2));
    s = __fmaf_rn(w, s, w2 * s2);
    m = mn;
}

template <bool Vec>
__global__ void __launch_bounds__(kThreads, 4) k_logprobs(const float *__restrict__ x, int vocab, int chunks, int tiles,
                                                          const int32_t *__restrict__ targets, float *logprob,
                                                          float *entropy, int top, int32_t *top_ids,
                                                          float *top_logprobs, Part *parts, u64 *lists,
                                                          unsigned *count, int *err) {
    __shared__ u64 best[kThreads], cand[kRoom], kept[kTopMost];
    __shared__ float red[3][kThreads / 32];
    __shared__ int n_cand;
    __shared__ u64 bound;
    __shared__ bool last;
    constexpr int E = kEach;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = (int)(blockIdx.x / (unsigned)chunks), c = (int)(blockIdx.x % (unsigned)chunks);
    const float *row = x + (size_t)r * vocab;
    const int from = c * tiles * kThreads * E, to = min(vocab, from + tiles * kThreads * E);

    // element e of this thread's share of a tile has id id_of(tile's first, e);
    // those past the row are absent
    const auto id_of = [&](int at, int e) {
        return Vec ? at + 4 * (tid + kThreads * (e / 4)) + e % 4 : at + tid + kThreads * e;
    };
    const auto load = [&](int at, float (&v)[E]) {
        if constexpr (Vec) {
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                const float4 f = id_of(at, e) < to ? __ldcs(reinterpret_cast<const float4 *>(row + id_of(at, e)))
                                                   : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = id_of(at, e) < to ? __ldcs(row + id_of(at, e)) : -INFINITY;
        }
    };
    if (tid == 0) n_cand = 0, bound = 0;

    // a thread's best element of a tile (0: none)
    const auto best_of = [&](int at, const float (&v)[E], float own, bool odd) {
        u64 b = 0;
        if (odd) {  // it holds NaN or +inf: their order is by key
#pragma unroll 1
            for (int e = 0; e < E; ++e) {
                const int id = id_of(at, e);
                const u64 k = id < to ? rank_of(row[id], id) : 0;
                b = k > b ? k : b;
            }
        } else {
            int id = to;
#pragma unroll
            for (int e = E - 1; e >= 0; --e) id = v[e] == own && id_of(at, e) < to ? id_of(at, e) : id;
            if (id < to) b = rank_of(own, id);
        }
        return b;
    };
    // raises the bound by the threads' bests of a tile
    const auto raise = [&](u64 b) {
        best[tid] = b;
        __syncthreads();
        if (warp == 0) {
            const u64 lo = bound_of(best, top);
            if (lane == 0 && lo > bound) bound = lo;
        }
        __syncthreads();
    };
    // leaves few more candidates than `top`: those that reach a bound made of
    // the best of each thread's share
    const auto narrow = [&]() {
        const int n = n_cand;
        if (n <= 2 * top + 16) return;
        u64 k[kRoom / kThreads], b = 0;
#pragma unroll
        for (int i = 0; i < kRoom / kThreads; ++i) {
            k[i] = tid + i * kThreads < n ? cand[tid + i * kThreads] : 0;
            b = k[i] > b ? k[i] : b;
        }
        best[tid] = b;
        __syncthreads();
        if (warp == 0) {
            const u64 lo = bound_of(best, top);
            if (lane == 0) bound = lo > 0 ? lo : 1, n_cand = 0;
        }
        __syncthreads();
        const u64 lo = bound;
#pragma unroll
        for (int i = 0; i < kRoom / kThreads; ++i)
            if (k[i] >= lo) cand[atomicAdd(&n_cand, 1)] = k[i];
        __syncthreads();
    };
    // appends the tile's elements that reach the bound (bound 0: fewer than `top`
    // threads have elements, and all of theirs do); NaN is above every value
    const auto append = [&](int at, const float (&v)[E], u64 least, float value) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (v[e] < value) continue;
            const u64 k = rank_of(v[e], id_of(at, e));
            if (id_of(at, e) < to && k >= least) {
                const int i = atomicAdd(&n_cand, 1);
                if (i < kRoom) cand[i] = k;
            }
        }
    };
    const auto most_of = [&](const float (&v)[E]) {
        float own = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) own = fmaxf(own, v[e]);
        return own;
    };

    float m = -INFINITY, s = 0.0f, d = 0.0f;
    float v[E], next[E];
    u64 least = 0;
    float value = 0.0f;
    load(from, v);
    for (int at = from; at < to; at += kThreads * E) {
        if (at + kThreads * E < to) load(at + kThreads * E, next);
        const float own = most_of(v);
        // NaN, and +inf through inf - inf, make s NaN; exp(-inf) (-inf) counts as 0
        const float mn = fmaxf(m, own), mb = mn == -INFINITY ? 0.0f : mn;
        if (mn > m) {
            const float t = fmaxf(m - mn, -1e30f), w = exp_of(t);
            d = w * __fmaf_rn(s, t, d);
            s *= w;
            m = mn;
        }
        float s1 = 0.0f, d1 = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float t = v[e] - mb, w = exp_of(t);
            s1 += w;
            d1 = __fmaf_rn(w, fmaxf(t, -1e30f), d1);
        }
        s += s1;
        d += d1;
        if (top) {
            const bool odd = s1 != s1;
            if (at == from) {  // the first tile's bound serves the whole chunk
                raise(best_of(at, v, own, odd));
                least = bound > 0 ? bound : 1;
                value = key_value((uint32_t)(least >> 32));
            }
            if (odd || !(own < value)) append(at, v, least, value);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = next[e];
    }
    __syncthreads();
    if (top && n_cand > kRoom) {
        // More reached the first tile's bound than there is room for (rows that
        // ascend, say): once more, raising the bound wherever many reach it and
        // keeping only the top so far.
        __syncthreads();
        if (tid == 0) n_cand = 0, bound = 0;
        for (int at = from; at < to; at += kThreads * E) {
            load(at, v);
            __syncthreads();
            float own = most_of(v);
            bool odd = false;
#pragma unroll
            for (int e = 0; e < E; ++e) odd |= !(v[e] < INFINITY);
            value = key_value((uint32_t)(bound >> 32));
            if (__syncthreads_count(odd || !(own < value)) > top + top / 4 + 4) raise(best_of(at, v, own, odd));
            const int n = n_cand;
            __syncthreads();  // all have read it before any thread appends
            if (n + kNew > kRoom) {
                take_top(cand, n, top, [&](int i, u64 k) { kept[i] = k; });
                __syncthreads();
                if (tid < top) cand[tid] = kept[tid];
                if (tid == 0) {
                    n_cand = top;
                    if (kept[top - 1] > bound) bound = kept[top - 1];
                }
                __syncthreads();
            }
            least = bound > 0 ? bound : 1;
            append(at, v, least, key_value((uint32_t)(least >> 32)));
        }
        __syncthreads();
    }

    // the chunk's threads meet, in a fixed order
    const auto meet = [&]() {
        for (int i = 16; i > 0; i >>= 1)
            join(m, s, d, __shfl_xor_sync(0xffffffffu, m, i), __shfl_xor_sync(0xffffffffu, s, i),
                 __shfl_xor_sync(0xffffffffu, d, i));
        if (lane == 0) red[0][warp] = m, red[1][warp] = s, red[2][warp] = d;
        __syncthreads();
        m = red[0][0], s = red[1][0], d = red[2][0];
#pragma unroll
        for (int w = 1; w < kThreads / 32; ++w) join(m, s, d, red[0][w], red[1][w], red[2][w]);
    };
    meet();
    if (top) narrow();
    const int mine = min(top, to - from);  // entries of this chunk's list

    if (chunks > 1) {
        const size_t at = (size_t)r * chunks + c;
        if (tid == 0) parts[at] = {m, s, d, 0.0f};
        if (top) {
            take_top(cand, n_cand, top, [&](int i, u64 k) { lists[at * top + i] = k; });
            if (tid >= mine && tid < top) lists[at * top + tid] = 0;  // absent
        }
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            last = atomicAdd(count + r, 1u) == (unsigned)chunks - 1;
            if (last) count[r] = 0, n_cand = 0;
        }
        __syncthreads();
        if (!last) return;
        __threadfence();
        const Part *p = parts + (size_t)r * chunks;
        m = -INFINITY, s = d = 0.0f;
        for (int i = tid; i < chunks; i += kThreads) {
            const float4 q = __ldcg(reinterpret_cast<const float4 *>(p + i));
            join(m, s, d, q.x, q.y, q.z);
        }
        const u64 *all = lists + (size_t)r * chunks * top;
        const int total = chunks * top;
        if (top) {
            u64 b = 0;
            for (int i = tid; i < total; i += kThreads) {
                const u64 k = __ldcg(all + i);
                b = k > b ? k : b;
            }
            best[tid] = b;
        }
        meet();
        if (top) {
            if (warp == 0) {
                const u64 lo = bound_of(best, top);
                if (lane == 0) bound = lo;
            }
            __syncthreads();
            // as many entries at a time as there is room for; what is kept of
            // them raises the bound for the next
            u64 b = bound;
            const int batch = kRoom - kTopMost;
            for (int at = 0; at < total; at += batch) {
                for (int i = at + tid; i < min(total, at + batch); i += kThreads) {
                    const u64 k = __ldcg(all + i);
                    if (k >= b && k > 0) cand[atomicAdd(&n_cand, 1)] = k;
                }
                __syncthreads();
                narrow();
                const int n = n_cand;
                __syncthreads();  // all have read it before the next batch comes
                if (n > top && at + batch < total) {
                    take_top(cand, n, top, [&](int i, u64 k) { kept[i] = k; });
                    __syncthreads();
                    if (tid < top) cand[tid] = kept[tid];
                    if (tid == 0) n_cand = top;
                    b = kept[top - 1] > b ? kept[top - 1] : b;
                    __syncthreads();
                }
            }
        }
    }

    const float lg = m == -INFINITY ? NAN : logf(s);
    if (tid == 0) {
        if (logprob) {
            const int t = targets[r];
            const bool in = t >= 0 && t < vocab;
            if (!in) atomicOr(err, ERR_TOKEN);
            logprob[r] = in ? (row[t] - m) - lg : NAN;
        }
        if (entropy) entropy[r] = lg - d / s;
    }
    if (top)
        take_top(cand, n_cand, top, [&](int i, u64 k) {
            const int id = (int)~(uint32_t)k;
            top_ids[(size_t)r * top + i] = id;
            top_logprobs[(size_t)r * top + i] = (row[id] - m) - lg;
        });
}

// How a row is cut: into chunks of as many tiles as leave every SM four CTAs, at
// most 16 (measured, 1024 x 49152 with 5 top entries: chunks of 6 tiles 69 us, of
// the row's 12 52 us; 1 x 151936 with 20: 38 chunks of a tile 12.7 us, 149 of a
// quarter of one 14.8 us).
constexpr int kTilesMost = 16;
struct Cut {
    int tiles, chunks;
};
Cut cut_of(int rows, int vocab) {
    constexpr int tile = kThreads * kEach;
    const size_t share = (size_t)rows * vocab / ((size_t)tile * 4 * device_sms());
    const int most = share > kTilesMost ? kTilesMost : share > 1 ? (int)share : 1;
    const int tiles = (vocab + tile - 1) / tile;  // of the row
    Cut c;
    c.chunks = (tiles + most - 1) / most;
    c.tiles = (tiles + c.chunks - 1) / c.chunks;
    c.chunks = (tiles + c.tiles - 1) / c.tiles;
    return c;
}

}  // namespace

int logprobs_chunks(int rows, int vocab) { return cut_of(rows, vocab).chunks; }

cudaError_t launch_logprobs(const float *x, int rows, int vocab, const int32_t *targets, float *logprob,
                            float *entropy, int top, int32_t *top_ids, float *top_logprobs, void *parts, void *lists,
                            unsigned *count, int *err, cudaStream_t s) {
    if (rows == 0) return cudaSuccess;
    const Cut c = cut_of(rows, vocab);
    const auto go = [&](auto kernel) {
        kernel<<<(unsigned)rows * (unsigned)c.chunks, kThreads, 0, s>>>(
            x, vocab, c.chunks, c.tiles, targets, logprob, entropy, top, top_ids, top_logprobs,
            static_cast<Part *>(parts), static_cast<u64 *>(lists), count, err);
    };
    if (vocab % 4 == 0) go(k_logprobs<true>);
    else go(k_logprobs<false>);
    count_launch();
    return cudaGetLastError();
}

}  // namespace krt
