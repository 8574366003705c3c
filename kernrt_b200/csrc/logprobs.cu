// Log probabilities of given tokens: per row of logits, with m the largest and
// L = m + log sum exp(x - m), the target's x_t - L, the entropy
// L - sum p x with p = exp(x - L), and the largest logits less L.
//
// Logits of -inf are tokens that cannot be drawn: probability 0, nothing to
// the entropy.  A row that holds NaN or +inf, or nothing above -inf, has no
// distribution: its log probabilities and entropy are NaN.  The order of the
// top entries is by value, NaN above +inf, ids ascending among equals (-0 and
// +0 are equal).
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
// Larger is better: the value's key, then the lower id.
__device__ __forceinline__ unsigned long long rank_of(float x, int id) {
    return ((unsigned long long)order_key(x) << 32) | (uint32_t)~id;
}

// A row is cut into chunks of 256 E elements, one CTA each, so that a few rows
// still fill the SMs and many keep HBM busy: E elements a thread are loaded
// at once and stay in registers, so the row is read once for the maximum, both
// sums and the top entries.  A chunk leaves (m, s, d) = (max, sum e, sum e (x -
// m)), e = exp(x - m), and its own top entries in order; the row's last CTA
// joins the chunks in their order.
//
// The chunk's top entries: each thread has its best element; a bound that at
// least `top` of these 256 reach keeps every element of the chunk's top, and
// only the elements of those threads can reach it.  A warp finds such a bound
// by bisection over (value, id), stopping as soon as few enough reach it; ties
// (whole rows of equal values) end in the ids and never overflow.
constexpr int kThreads = 256;
constexpr int kMostEach = 32;                           // E at most
constexpr int kSlack = 16;                              // how many more than `top` may reach a bound
constexpr int kRoom = (kTopMost + kSlack) * kMostEach;  // elements that can
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

// A bound that at least `top` of the block's best[] reach and at most kSlack
// more (0 if fewer than `top` are above 0): one warp bisects.
__device__ __forceinline__ u64 bound_of(const u64 *best, int top) {
    const int lane = threadIdx.x & 31;
    u64 b[kThreads / 32];
    u64 lo = ~0ull, hi = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
        b[i] = best[lane + 32 * i];
        lo = b[i] < lo ? b[i] : lo;
        hi = b[i] > hi ? b[i] : hi;
    }
    for (int i = 16; i > 0; i >>= 1) {
        const u64 l = __shfl_xor_sync(0xffffffffu, lo, i), h = __shfl_xor_sync(0xffffffffu, hi, i);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
    }
    // at least `top` reach lo (all do), fewer reach hi + 1
    while (lo < hi) {
        const u64 mid = lo + (hi - lo + 1) / 2;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) n += b[i] >= mid;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n < top) {
            hi = mid - 1;
        } else {
            lo = mid;
            if (n <= top + kSlack) break;
        }
    }
    return lo;
}

template <int E, bool Vec>
__global__ void __launch_bounds__(kThreads, 4) k_logprobs(const float *__restrict__ x, int vocab, int chunks,
                                                       const int32_t *__restrict__ targets, float *logprob,
                                                       float *entropy, int top, int32_t *top_ids, float *top_logprobs,
                                                       Part *parts, u64 *lists, unsigned *count, int *err) {
    __shared__ u64 best[kThreads], cand[kRoom], kept[kTopMost];
    __shared__ float red[3][kThreads / 32];
    __shared__ int n_cand;
    __shared__ u64 bound;
    __shared__ bool last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = (int)(blockIdx.x / (unsigned)chunks), c = (int)(blockIdx.x % (unsigned)chunks);
    const float *row = x + (size_t)r * vocab;
    const int from = c * kThreads * E;

    // element e of this thread has id id_of(e); those past the row are absent
    const auto id_of = [&](int e) { return Vec ? from + 4 * (tid + kThreads * (e / 4)) + e % 4 : from + tid + kThreads * e; };
    float v[E];
    if constexpr (Vec) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 f = id_of(e) < vocab ? __ldcs(reinterpret_cast<const float4 *>(row + id_of(e)))
                                              : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = id_of(e) < vocab ? __ldcs(row + id_of(e)) : -INFINITY;
    }
    if (tid == 0) n_cand = 0;

    float own = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) own = fmaxf(own, v[e]);
    float m = own;
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, red[0][w]);
    // NaN, and +inf through inf - inf, make s NaN; exp(-inf) (-inf) counts as 0
    const float mb = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, d = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float t = v[e] - mb, w = exp_of(t);
        s += w;
        d = __fmaf_rn(w, fmaxf(t, -1e30f), d);
    }
    if (top) {
        u64 b = 0;
        if (s != s) {  // the thread holds one of them: their order is by key
#pragma unroll 1
            for (int e = 0; e < E; ++e) {
                const int id = id_of(e);
                const u64 k = id < vocab ? rank_of(row[id], id) : 0;
                b = k > b ? k : b;
            }
        } else {
            int id = vocab;
#pragma unroll
            for (int e = E - 1; e >= 0; --e) id = v[e] == own && id_of(e) < vocab ? id_of(e) : id;
            if (id < vocab) b = rank_of(own, id);
        }
        best[tid] = b;
    }
    for (int i = 16; i > 0; i >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, i);
        d += __shfl_xor_sync(0xffffffffu, d, i);
    }
    if (lane == 0) red[1][warp] = s, red[2][warp] = d;

    if (top) {
        __syncthreads();
        if (warp == 0) {
            const u64 lo = bound_of(best, top);
            if (lane == 0) bound = lo;
        }
        __syncthreads();
        // (a bound of 0: fewer than `top` threads have elements; absent ones stay out)
        const u64 least = bound > 0 ? bound : 1;
        if (best[tid] >= least) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const u64 k = rank_of(v[e], id_of(e));
                if (id_of(e) < vocab && k >= least) cand[atomicAdd(&n_cand, 1)] = k;
            }
        }
    }
    __syncthreads();
    s = d = 0.0f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) s += red[1][w], d += red[2][w];
    const int mine = min(top, min(vocab - from, kThreads * E));  // entries of this chunk's list

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
        // the row: maximum, then the sums in the chunks' order
        const Part *p = parts + (size_t)r * chunks;
        m = -INFINITY;
        bool bad = false;
        for (int i = tid; i < chunks; i += kThreads) {
            const float4 q = __ldcg(reinterpret_cast<const float4 *>(p + i));
            m = fmaxf(m, q.x);
            bad |= q.y != q.y;
        }
        for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
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
        if (lane == 0) red[0][warp] = m;
        bad = __syncthreads_or(bad);
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, red[0][w]);
        if (top && warp == 0) {
            const u64 lo = bound_of(best, top);
            if (lane == 0) bound = lo;
        }
        s = d = 0.0f;
        for (int i = tid; i < chunks; i += kThreads) {
            const float4 q = __ldcg(reinterpret_cast<const float4 *>(p + i));
            // exp(x - m) (x - m) with x - m = (x - m_i) + (m_i - m)
            if (q.x > -INFINITY) {
                const float t = fmaxf(q.x - m, -1e30f), w = exp_of(t);
                s = __fmaf_rn(q.y, w, s);
                d = __fmaf_rn(w, __fmaf_rn(q.y, t, q.z), d);
            }
        }
        for (int i = 16; i > 0; i >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, i);
            d += __shfl_xor_sync(0xffffffffu, d, i);
        }
        if (lane == 0) red[1][warp] = s, red[2][warp] = d;
        __syncthreads();
        if (top) {
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
                const int n = n_cand;
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
        __syncthreads();
        s = d = 0.0f;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) s += red[1][w], d += red[2][w];
        if (bad) s = NAN;
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

// Elements a thread: as many as leave every SM two CTAs, from 4 to 32.
int each_of(int rows, int vocab) {
    const size_t share = (size_t)rows * vocab / ((size_t)kThreads * 2 * device_sms());
    return share >= 32 ? 32 : share >= 16 ? 16 : share >= 8 ? 8 : 4;
}

template <int E>
void launch(const float *x, int rows, int vocab, int chunks, const int32_t *targets, float *logprob, float *entropy,
            int top, int32_t *top_ids, float *top_logprobs, void *parts, void *lists, unsigned *count, int *err,
            cudaStream_t s) {
    const auto kernel = vocab % 4 == 0 ? k_logprobs<E, true> : k_logprobs<E, false>;
    kernel<<<(unsigned)rows * (unsigned)chunks, kThreads, 0, s>>>(x, vocab, chunks, targets, logprob, entropy, top,
                                                                  top_ids, top_logprobs, static_cast<Part *>(parts),
                                                                  static_cast<u64 *>(lists), count, err);
}

}  // namespace

int logprobs_chunks(int rows, int vocab) {
    const int chunk = kThreads * each_of(rows, vocab);
    return vocab / chunk + (vocab % chunk != 0);
}

cudaError_t launch_logprobs(const float *x, int rows, int vocab, const int32_t *targets, float *logprob,
                            float *entropy, int top, int32_t *top_ids, float *top_logprobs, void *parts, void *lists,
                            unsigned *count, int *err, cudaStream_t s) {
    if (rows == 0) return cudaSuccess;
    const int chunks = logprobs_chunks(rows, vocab);
    const auto go = [&](auto f) {
        f(x, rows, vocab, chunks, targets, logprob, entropy, top, top_ids, top_logprobs, parts, lists, count, err, s);
    };
    switch (each_of(rows, vocab)) {
    case 32: go(launch<32>); break;
    case 16: go(launch<16>); break;
    case 8: go(launch<8>); break;
    default: go(launch<4>); break;
    }
    count_launch();
    return cudaGetLastError();
}

}  // namespace krt
