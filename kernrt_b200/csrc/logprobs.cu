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

__device__ __forceinline__ unsigned long long max_u64(unsigned long long a, unsigned long long b) {
    return a > b ? a : b;
}

constexpr int kThreads = 512;

// One CTA per row.
__global__ void __launch_bounds__(kThreads) k_logprobs(const float *__restrict__ x, int vocab,
                                                       const int32_t *__restrict__ targets, float *logprob,
                                                       float *entropy, int top, int32_t *top_ids, float *top_logprobs,
                                                       int *err) {
    __shared__ float sh[3][32];
    __shared__ unsigned long long best[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float *row = x + (size_t)blockIdx.x * vocab;
    float m = -INFINITY;
    bool bad = false;
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
        const float v = row[i];
        bad |= v != v || v == INFINITY;
        m = fmaxf(m, v);
    }
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (lane == 0) sh[0][warp] = m;
    bad = __syncthreads_or(bad);
    for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, sh[0][w]);
    bad |= m == -INFINITY;
    float sum = 0.0f, dot = 0.0f;
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
        const float d = row[i] - m, e = expf(d);
        sum += e;
        if (e > 0.0f) dot = __fmaf_rn(e, d, dot);
    }
    for (int d = 16; d > 0; d >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        dot += __shfl_xor_sync(0xffffffffu, dot, d);
    }
    if (lane == 0) {
        sh[1][warp] = sum;
        sh[2][warp] = dot;
    }
    __syncthreads();
    sum = dot = 0.0f;
    for (int w = 0; w < kThreads / 32; ++w) {
        sum += sh[1][w];
        dot += sh[2][w];
    }
    const float lg = bad ? NAN : logf(sum);
    if (threadIdx.x == 0) {
        if (logprob) {
            const int t = targets[blockIdx.x];
            const bool in = t >= 0 && t < vocab;
            if (!in) atomicOr(err, ERR_TOKEN);
            logprob[blockIdx.x] = in ? (row[t] - m) - lg : NAN;
        }
        if (entropy) entropy[blockIdx.x] = lg - dot / sum;
    }
    unsigned long long last = ~0ull;
    for (int j = 0; j < top; ++j) {
        unsigned long long b = 0;
        for (int i = threadIdx.x; i < vocab; i += kThreads) {
            const unsigned long long r = rank_of(row[i], i);
            if (j == 0 || r < last) b = max_u64(b, r);
        }
        for (int d = 16; d > 0; d >>= 1) b = max_u64(b, __shfl_xor_sync(0xffffffffu, b, d));
        if (lane == 0) best[warp] = b;
        __syncthreads();
        for (int w = 0; w < kThreads / 32; ++w) b = max_u64(b, best[w]);
        __syncthreads();
        last = b;
        if (threadIdx.x == 0) {
            const int id = (int)~(uint32_t)b;
            top_ids[(size_t)blockIdx.x * top + j] = id;
            top_logprobs[(size_t)blockIdx.x * top + j] = (row[id] - m) - lg;
        }
    }
}

}  // namespace

cudaError_t launch_logprobs(const float *x, int rows, int vocab, const int32_t *targets, float *logprob,
                            float *entropy, int top, int32_t *top_ids, float *top_logprobs, int *err, cudaStream_t s) {
    if (rows == 0) return cudaSuccess;
    k_logprobs<<<(unsigned)rows, kThreads, 0, s>>>(x, vocab, targets, logprob, entropy, top, top_ids, top_logprobs,
                                                   err);
    count_launch();
    return cudaGetLastError();
}

}  // namespace krt
