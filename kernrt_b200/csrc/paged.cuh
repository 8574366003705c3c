// Launch interface of the paged key/value cache's kernels (paged.cu) and of
// the token log probabilities (logprobs.cu).  All pointers are device
// pointers; all launches are asynchronous on the given stream.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace krt {

// One layer-major cache: [n_layers][2][n_pages][n_kv_heads][page_size][head],
// K at 0 and V at 1 of the second axis, bf16 or f32.
struct PagesView {
    void *kv;
    int f32;
    int n_layers, n_pages, kv_heads, heads, group, head, page_shift;
    const int32_t *table;  // [max_seqs][max_pages] page ids
    int max_pages;
};

// One sequence of the current step: its `rows` new positions ctx .. ctx +
// rows - 1 are rows row0 .. of the step's q, k, v and out.
struct StepSeq {
    int32_t slot, ctx, rows, row0;
    // table entries [dirty, dirty + n_dirty) come from delta[delta ..]
    int32_t dirty, n_dirty, delta, pad;
};

// A piece of the step's attention for one kv head: `rows` query rows from `row`
// on (row = token * group + head of the group) of sequence `seq` of the step
// over its positions [lo, hi).  n_parts pieces with the same rows, first ..
// first + n_parts - 1, share the sequence's length and are joined; `join` is
// the place of their counter.
struct AttnItem {
    int32_t seq, row, rows, lo, hi, first, n_parts, join;
};

// Partial results of the pieces: per (piece, kv head, row of the piece) the
// values o [head] and (m, l), and per (join, kv head) a counter that is 0
// between launches.
struct AttnScratch {
    float *o;
    float2 *ml;
    unsigned *count;
};

// Page copies (PageCopy of pages.h): src, dst, rows.
struct CopyItem {
    int32_t src, dst, rows;
};

// staged: StepSeq[n], then the table deltas; copies the descriptors to `seqs`,
// the deltas into the table, and the pages of `items`.
cudaError_t launch_pages_step(const PagesView &p, const StepSeq *staged, int n, StepSeq *seqs, int32_t *table,
                              const CopyItem *items, int n_items, cudaStream_t s);
// Row r of k and v [rows, kv_heads * head] f32 into its position of `layer`.
cudaError_t launch_pages_write(const PagesView &p, int layer, const StepSeq *seqs, int n, int rows, const float *k,
                               const float *v, cudaStream_t s);
cudaError_t launch_pages_copy(const PagesView &p, const CopyItem *items, int n, cudaStream_t s);
// out[r, h] = softmax(q[r, h] . K / sqrt(head)) V over positions 0 .. ctx + i
// of the row's sequence, for pieces of at most kDecodeRows rows.
constexpr int kDecodeRows = 8;
constexpr int kDecodeKeys = 64;  // positions a CTA takes at once: what splits are rounded to
cudaError_t launch_pages_decode(const PagesView &p, int layer, const StepSeq *seqs, const AttnItem *items, int n_items,
                                const AttnScratch &scratch, const float *q, float *out, cudaStream_t s);

int pages_decode_ctas(const PagesView &p);  // CTAs an SM runs at once

// The same for pieces of many rows (paged_prompt.cu); `split`: some piece has
// more than one part.
constexpr int kPromptRows = 256;
constexpr int kPromptKeys = 128;  // what splits are rounded to
cudaError_t launch_pages_prompt(const PagesView &p, int layer, const StepSeq *seqs, const AttnItem *items, int n_items,
                                bool split, const AttnScratch &scratch, const float *q, float *out, int *err,
                                cudaStream_t s);

// Per row of x [rows, vocab]: the target's log probability, the entropy, and
// the `top` largest (ids ascending among equals) with their log probabilities.
// Rows of more than one chunk take scratch: `parts` 16 bytes and `lists` 8 top
// bytes for each of rows * logprobs_chunks(rows, vocab), and `count`, rows
// counters that are 0 between launches.
constexpr int kTopMost = 64;
int logprobs_chunks(int rows, int vocab);
cudaError_t launch_logprobs(const float *x, int rows, int vocab, const int32_t *targets, float *logprob,
                            float *entropy, int top, int32_t *top_ids, float *top_logprobs, void *parts, void *lists,
                            unsigned *count, int *err, cudaStream_t s);

}  // namespace krt
