// Host bookkeeping of a paged key/value cache: which pages each sequence
// holds, how many sequences share a page, and which pages are free.  No device
// calls: every operation that moves cache contents returns the page copies the
// caller has to enqueue.  A failing call throws PageError and changes nothing; a
// caller that cannot enqueue the copies takes the operation back (undo_extend;
// close for copy; compaction is planned first and made after).
//
// Pages are taken lowest id first.  A page several sequences share is never
// written: a sequence that grows into its last, partly filled page while others
// hold that page gets a page of its own and a copy of the used rows.
#pragma once

#include <cstddef>
#include <cstdint>
#include <string>
#include <vector>

namespace krt {

struct PageError {
    bool exhausted;  // out of pages or sequences (the arguments were fine)
    std::string msg;
};

// Rows [0, rows) of page src to page dst, every layer and head, K and V.
struct PageCopy {
    int32_t src, dst, rows;
};

class PageMap {
public:
    struct Seq {
        bool open = false;
        uint32_t generation = 0;
        size_t len = 0;
        std::vector<int32_t> pages;
        // pages[dirty..] have changed since the caller last uploaded them
        size_t dirty = 0;
    };

    PageMap(size_t n_pages, size_t page_size, size_t max_seqs, size_t max_len);

    uint64_t open();
    // n sequences that share the first `length` positions of `seq`.
    std::vector<uint64_t> fork(uint64_t seq, size_t length, size_t n);
    // One sequence with pages of its own holding a copy of them.
    uint64_t copy(uint64_t seq, size_t length, std::vector<PageCopy> *copies);
    void trim(uint64_t seq, size_t length);
    void close(const uint64_t *seqs, size_t n);
    // Every sequence seqs[i] grows by rows[i] positions.
    void extend(const uint64_t *seqs, const uint64_t *rows, size_t n, std::vector<PageCopy> *copies);
    // Takes the last call back, an extend with these sequences, rows and copies.
    void undo_extend(const uint64_t *seqs, const uint64_t *rows, size_t n, std::vector<PageCopy> copies);
    // Moves the highest pages in use into the lowest free ones until the pages
    // in use are 0 .. count - 1; returns the moves.
    std::vector<PageCopy> compact() {
        std::vector<PageCopy> moves = plan_compact();
        make_compact(moves);
        return moves;
    }
    std::vector<PageCopy> plan_compact() const;        // the moves, nothing changed
    void make_compact(const std::vector<PageCopy> &);  // as planned, nothing between

    size_t slot(uint64_t seq) const;  // throws on a closed or unknown handle
    Seq &at(size_t slot) { return seqs_[slot]; }
    const Seq &at(size_t slot) const { return seqs_[slot]; }
    size_t available() const { return free_.size(); }
    size_t page_size() const { return page_size_; }
    size_t max_pages() const { return max_pages_; }  // of one sequence
    size_t max_seqs() const { return seqs_.size(); }

private:
    int32_t take();
    void release(int32_t page);
    std::vector<size_t> free_slots(size_t n) const;
    uint64_t handle(size_t slot) const { return ((uint64_t)seqs_[slot].generation << 32) | (uint64_t)(slot + 1); }
    size_t pages_for(size_t len) const { return (len + page_size_ - 1) / page_size_; }

    size_t page_size_, max_len_, max_pages_;
    std::vector<uint32_t> refs_;
    std::vector<int32_t> free_;  // min-heap
    std::vector<Seq> seqs_;
};

}  // namespace krt
