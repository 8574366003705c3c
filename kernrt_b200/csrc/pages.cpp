#include "pages.h"

#include <algorithm>
#include <functional>
#include <unordered_map>

namespace krt {

namespace {
[[noreturn]] void invalid(const std::string &msg) { throw PageError{false, msg}; }
[[noreturn]] void exhausted(const std::string &msg) { throw PageError{true, msg}; }
}  // namespace

PageMap::PageMap(size_t n_pages, size_t page_size, size_t max_seqs, size_t max_len)
    : page_size_(page_size), max_len_(max_len), max_pages_(pages_for(max_len)), refs_(n_pages, 0), free_(n_pages),
      seqs_(max_seqs) {
    for (size_t i = 0; i < n_pages; ++i) free_[i] = (int32_t)i;  // ascending: a min-heap
}

int32_t PageMap::take() {
    std::pop_heap(free_.begin(), free_.end(), std::greater<int32_t>());
    const int32_t p = free_.back();
    free_.pop_back();
    refs_[(size_t)p] = 1;
    return p;
}

void PageMap::release(int32_t page) {
    if (--refs_[(size_t)page] == 0) {
        free_.push_back(page);
        std::push_heap(free_.begin(), free_.end(), std::greater<int32_t>());
    }
}

size_t PageMap::slot(uint64_t seq) const {
    const uint64_t low = seq & 0xffffffffu;
    if (low == 0 || low > seqs_.size() || !seqs_[low - 1].open || seqs_[low - 1].generation != (uint32_t)(seq >> 32))
        invalid("invalid or closed sequence " + std::to_string(seq));
    return (size_t)low - 1;
}

std::vector<size_t> PageMap::free_slots(size_t n) const {
    std::vector<size_t> got;
    for (size_t i = 0; i < seqs_.size() && got.size() < n; ++i)
        if (!seqs_[i].open) got.push_back(i);
    if (got.size() < n)
        exhausted("out of sequences: " + std::to_string(n) + " wanted, " + std::to_string(got.size()) + " of " +
                  std::to_string(seqs_.size()) + " free");
    return got;
}

uint64_t PageMap::open() {
    const size_t s = free_slots(1)[0];
    Seq &q = seqs_[s];
    q.open = true;
    ++q.generation;
    q.len = 0;
    q.pages.clear();
    q.dirty = 0;
    return handle(s);
}

std::vector<uint64_t> PageMap::fork(uint64_t seq, size_t length, size_t n) {
    const size_t parent = slot(seq);
    if (length > seqs_[parent].len)
        invalid("fork at " + std::to_string(length) + " of a sequence of " + std::to_string(seqs_[parent].len));
    const std::vector<size_t> slots = free_slots(n);
    const std::vector<int32_t> shared(seqs_[parent].pages.begin(),
                                      seqs_[parent].pages.begin() + (long)pages_for(length));
    std::vector<uint64_t> out;
    for (size_t s : slots) {
        Seq &q = seqs_[s];
        q.open = true;
        ++q.generation;
        q.len = length;
        q.pages = shared;
        q.dirty = 0;
        for (int32_t p : shared) ++refs_[(size_t)p];
        out.push_back(handle(s));
    }
    return out;
}

uint64_t PageMap::copy(uint64_t seq, size_t length, std::vector<PageCopy> *copies) {
    const size_t from = slot(seq);
    if (length > seqs_[from].len)
        invalid("copy of " + std::to_string(length) + " positions of a sequence of " + std::to_string(seqs_[from].len));
    const size_t need = pages_for(length);
    if (need > free_.size())
        exhausted("out of pages: " + std::to_string(need) + " wanted, " + std::to_string(free_.size()) + " free");
    const size_t s = free_slots(1)[0];
    Seq &q = seqs_[s];
    q.open = true;
    ++q.generation;
    q.len = length;
    q.pages.clear();
    q.dirty = 0;
    for (size_t i = 0; i < need; ++i) {
        const int32_t p = take();
        q.pages.push_back(p);
        copies->push_back({seqs_[from].pages[i], p, (int32_t)std::min(page_size_, length - i * page_size_)});
    }
    return handle(s);
}

void PageMap::trim(uint64_t seq, size_t length) {
    Seq &q = seqs_[slot(seq)];
    if (length > q.len) invalid("trim to " + std::to_string(length) + " of a sequence of " + std::to_string(q.len));
    while (q.pages.size() > pages_for(length)) {
        release(q.pages.back());
        q.pages.pop_back();
    }
    q.len = length;
    q.dirty = std::min(q.dirty, q.pages.size());
}

void PageMap::close(const uint64_t *seqs, size_t n) {
    std::vector<size_t> slots(n);
    for (size_t i = 0; i < n; ++i) slots[i] = slot(seqs[i]);
    std::vector<size_t> sorted = slots;
    std::sort(sorted.begin(), sorted.end());
    if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end()) invalid("a sequence is closed twice");
    for (size_t s : slots) {
        for (int32_t p : seqs_[s].pages) release(p);
        seqs_[s].pages.clear();
        seqs_[s].len = 0;
        seqs_[s].open = false;
    }
}

void PageMap::extend(const uint64_t *seqs, const uint64_t *rows, size_t n, std::vector<PageCopy> *copies) {
    std::vector<size_t> slots(n);
    for (size_t i = 0; i < n; ++i) slots[i] = slot(seqs[i]);
    std::vector<size_t> sorted = slots;
    std::sort(sorted.begin(), sorted.end());
    if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end())
        invalid("a sequence appears twice in one step");
    // what the step takes, before anything changes: in the order below, the
    // last holder of a shared page keeps it
    size_t need = 0;
    std::unordered_map<int32_t, uint32_t> left;
    for (size_t i = 0; i < n; ++i) {
        const Seq &q = seqs_[slots[i]];
        if (rows[i] > max_len_ || q.len + (size_t)rows[i] > max_len_)
            invalid("a sequence of " + std::to_string(q.len) + " grows by " + std::to_string(rows[i]) + " past max_len " +
                    std::to_string(max_len_));
        if (rows[i] == 0) continue;
        need += pages_for(q.len + (size_t)rows[i]) - q.pages.size();
        if (q.len % page_size_ != 0) {
            auto it = left.emplace(q.pages.back(), refs_[(size_t)q.pages.back()]).first;
            if (it->second > 1) {
                ++need;
                --it->second;
            }
        }
    }
    if (need > free_.size())
        exhausted("out of pages: " + std::to_string(need) + " wanted, " + std::to_string(free_.size()) + " free");
    for (size_t i = 0; i < n; ++i) {
        Seq &q = seqs_[slots[i]];
        if (rows[i] == 0) continue;
        const size_t used = q.len % page_size_;
        if (used != 0 && refs_[(size_t)q.pages.back()] > 1) {
            const int32_t src = q.pages.back(), dst = take();
            --refs_[(size_t)src];
            q.pages.back() = dst;
            q.dirty = std::min(q.dirty, q.pages.size() - 1);
            copies->push_back({src, dst, (int32_t)used});
        }
        q.len += (size_t)rows[i];
        while (q.pages.size() < pages_for(q.len)) q.pages.push_back(take());
    }
}

void PageMap::undo_extend(const uint64_t *seqs, const uint64_t *rows, size_t n, std::vector<PageCopy> copies) {
    for (size_t i = n; i-- > 0;) {
        if (rows[i] == 0) continue;
        Seq &q = seqs_[slot(seqs[i])];
        q.len -= (size_t)rows[i];
        while (q.pages.size() > pages_for(q.len)) {
            release(q.pages.back());
            q.pages.pop_back();
        }
        // the copies are in the order of the sequences that took them
        if (!copies.empty() && q.len % page_size_ != 0 && copies.back().dst == q.pages.back()) {
            release(q.pages.back());
            q.pages.back() = copies.back().src;
            ++refs_[(size_t)copies.back().src];
            copies.pop_back();
        }
        q.dirty = std::min(q.dirty, q.pages.size());
    }
}

std::vector<PageCopy> PageMap::plan_compact() const {
    const size_t used = refs_.size() - free_.size();
    std::vector<PageCopy> moves;
    size_t hole = 0;
    for (size_t p = refs_.size(); p-- > used;) {
        if (refs_[p] == 0) continue;
        while (refs_[hole] != 0) ++hole;
        moves.push_back({(int32_t)p, (int32_t)hole++, (int32_t)page_size_});
    }
    return moves;
}

void PageMap::make_compact(const std::vector<PageCopy> &moves) {
    if (moves.empty()) return;
    const size_t used = refs_.size() - free_.size();
    std::vector<int32_t> to(refs_.size());
    for (size_t i = 0; i < to.size(); ++i) to[i] = (int32_t)i;
    for (const PageCopy &m : moves) {
        to[(size_t)m.src] = m.dst;
        refs_[(size_t)m.dst] = refs_[(size_t)m.src];
        refs_[(size_t)m.src] = 0;
    }
    for (Seq &q : seqs_) {
        if (!q.open) continue;
        for (size_t i = 0; i < q.pages.size(); ++i) {
            const int32_t p = to[(size_t)q.pages[i]];
            if (p == q.pages[i]) continue;
            q.pages[i] = p;
            q.dirty = std::min(q.dirty, i);
        }
    }
    free_.clear();
    for (size_t p = used; p < refs_.size(); ++p) free_.push_back((int32_t)p);
}

}  // namespace krt
