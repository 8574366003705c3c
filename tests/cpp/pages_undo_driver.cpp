// pages_driver.cpp, and the calls that take an operation back.
#include "pages_driver.cpp"

extern "C" {
void pm_undo_extend(void *m, const uint64_t *seqs, const uint64_t *rows, size_t n, const int32_t *copies, size_t n_copies) {
    std::vector<PageCopy> c;
    for (size_t i = 0; i < n_copies; ++i) c.push_back({copies[3 * i], copies[3 * i + 1], copies[3 * i + 2]});
    static_cast<PageMap *>(m)->undo_extend(seqs, rows, n, c);
}
size_t pm_plan_compact(void *m, int32_t *copies) { return put(static_cast<PageMap *>(m)->plan_compact(), copies); }
}
