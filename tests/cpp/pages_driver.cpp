// The page bookkeeping behind a C interface, for tests/test_pages.py.
#include "../../kernrt_b200/csrc/pages.h"

#include <cstring>

using namespace krt;

namespace {
char g_msg[512];
template <class F>
int run(F &&fn) {
    try {
        fn();
        return 0;
    } catch (const PageError &e) {
        std::strncpy(g_msg, e.msg.c_str(), sizeof g_msg - 1);
        return e.exhausted ? 2 : 1;
    }
}
size_t put(const std::vector<PageCopy> &c, int32_t *out) {
    for (size_t i = 0; i < c.size(); ++i) {
        out[3 * i] = c[i].src;
        out[3 * i + 1] = c[i].dst;
        out[3 * i + 2] = c[i].rows;
    }
    return c.size();
}
}  // namespace

extern "C" {
const char *pm_msg() { return g_msg; }
void *pm_new(size_t pages, size_t page, size_t seqs, size_t len) { return new PageMap(pages, page, seqs, len); }
void pm_delete(void *m) { delete static_cast<PageMap *>(m); }
size_t pm_available(void *m) { return static_cast<PageMap *>(m)->available(); }
int pm_open(void *m, uint64_t *out) {
    return run([&] { *out = static_cast<PageMap *>(m)->open(); });
}
int pm_fork(void *m, uint64_t seq, size_t len, size_t n, uint64_t *out) {
    return run([&] {
        const auto got = static_cast<PageMap *>(m)->fork(seq, len, n);
        for (size_t i = 0; i < got.size(); ++i) out[i] = got[i];
    });
}
int pm_copy(void *m, uint64_t seq, size_t len, uint64_t *out, int32_t *copies, size_t *n) {
    return run([&] {
        std::vector<PageCopy> c;
        *out = static_cast<PageMap *>(m)->copy(seq, len, &c);
        *n = put(c, copies);
    });
}
int pm_trim(void *m, uint64_t seq, size_t len) {
    return run([&] { static_cast<PageMap *>(m)->trim(seq, len); });
}
int pm_close(void *m, const uint64_t *seqs, size_t n) {
    return run([&] { static_cast<PageMap *>(m)->close(seqs, n); });
}
int pm_extend(void *m, const uint64_t *seqs, const uint64_t *rows, size_t n, int32_t *copies, size_t *n_copies) {
    return run([&] {
        std::vector<PageCopy> c;
        static_cast<PageMap *>(m)->extend(seqs, rows, n, &c);
        *n_copies = put(c, copies);
    });
}
size_t pm_compact(void *m, int32_t *copies) { return put(static_cast<PageMap *>(m)->compact(), copies); }
// length, pages, and the first page that changed since the last call
int pm_table(void *m, uint64_t seq, size_t *len, int32_t *pages, size_t *n, size_t *dirty) {
    return run([&] {
        auto *p = static_cast<PageMap *>(m);
        PageMap::Seq &q = p->at(p->slot(seq));
        *len = q.len;
        *n = q.pages.size();
        *dirty = q.dirty;
        for (size_t i = 0; i < q.pages.size(); ++i) pages[i] = q.pages[i];
        q.dirty = q.pages.size();
    });
}
}
