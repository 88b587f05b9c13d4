// The page books of a cache (adam_b200/csrc/kv_pages.h) behind a C interface, with host arrays in the place of the device's:
// a position is one number.
#include "../adam_b200/csrc/kv_pages.h"

#include <cstring>
#include <string>

using namespace ab;

struct Cache { KvPages books; std::vector<int32_t> pool, table, lens, own; std::string why; };

static int apply(Cache* c, int rc, const KvUpdate& u) {
    c->why = rc ? c->books.why : "";
    if (rc) return rc;
    for (const KvCopy& k : u.copies) std::copy_n(&c->pool[(size_t)k.src * c->books.page], k.rows, &c->pool[(size_t)k.dst * c->books.page]);
    for (const KvRec& r : u.recs) {
        const uint32_t seq = r.x & 0x0FFFFFFFu;
        int32_t* row = &c->table[(size_t)seq * c->books.max_pages];
        switch (r.x >> 28) {
        case REC_RUN: for (uint32_t j = 0; j < r.w; ++j) row[r.y + j] = (int32_t)(r.z + j); break;
        case REC_LEN: c->lens[seq] = (int32_t)r.y; c->own[seq] = (int32_t)r.z; break;
        case REC_ROW: std::copy_n(&c->table[(size_t)r.y * c->books.max_pages], r.w, row); break;
        default: std::fill(row + r.y, row + r.z, -1);
        }
    }
    return rc;
}

extern "C" {
Cache* kv_new(uint32_t page, uint32_t n_pages, uint32_t max_seqs, uint32_t max_pages) {
    Cache* c = new Cache;
    c->books.init(page, n_pages, max_seqs, max_pages);
    c->pool.assign((size_t)page * n_pages, 0); c->table.assign((size_t)max_seqs * max_pages, -1);
    c->lens.assign(max_seqs, 0); c->own.assign(max_seqs, 0);
    return c;
}
void kv_delete(Cache* c) { delete c; }
int kv_extend(Cache* c, uint32_t n, const uint32_t* s, const uint32_t* t) { KvUpdate u; return apply(c, c->books.extend(n, s, t, u), u); }
int kv_fork(Cache* c, uint32_t src, uint32_t n, const uint32_t* d, uint32_t t) { KvUpdate u; return apply(c, c->books.fork(src, n, d, t, u), u); }
int kv_truncate(Cache* c, uint32_t n, const uint32_t* s, const uint32_t* t) { KvUpdate u; return apply(c, c->books.truncate(n, s, t, u), u); }
int kv_compact(Cache* c, uint32_t* live) { KvUpdate u; return apply(c, c->books.compact(live, u), u); }
const char* kv_why(Cache* c) { return c->why.c_str(); }
// host books: table, lens, own, free pages; the "device's": pool, table, lens, own
void kv_read(Cache* c, int32_t* table, int32_t* lens, int32_t* own, uint32_t* n_free, int32_t* pool, int32_t* d_table, int32_t* d_lens, int32_t* d_own) {
    auto put = [](const std::vector<int32_t>& v, int32_t* to) { std::copy(v.begin(), v.end(), to); };
    put(c->books.table, table); put(c->books.lens, lens); put(c->books.own, own); *n_free = c->books.n_free;
    put(c->pool, pool); put(c->table, d_table); put(c->lens, d_lens); put(c->own, d_own);
}
uint32_t kv_longest(Cache* c) { return c->books.longest(); }
// position p of sequence s as the append operator writes it: refused below the first writable position
int kv_write(Cache* c, uint32_t s, uint32_t p, int32_t value) {
    if (p >= (uint32_t)c->lens[s] || p < (uint32_t)c->own[s]) return -1;
    c->pool[(size_t)c->table[(size_t)s * c->books.max_pages + p / c->books.page] * c->books.page + p % c->books.page] = value;
    return 0;
}
}
