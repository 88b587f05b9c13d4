// Who holds which page of a paged key / value cache: host arithmetic alone, no CUDA.  Every call checks its arguments, changes
// the books and leaves behind what has to change on the device; a call that fails changes nothing.
#pragma once
#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <vector>

namespace ab {

struct KvCopy { uint32_t src, dst, rows; };         // pages; the first `rows` positions of every layer's keys and values
// kind << 28 | sequence, then  RUN: w entries of the table's row from entry y on are z, z + 1, ..;  LEN: length y, first
// writable position z;  ROW: the first w entries are those of sequence y's row;  CLEAR: entries y .. z - 1 are -1
struct KvRec { uint32_t x, y, z, w; };
enum : uint32_t { REC_RUN, REC_LEN, REC_ROW, REC_CLEAR };
// Copies are made first (a page that a record gives to another sequence is still its old one), then the records, in any order.
struct KvUpdate { std::vector<KvCopy> copies; std::vector<KvRec> recs; };

enum { PAGES_OK = 0, PAGES_FULL = -2, PAGES_INVALID = -3 };     // ADAMAH_OK, ADAMAH_ERR_MEMORY, ADAMAH_ERR_INVALID

class KvPages {
public:
    static constexpr uint32_t NONE = 0xFFFFFFFFu;
    uint32_t page = 0, n_pages = 0, max_seqs = 0, max_pages = 0, n_free = 0;
    std::vector<int32_t> table, lens, own;          // [max_seqs][max_pages], positions, first position that the sequence may write
    char why[160] = "";

    void init(uint32_t page_size, uint32_t pages, uint32_t seqs, uint32_t pages_per_seq) {
        page = page_size; n_pages = n_free = pages; max_seqs = seqs; max_pages = pages_per_seq;
        table.assign((size_t)seqs * pages_per_seq, -1); lens.assign(seqs, 0); own.assign(seqs, 0);
        refs.assign(pages, 0); stamp.assign(seqs, 0);
    }

    uint32_t longest() {                            // the largest length
        if (stale) { most = 0; for (int32_t n : lens) most = std::max(most, (uint32_t)n); stale = false; }
        return most;
    }

    int extend(uint32_t n, const uint32_t* seqs, const uint32_t* n_tokens, KvUpdate& u) {
        if (int rc = check("kv_extend", seqs, n, n_tokens)) return rc;
        const uint64_t cap = (uint64_t)max_pages * page;
        uint64_t grown = 0;
        for (uint32_t i = 0; i < n; ++i) {
            const uint64_t len = (uint64_t)lens[seqs[i]], to = len + n_tokens[i];
            if (to > cap) return bad("kv_extend: sequence %u to %llu positions of at most %llu", seqs[i], (unsigned long long)to, (unsigned long long)cap);
            grown += pages_for(to) - pages_for(len);
        }
        if (grown > n_free) return full(grown);
        u.copies.reserve(n); u.recs.reserve(2 * (size_t)n + grown);
        std::vector<uint32_t> shared(n, NONE);      // the page that an entry writes into and others hold: the last holder keeps it
        uint64_t need = grown;
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t len = (uint32_t)lens[seqs[i]];
            if (!n_tokens[i] || len % page == 0) continue;
            const uint32_t p = (uint32_t)at(seqs[i], len / page);
            if (refs[p] > 1) { --refs[p]; shared[i] = p; ++need; }
        }
        if (need > n_free) {
            for (uint32_t p : shared) if (p != NONE) ++refs[p];
            return full(need);
        }
        for (uint32_t i = 0; i < n; ++i) {
            if (!n_tokens[i]) continue;
            const uint32_t s = seqs[i], len = (uint32_t)lens[s], to = len + n_tokens[i];
            if (shared[i] != NONE) {
                const uint32_t p = take();
                u.copies.push_back({shared[i], p, len % page});
                give(u, s, len / page, p);
            }
            for (uint32_t j = pages_for(len); j < pages_for(to); ++j) give(u, s, j, take());
            lens[s] = (int32_t)to;
            most = std::max(most, to);
            add_len(u, s);
        }
        return PAGES_OK;
    }

    int fork(uint32_t src, uint32_t n, const uint32_t* dsts, uint32_t n_tokens, KvUpdate& u) {
        if (int rc = check("kv_fork", dsts, n, dsts)) return rc;
        if (src >= max_seqs) return bad("kv_fork: sequence %u of a cache for %u", src, max_seqs);
        if (n_tokens > (uint32_t)lens[src]) return bad("kv_fork: %u positions of a sequence of %d", n_tokens, lens[src]);
        for (uint32_t i = 0; i < n; ++i)
            if (dsts[i] == src || lens[dsts[i]]) return bad("kv_fork: sequence %u is not empty", dsts[i]);
        if (!n || !n_tokens) return PAGES_OK;
        const uint32_t pages = pages_for(n_tokens);
        u.recs.reserve(2 * (size_t)n + 1);
        for (uint32_t j = 0; j < pages; ++j) refs[(uint32_t)at(src, j)] += n;
        for (uint32_t i = 0; i < n; ++i) {
            std::copy_n(&at(src, 0), pages, &at(dsts[i], 0));
            lens[dsts[i]] = own[dsts[i]] = (int32_t)n_tokens;
            u.recs.push_back(rec(REC_ROW, dsts[i], src, 0, pages));
            add_len(u, dsts[i]);
        }
        // what it shares now, and anything before it, is not the source's to write either
        if (own[src] < (int32_t)n_tokens) { own[src] = (int32_t)n_tokens; add_len(u, src); }
        return PAGES_OK;
    }

    int truncate(uint32_t n, const uint32_t* seqs, const uint32_t* to, KvUpdate& u) {
        if (int rc = check("kv_truncate", seqs, n, to)) return rc;
        for (uint32_t i = 0; i < n; ++i)
            if (to[i] > (uint32_t)lens[seqs[i]]) return bad("kv_truncate: sequence %u of %d positions to %u", seqs[i], lens[seqs[i]], to[i]);
        u.recs.reserve(2 * (size_t)n);
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t s = seqs[i], old = pages_for((uint32_t)lens[s]), now = pages_for(to[i]);
            if (to[i] == (uint32_t)lens[s]) continue;
            for (uint32_t j = now; j < old; ++j) { drop((uint32_t)at(s, j)); at(s, j) = -1; }
            stale |= (uint32_t)lens[s] == most;
            lens[s] = (int32_t)to[i];
            own[s] = std::min(own[s], (int32_t)to[i]);
            if (now < old) u.recs.push_back(rec(REC_CLEAR, s, now, old, 0));
            add_len(u, s);
        }
        return PAGES_OK;
    }

    int compact(uint32_t* n_live, KvUpdate& u) {
        const uint32_t live = n_pages - n_free;
        std::vector<int32_t> to(n_pages, -1);
        uint32_t hole = 0;
        for (uint32_t p = live; p < n_pages; ++p) {
            if (!refs[p]) continue;
            while (refs[hole]) ++hole;              // below `live` as many pages are free as are held above
            to[p] = (int32_t)hole;
            u.copies.push_back({p, hole++, page});
        }
        auto held = [&](auto f) {
            for (uint32_t s = 0; s < max_seqs; ++s)
                for (uint32_t j = 0, m = pages_for((uint32_t)lens[s]); j < m; ++j) f(s, j);
        };
        if (!u.copies.empty()) {
            held([&](uint32_t s, uint32_t j) { if (const int32_t t = to[(uint32_t)at(s, j)]; t >= 0) add_page(u, s, j, (uint32_t)t); });
            // nothing below can fail
            held([&](uint32_t s, uint32_t j) { if (const int32_t t = to[(uint32_t)at(s, j)]; t >= 0) at(s, j) = t; });
            for (const KvCopy& c : u.copies) { refs[c.dst] = refs[c.src]; refs[c.src] = 0; }
            first_free = live;
        }
        *n_live = live;
        return PAGES_OK;
    }

private:
    std::vector<uint32_t> refs, stamp;              // sequences that hold a page; of a sequence, the call that named it last
    uint32_t call = 0, first_free = 0;              // no page below first_free is free
    uint32_t most = 0;                              // longest(), unless it is `stale`: then at least that
    bool stale = false;

    uint32_t pages_for(uint64_t n) const { return (uint32_t)((n + page - 1) / page); }
    int32_t& at(uint32_t seq, uint32_t i) { return table[(size_t)seq * max_pages + i]; }
    static KvRec rec(uint32_t kind, uint32_t seq, uint32_t y, uint32_t z, uint32_t w) { return KvRec{kind << 28 | seq, y, z, w}; }
    uint32_t take() {                               // the lowest free page; the caller knows that there is one
        while (refs[first_free]) ++first_free;
        refs[first_free] = 1; --n_free;
        return first_free++;
    }
    void drop(uint32_t p) { if (--refs[p] == 0) { ++n_free; first_free = std::min(first_free, p); } }
    void give(KvUpdate& u, uint32_t seq, uint32_t i, uint32_t p) { at(seq, i) = (int32_t)p; add_page(u, seq, i, p); }
    void add_page(KvUpdate& u, uint32_t seq, uint32_t i, uint32_t p) {
        if (!u.recs.empty()) {
            KvRec& l = u.recs.back();
            if (l.x == (REC_RUN << 28 | seq) && l.y + l.w == i && l.z + l.w == p) { ++l.w; return; }
        }
        u.recs.push_back(rec(REC_RUN, seq, i, p, 1));
    }
    void add_len(KvUpdate& u, uint32_t seq) { u.recs.push_back(rec(REC_LEN, seq, (uint32_t)lens[seq], (uint32_t)own[seq], 0)); }

    int bad(const char* fmt, ...) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(why, sizeof why, fmt, ap);
        va_end(ap);
        return PAGES_INVALID;
    }
    int full(uint64_t need) {
        snprintf(why, sizeof why, "kv_extend: %llu pages needed, %u of %u free", (unsigned long long)need, n_free, n_pages);
        return PAGES_FULL;
    }
    // Every sequence of a call exists and stands in it once.
    int check(const char* name, const uint32_t* seqs, uint32_t n, const uint32_t* with) {
        if (n && (!seqs || !with)) return bad("%s: null pointer", name);
        if (++call == 0) { std::fill(stamp.begin(), stamp.end(), 0u); call = 1; }
        for (uint32_t i = 0; i < n; ++i) {
            if (seqs[i] >= max_seqs) return bad("%s: sequence %u of a cache for %u", name, seqs[i], max_seqs);
            if (stamp[seqs[i]] == call) return bad("%s: sequence %u is named twice", name, seqs[i]);
            stamp[seqs[i]] = call;
        }
        return PAGES_OK;
    }
};

}  // namespace ab
