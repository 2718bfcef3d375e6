// Which pages the sequences of a pool have: plain host bookkeeping, no device. Every operation either finds what it needs and then
// changes the books without a step that can fail, or changes nothing. What has to follow on the device is left in two lists:
// changes of the device's page tables and copies of pages.
#pragma once
#include <stdint.h>

#include <algorithm>
#include <new>
#include <vector>

#include "../../include/mechta_kv.h"

namespace mkv {

void set_error(const char *fmt, ...);

// table[dst + i] = val + i for i < n, or with COPY in n: = table[val + i]
struct TableOp {
    static constexpr uint32_t COPY = 0x80000000u;
    uint32_t dst, val, n;
};
// the first `rows` rows of page src, K and V of every layer, to page dst
struct PageCopy {
    uint32_t src, dst, rows;
};

// A set of free numbers that gives out its lowest.
class FreeSet {
    std::vector<uint64_t> bits;
    size_t low = 0; // no free number below word `low`
    uint32_t count = 0;

  public:
    explicit FreeSet(uint32_t n = 0) : bits((n + 63ull) / 64ull, ~0ull), count(n) {
        if (n % 64u) bits.back() = (1ull << (n % 64u)) - 1ull;
    }
    uint32_t size() const { return count; }
    bool has(uint32_t x) const { return bits[x / 64u] >> (x % 64u) & 1u; }
    uint32_t lowest() { // (not when empty)
        while (!bits[low]) low++;
        return (uint32_t)(low * 64u) + (uint32_t)__builtin_ctzll(bits[low]);
    }
    uint32_t take() { // (not when empty)
        const uint32_t x = lowest();
        bits[low] &= bits[low] - 1ull;
        count--;
        return x;
    }
    void take(uint32_t x) {
        bits[x / 64u] &= ~(1ull << (x % 64u));
        count--;
    }
    // Calls f for the numbers in [a, b) that are free, or that are not, in ascending order, until it returns false.
    template <class F> void each(uint32_t a, uint32_t b, bool free, const F &f) const {
        for (size_t w = a / 64u; w * 64u < b; w++) {
            uint64_t x = free ? bits[w] : ~bits[w];
            if (w == a / 64u) x &= ~0ull << (a % 64u);
            if ((w + 1u) * 64u > b) x &= (1ull << (b % 64u)) - 1ull;
            for (; x; x &= x - 1ull)
                if (!f((uint32_t)(w * 64u) + (uint32_t)__builtin_ctzll(x))) return;
        }
    }
    void give(uint32_t x) {
        bits[x / 64u] |= 1ull << (x % 64u);
        low = std::min<size_t>(low, x / 64u);
        count++;
    }
};

class PageBook {
  public:
    struct Seq {
        bool live = false;
        uint32_t len = 0, before = 0;  // before: len in front of the last write
        uint64_t stamp = 0;            // the last call that named the sequence, to find one that is named twice
        std::vector<uint32_t> pages;
        std::vector<uint32_t> written; // per layer: rows [0, written) are there
    };
    uint32_t n_pages = 0, page = 0, max_seqs = 0, max_pages = 0; // max_pages: of one sequence
    uint64_t max_tokens = 0;
    int n_layers = 0;
    std::vector<Seq> seqs;
    std::vector<TableOp> ops;
    std::vector<PageCopy> copies;

    PageBook(uint32_t n_pages_, uint32_t page_, uint32_t max_seqs_, uint32_t max_tokens_, int layers)
        : n_pages(n_pages_), page(page_), max_seqs(max_seqs_), max_tokens(max_tokens_), n_layers(layers), seqs(max_seqs_),
          free_pages(n_pages_), free_seqs(max_seqs_), refs(n_pages_, 0u) {
        max_pages = std::min(pages_of(max_tokens_), n_pages_);
    }
    uint32_t free_count() const { return free_pages.size(); }
    uint32_t pages_of(uint64_t rows) const { return (uint32_t)((rows + page - 1u) / page); }
    bool alive(uint32_t s) const { return s < max_seqs && seqs[s].live; }
    mkv_status need(uint32_t s) const {
        if (alive(s)) return MKV_OK;
        set_error("no sequence %u", s);
        return MKV_ERR_INVALID;
    }

    mkv_status create(uint32_t *out) {
        if (free_seqs.size() == 0) {
            set_error("all %u sequences are in use", max_seqs);
            return MKV_ERR_NOMEM;
        }
        const uint32_t c = free_seqs.lowest();
        seqs[c].written.assign((size_t)n_layers, 0u); // (what may fail for want of memory comes first)
        open(*out = free_seqs.take(), 0u);
        return MKV_OK;
    }

    mkv_status fork(uint32_t s, uint32_t len, bool copy, int n, uint32_t *children) {
        mkv_status st = need(s);
        if (st != MKV_OK) return st;
        if (n < 1 || (uint32_t)n > max_seqs) {
            set_error("fork of %d sequences: 1 to %u", n, max_seqs);
            return MKV_ERR_INVALID;
        }
        if (len > seqs[s].len) {
            set_error("fork at %u: only %u rows are valid", len, seqs[s].len);
            return MKV_ERR_STATE;
        }
        const uint32_t np = pages_of(len);
        if (free_seqs.size() < (uint32_t)n || (copy && (uint64_t)np * (uint32_t)n > free_pages.size())) {
            set_error("fork of %d sequences: %u sequences and %u pages are free", n, free_seqs.size(), free_pages.size());
            return MKV_ERR_NOMEM;
        }
        // All that may fail for want of memory comes first; a sequence keeps its vectors' room for the next one of its number.
        for (uint32_t i = 0, c = free_seqs.lowest(); i < (uint32_t)n; i++, c++) {
            while (!free_seqs.has(c)) c++;
            seqs[c].pages.reserve(np);
            seqs[c].written.assign((size_t)n_layers, 0u);
        }
        ops.reserve(ops.size() + (size_t)n * (copy ? np : 1u));
        if (copy) copies.reserve(copies.size() + (size_t)n * np);
        const std::vector<uint32_t> &pages = seqs[s].pages;
        for (int i = 0; i < n; i++) {
            const uint32_t c = children[i] = free_seqs.take();
            open(c, len);
            for (int l = 0; l < n_layers; l++) seqs[c].written[(size_t)l] = std::min(seqs[s].written[(size_t)l], len);
            if (!copy) {
                seqs[c].pages.assign(pages.begin(), pages.begin() + np);
                if (np > 0u) ops.push_back({c * max_pages, s * max_pages, np | TableOp::COPY});
                continue;
            }
            for (uint32_t j = 0; j < np; j++) {
                const uint32_t d = take_page();
                copies.push_back({pages[j], d, std::min(page, len - j * page)});
                seqs[c].pages.push_back(d);
                entry(c, j, d);
            }
        }
        for (uint32_t j = 0; !copy && j < np; j++) refs[pages[j]] += (uint32_t)n;
        return MKV_OK;
    }

    mkv_status free_all(const uint32_t *list, int n) {
        clock++;
        for (int i = 0; i < n; i++) {
            mkv_status st = need(list[i]);
            if (st != MKV_OK) return st;
            if (seqs[list[i]].stamp == clock) {
                set_error("sequence %u is named twice", list[i]);
                return MKV_ERR_INVALID;
            }
            seqs[list[i]].stamp = clock;
        }
        for (int i = 0; i < n; i++) {
            shrink(list[i], 0u);
            seqs[list[i]].live = false;
            free_seqs.give(list[i]);
        }
        return MKV_OK;
    }

    mkv_status truncate(uint32_t s, uint32_t len) {
        mkv_status st = need(s);
        if (st != MKV_OK) return st;
        if (len > seqs[s].len) {
            set_error("cannot truncate to %u: only %u rows are valid", len, seqs[s].len);
            return MKV_ERR_STATE;
        }
        cut(s, len);
        return MKV_OK;
    }

    mkv_status set_len(uint32_t s, uint32_t len) {
        mkv_status st = need(s);
        if (st != MKV_OK) return st;
        if (len > max_tokens) {
            set_error("length %u beyond the pool's longest sequence %llu", len, (unsigned long long)max_tokens);
            return MKV_ERR_CAPACITY;
        }
        if (len < seqs[s].len) {
            set_error("length %u below the current one %u: truncate", len, seqs[s].len);
            return MKV_ERR_STATE;
        }
        const uint32_t have = (uint32_t)seqs[s].pages.size(), want = std::max(have, pages_of(len));
        if (want - have > free_pages.size()) {
            set_error("%u pages are wanted, %u are free", want - have, free_pages.size());
            return MKV_ERR_NOMEM;
        }
        grow_room(seqs[s].pages, want);
        ops.reserve(ops.size() + (want - have));
        extend(s, want);
        seqs[s].len = len;
        for (uint32_t &w : seqs[s].written) w = len;
        return MKV_OK;
    }

    // Room for the rows of the items in one layer: missing pages, own pages in place of shared ones. dry: the checks alone.
    mkv_status write(int layer, const mkv_seq_rows *items, int n, bool dry) {
        clock++;
        uint64_t fresh = 0;
        // Pages that an item of this call leaves to their other holders count one holder less for the items behind it. refs is put back
        // before anything is decided.
        left.clear();
        const mkv_status st = plan(layer, items, n, fresh);
        for (uint32_t p : left) refs[p]++;
        if (st != MKV_OK) return st;
        if (fresh > free_pages.size()) {
            set_error("%llu pages are wanted, %u are free", (unsigned long long)fresh, free_pages.size());
            return MKV_ERR_NOMEM;
        }
        if (dry) return MKV_OK;
        ops.reserve(ops.size() + fresh);
        copies.reserve(copies.size() + fresh);
        for (int i = 0; i < n; i++) {
            const mkv_seq_rows &it = items[i];
            if (it.ntok == 0u) continue;
            Seq &s = seqs[it.seq];
            s.before = s.len;
            const uint32_t have = (uint32_t)s.pages.size(), last = (it.pos + it.ntok - 1u) / page;
            bool own = true;
            for (uint32_t j = it.pos / page; j <= last && j < have; j++) {
                const uint32_t p = s.pages[j];
                if (refs[p] == 1u) continue;
                own = false;
                const uint32_t d = take_page(), rows = j * page < it.pos ? it.pos - j * page : 0u;
                refs[p]--;
                if (rows) copies.push_back({p, d, rows});
                s.pages[j] = d;
                entry(it.seq, j, d);
            }
            if (last >= have) extend(it.seq, last + 1u);
            if (!own) // the new pages have no layer's rows from pos on
                for (uint32_t &w : s.written) w = std::min(w, it.pos);
        }
        // Pages that rows behind the new end had go back only now: none of them is a page that this call has taken or copies.
        for (int i = 0; i < n; i++) {
            const mkv_seq_rows &it = items[i];
            if (it.ntok == 0u) continue;
            Seq &s = seqs[it.seq];
            const uint32_t end = it.pos + it.ntok;
            if (end < s.len) cut(it.seq, end);
            s.len = end;
            s.written[(size_t)layer] = end;
        }
        return MKV_OK;
    }

    // The rows of the last write() did not get to the device: they do not count. (What else it did stays: pages taken or copied are the
    // sequences' own, rows behind the new ones are forgotten.)
    void not_written(int layer, const mkv_seq_rows *items, int n) {
        for (int i = 0; i < n; i++) {
            if (items[i].ntok == 0u) continue;
            Seq &s = seqs[items[i].seq];
            s.written[(size_t)layer] = std::min(s.written[(size_t)layer], items[i].pos);
            if (s.len > s.before) cut(items[i].seq, s.before);
        }
    }

    mkv_status compact(uint32_t *moved) {
        const uint32_t used = n_pages - free_pages.size();
        if (moved) *moved = 0u;
        if (used == n_pages || free_pages.lowest() >= used) return MKV_OK; // the pages in use are the lowest
        std::vector<uint32_t> src, dst;
        free_pages.each(used, n_pages, false, [&](uint32_t p) { return src.push_back(p), true; });
        dst.reserve(src.size());
        free_pages.each(0u, used, true, [&](uint32_t p) { return dst.push_back(p), dst.size() < src.size(); });
        size_t entries = 0;
        for (const Seq &s : seqs)
            for (uint32_t p : s.pages) entries += p >= used;
        ops.reserve(ops.size() + entries);
        copies.reserve(copies.size() + src.size());
        for (size_t i = 0; i < src.size(); i++) {
            copies.push_back({src[i], dst[i], page});
            free_pages.take(dst[i]);
            free_pages.give(src[i]);
            refs[dst[i]] = refs[src[i]];
            refs[src[i]] = 0u;
        }
        for (uint32_t q = 0; q < max_seqs; q++) {
            Seq &s = seqs[q];
            for (uint32_t j = 0; j < s.pages.size(); j++)
                if (s.pages[j] >= used) {
                    s.pages[j] = dst[(size_t)(std::lower_bound(src.begin(), src.end(), s.pages[j]) - src.begin())];
                    entry(q, j, s.pages[j]);
                }
        }
        if (moved) *moved = (uint32_t)src.size();
        return MKV_OK;
    }

  private:
    FreeSet free_pages, free_seqs;
    std::vector<uint32_t> refs; // sequences that have the page
    std::vector<uint32_t> left; // of write()
    uint64_t clock = 0;

    static void grow_room(std::vector<uint32_t> &v, size_t n) {
        if (n > v.capacity()) v.reserve(std::max(n, 2u * v.capacity()));
    }
    void open(uint32_t s, uint32_t len) {
        seqs[s].live = true;
        seqs[s].len = len;
        seqs[s].pages.clear();
    }
    // The checks of write(); `fresh`: the pages that it needs.
    mkv_status plan(int layer, const mkv_seq_rows *items, int n, uint64_t &fresh) {
        for (int i = 0; i < n; i++) {
            const mkv_seq_rows &it = items[i];
            mkv_status st = need(it.seq);
            if (st != MKV_OK) return st;
            Seq &s = seqs[it.seq];
            if (s.stamp == clock) {
                set_error("sequence %u is named twice", it.seq);
                return MKV_ERR_INVALID;
            }
            s.stamp = clock;
            const uint64_t end = (uint64_t)it.pos + it.ntok;
            if (end > max_tokens) {
                set_error("rows [%u, %llu) do not fit a sequence of %llu", it.pos, (unsigned long long)end, (unsigned long long)max_tokens);
                return MKV_ERR_CAPACITY;
            }
            if (it.pos > s.written[(size_t)layer]) {
                set_error("sequence %u has %u rows in layer %d: a write at %u would leave a gap", it.seq, s.written[(size_t)layer], layer, it.pos);
                return MKV_ERR_STATE;
            }
            if (it.ntok == 0u) continue;
            const uint32_t have = (uint32_t)s.pages.size(), last = (uint32_t)((end - 1u) / page);
            if (last >= max_pages) { // (a pool of fewer pages than its longest sequence would need)
                set_error("rows [%u, %llu) need more pages than the pool has", it.pos, (unsigned long long)end);
                return MKV_ERR_NOMEM;
            }
            for (uint32_t j = it.pos / page; j <= last && j < have; j++) {
                const uint32_t p = s.pages[j];
                if (refs[p] == 1u) continue;
                try {
                    left.push_back(p);
                } catch (const std::bad_alloc &) {
                    set_error("out of host memory");
                    return MKV_ERR_NOMEM;
                }
                refs[p]--;
                fresh++;
            }
            if (last >= have) fresh += last + 1u - have;
            try {
                grow_room(s.pages, last + 1u);
            } catch (const std::bad_alloc &) {
                set_error("out of host memory");
                return MKV_ERR_NOMEM;
            }
        }
        return MKV_OK;
    }
    uint32_t take_page() {
        const uint32_t p = free_pages.take();
        refs[p] = 1u;
        return p;
    }
    void extend(uint32_t s, uint32_t want) { // (room and pages are there)
        while (seqs[s].pages.size() < want) {
            const uint32_t p = take_page();
            seqs[s].pages.push_back(p);
            entry(s, (uint32_t)seqs[s].pages.size() - 1u, p);
        }
    }
    void shrink(uint32_t s, uint32_t want) {
        std::vector<uint32_t> &v = seqs[s].pages;
        if (v.size() <= want) return;
        for (size_t j = want; j < v.size(); j++)
            if (--refs[v[j]] == 0u) free_pages.give(v[j]);
        v.resize(want);
    }
    void cut(uint32_t s, uint32_t len) {
        shrink(s, pages_of(len));
        seqs[s].len = len;
        for (uint32_t &w : seqs[s].written) w = std::min(w, len);
    }
    // the sequence's page number j is p: joins the run of the entry in front where it continues it
    void entry(uint32_t s, uint32_t j, uint32_t p) {
        const uint32_t at = s * max_pages + j;
        if (!ops.empty()) {
            TableOp &o = ops.back();
            if (!(o.n & TableOp::COPY) && o.dst + o.n == at && o.val + o.n == p) {
                o.n++;
                return;
            }
        }
        ops.push_back({at, p, 1u});
    }
};

} // namespace mkv
