// hq_kv_pool.cu -- host bookkeeping of the paged key/value cache: which pages a
// sequence has, how many sequences share a page.
//
// A fork shares every page; the first of the sharers that writes into a partly
// filled last page gets a copy of it (copy on write), so a fork moves nothing
// until it is written to, and then at most one page.  Every call works out what
// it needs before it changes anything.
#include "hq.h"

#include <algorithm>
#include <functional>
#include <new>
#include <queue>
#include <vector>

namespace {

struct Seq {
    bool live = false;
    int len = 0;
    std::vector<int32_t> pages;
};

}  // namespace

struct hq_kv_pool {
    int page_size = 0;
    int in_use = 0;
    std::vector<int> refs;  // per page
    std::priority_queue<int, std::vector<int>, std::greater<int>> free_pages, free_seqs;
    std::vector<Seq> seqs;

    bool has(int s) const { return s >= 0 && s < (int)seqs.size() && seqs[s].live; }
    int new_seq() {
        if (free_seqs.empty()) {
            seqs.emplace_back();
            seqs.back().live = true;
            return (int)seqs.size() - 1;
        }
        const int s = free_seqs.top();
        free_seqs.pop();
        seqs[s].live = true;
        return s;
    }
};

extern "C" {

HQ_API hq_kv_pool* hq_kv_pool_create(int num_pages, int page_size) {
    if (num_pages <= 0 || page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) ||
        (long long)num_pages * page_size > 0x7fffffffLL)
        return nullptr;
    hq_kv_pool* p = nullptr;
    try {
        p = new hq_kv_pool();
        p->page_size = page_size;
        p->refs.assign((size_t)num_pages, 0);
        std::vector<int> all((size_t)num_pages);
        for (int i = 0; i < num_pages; ++i) all[i] = i;
        p->free_pages = decltype(p->free_pages)(std::greater<int>(), std::move(all));
        return p;
    } catch (const std::bad_alloc&) {
        delete p;
        return nullptr;
    }
}

HQ_API void hq_kv_pool_destroy(hq_kv_pool* p) { delete p; }

HQ_API int hq_kv_pool_free_pages(const hq_kv_pool* p) { return p ? (int)p->free_pages.size() : 0; }

HQ_API int hq_kv_pool_new_seq(hq_kv_pool* p) {
    if (!p) return -1;
    try {
        return p->new_seq();
    } catch (const std::bad_alloc&) {
        return -1;
    }
}

HQ_API int hq_kv_pool_fork(hq_kv_pool* p, int seq) {
    if (!p || !p->has(seq)) return -1;
    try {
        std::vector<int32_t> pages = p->seqs[seq].pages;
        const int s = p->new_seq();
        for (int32_t g : pages) ++p->refs[g];
        p->seqs[s].pages.swap(pages);
        p->seqs[s].len = p->seqs[seq].len;
        return s;
    } catch (const std::bad_alloc&) {
        return -1;
    }
}

HQ_API hq_status hq_kv_pool_extend(hq_kv_pool* p, const int32_t* seqs, const int32_t* n_tokens, int n, hq_page_move* moves,
                                   int* n_moves) {
    if (!p || n < 0 || !n_moves || (n > 0 && (!seqs || !n_tokens || !moves))) return HQ_ERR_INVALID_ARG;
    for (int i = 0; i < n; ++i)
        if (n_tokens[i] < 0 || !p->has(seqs[i])) return HQ_ERR_INVALID_ARG;
    struct Before {
        int len;
        size_t pages;
        int32_t shared;  // the last page, where it was replaced by a copy; else -1
    };
    std::vector<Before> before;
    try {
        before.reserve((size_t)n);
    } catch (const std::bad_alloc&) {
        return HQ_ERR_OUT_OF_MEMORY;
    }
    auto take = [p] {
        const int g = p->free_pages.top();
        p->free_pages.pop();
        p->refs[g] = 1;
        ++p->in_use;
        return g;
    };
    auto give = [p](int32_t g) {
        p->refs[g] = 0;
        p->free_pages.push(g);  // within the room that the heap had when every page was free
        --p->in_use;
    };
    hq_status status = HQ_OK;
    int copies = 0;
    for (int i = 0; i < n && status == HQ_OK; ++i) {
        Seq& s = p->seqs[seqs[i]];
        Before was{s.len, s.pages.size(), -1};
        if ((long long)s.len + n_tokens[i] > 0x7fffffffLL) status = HQ_ERR_UNSUPPORTED_SHAPE;
        else if (n_tokens[i] > 0) {
            const bool copy = s.len % p->page_size && p->refs[s.pages.back()] > 1;
            const size_t want = ((size_t)s.len + n_tokens[i] + p->page_size - 1) / p->page_size;
            if (want - s.pages.size() + (copy ? 1 : 0) > p->free_pages.size()) status = HQ_ERR_OUT_OF_PAGES;
            else
                try {
                    s.pages.reserve(want);
                    if (copy) {
                        was.shared = s.pages.back();
                        s.pages.back() = take();
                        --p->refs[was.shared];
                        moves[copies++] = hq_page_move{was.shared, s.pages.back()};
                    }
                    while (s.pages.size() < want) s.pages.push_back(take());
                    s.len += n_tokens[i];
                } catch (const std::bad_alloc&) {  // of the reserve: nothing was taken
                    status = HQ_ERR_OUT_OF_MEMORY;
                }
        }
        if (status == HQ_OK) before.push_back(was);
    }
    if (status != HQ_OK) {  // last one first: a sequence may be named twice
        for (int i = (int)before.size() - 1; i >= 0; --i) {
            Seq& s = p->seqs[seqs[i]];
            for (; s.pages.size() > before[i].pages; s.pages.pop_back()) give(s.pages.back());
            if (before[i].shared >= 0) {
                give(s.pages.back());
                s.pages.back() = before[i].shared;
                ++p->refs[before[i].shared];
            }
            s.len = before[i].len;
        }
        return status;
    }
    *n_moves = copies;
    return HQ_OK;
}

HQ_API hq_status hq_kv_pool_free(hq_kv_pool* p, int seq) {
    if (!p || !p->has(seq)) return HQ_ERR_INVALID_ARG;
    Seq& s = p->seqs[seq];
    try {
        p->free_seqs.push(seq);
    } catch (const std::bad_alloc&) {
        return HQ_ERR_OUT_OF_MEMORY;
    }
    for (int32_t g : s.pages)
        if (--p->refs[g] == 0) {
            p->free_pages.push(g);  // within the room that the heap had when every page was free
            --p->in_use;
        }
    s.pages.clear();
    s.len = 0;
    s.live = false;
    return HQ_OK;
}

HQ_API int hq_kv_pool_seq_len(const hq_kv_pool* p, int seq) { return p && p->has(seq) ? p->seqs[seq].len : -1; }

HQ_API int hq_kv_pool_seq_pages(const hq_kv_pool* p, int seq, int32_t* pages, int max_pages) {
    if (!p || !p->has(seq) || max_pages < 0 || (max_pages > 0 && !pages)) return -1;
    const Seq& s = p->seqs[seq];
    std::copy_n(s.pages.begin(), std::min((size_t)max_pages, s.pages.size()), pages);
    return (int)s.pages.size();
}

HQ_API int hq_kv_pool_tables(const hq_kv_pool* p, const int32_t* seqs, int n, int32_t* page_table, int max_pages,
                             int32_t* kv_lens) {
    if (!p || n < 0 || max_pages < 0 || (n > 0 && !seqs) || (n > 0 && max_pages > 0 && !page_table)) return -1;
    size_t most = 0;
    for (int i = 0; i < n; ++i) {
        if (!p->has(seqs[i])) return -1;
        most = std::max(most, p->seqs[seqs[i]].pages.size());
    }
    for (int i = 0; i < n; ++i) {
        const Seq& s = p->seqs[seqs[i]];
        int32_t* row = page_table + (size_t)i * max_pages;
        const size_t m = std::min((size_t)max_pages, s.pages.size());
        std::copy_n(s.pages.begin(), m, row);
        std::fill(row + m, row + max_pages, 0);
        if (kv_lens) kv_lens[i] = s.len;
    }
    return (int)most;
}

HQ_API hq_status hq_kv_pool_compact(hq_kv_pool* p, hq_page_move* moves, int max_moves, int* n_moves) {
    if (!p || !n_moves || max_moves < 0 || (max_moves > 0 && !moves)) return HQ_ERR_INVALID_ARG;
    try {
        // pages in use at or above in_use go, in order, into the free ones below it
        std::vector<int32_t> to(p->refs.size(), -1);
        int hole = 0, n = 0;
        for (int g = p->in_use; g < (int)p->refs.size(); ++g) {
            if (!p->refs[g]) continue;
            while (p->refs[hole]) ++hole;
            if (n == max_moves) return HQ_ERR_INVALID_ARG;
            moves[n++] = hq_page_move{g, hole};
            to[g] = hole++;
        }
        std::vector<int> rest;
        rest.reserve(p->refs.size());
        for (int g = p->in_use; g < (int)p->refs.size(); ++g) rest.push_back(g);
        for (int i = 0; i < n; ++i) {
            p->refs[moves[i].dst] = p->refs[moves[i].src];
            p->refs[moves[i].src] = 0;
        }
        for (Seq& s : p->seqs)
            for (int32_t& g : s.pages)
                if (to[g] >= 0) g = to[g];
        p->free_pages = decltype(p->free_pages)(std::greater<int>(), std::move(rest));
        *n_moves = n;
        return HQ_OK;
    } catch (const std::bad_alloc&) {
        return HQ_ERR_OUT_OF_MEMORY;
    }
}

}  // extern "C"
