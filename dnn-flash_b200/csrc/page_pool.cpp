// page_pool.cpp -- host-side page pool of the paged key-value cache (include/odf_paged_sm100.h).
//
// Reference counts per page, a free list that hands out the lowest ids first (so a pool that is
// not full stays near compact), and one table per sequence.  Every call either does all of its
// change or none: what can fail (ids, room, memory) is checked or reserved before the first write.
#include <algorithm>
#include <cstdint>
#include <functional>
#include <new>
#include <queue>
#include <unordered_map>
#include <vector>

#include "odf_internal.h"
#include "odf_paged_sm100.h"

namespace {

struct Sequence {
    std::vector<int32_t> pages;
    int64_t tokens = 0;
};

}  // namespace

struct odf_page_pool {
    int64_t page_size = 0;
    std::vector<int32_t> refs;  // per page: how many sequences hold it
    // min-heap of free ids; its storage is reserved for every page, so pushing never allocates
    std::vector<int32_t> free_ids;
    std::unordered_map<int64_t, Sequence> seqs;
    int64_t next_seq = 0;

    int32_t take() {
        std::pop_heap(free_ids.begin(), free_ids.end(), std::greater<int32_t>());
        const int32_t id = free_ids.back();
        free_ids.pop_back();
        refs[id] = 1;
        return id;
    }
    void drop(int32_t id) {
        if (--refs[id] == 0) {
            free_ids.push_back(id);
            std::push_heap(free_ids.begin(), free_ids.end(), std::greater<int32_t>());
        }
    }
};

namespace {

using odf::set_error;

// Nothing throws across the C boundary: allocation failures become ODF_ERR_NO_PAGES.
template <typename F>
int guarded(F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return set_error(ODF_ERR_NO_PAGES, "out of host memory for the page pool");
    } catch (...) {
        return set_error(ODF_ERR_INVALID_ARG, "the page pool failed");
    }
}

Sequence* find(odf_page_pool* pool, int64_t seq) {
    const auto it = pool->seqs.find(seq);
    return it == pool->seqs.end() ? nullptr : &it->second;
}

int no_pool() { return set_error(ODF_ERR_INVALID_ARG, "page pool and output pointers must be non-null"); }
int no_seq() { return set_error(ODF_ERR_INVALID_ARG, "no such sequence in the page pool"); }

}  // namespace

extern "C" {

int odf_page_pool_create(int64_t num_pages, int64_t page_size, odf_page_pool** out) {
    if (out == nullptr) return no_pool();
    *out = nullptr;
    if (num_pages <= 0 || num_pages > 0x7fffffffLL || page_size <= 0 || page_size > 65536)
        return set_error(ODF_ERR_INVALID_ARG, "num_pages must be in [1, 2^31) and page_size in [1, 65536]");
    return guarded([&] {
        odf_page_pool* pool = new odf_page_pool;
        try {
            pool->page_size = page_size;
            pool->refs.assign(static_cast<size_t>(num_pages), 0);
            pool->free_ids.resize(static_cast<size_t>(num_pages));
            for (int64_t i = 0; i < num_pages; ++i) pool->free_ids[i] = static_cast<int32_t>(i);  // sorted: a min-heap
        } catch (...) {
            delete pool;
            throw;
        }
        *out = pool;
        return ODF_OK;
    });
}

void odf_page_pool_destroy(odf_page_pool* pool) { delete pool; }

int odf_page_pool_add(odf_page_pool* pool, int64_t* seq) {
    if (pool == nullptr || seq == nullptr) return no_pool();
    return guarded([&] {
        pool->seqs.emplace(pool->next_seq, Sequence{});
        *seq = pool->next_seq++;
        return ODF_OK;
    });
}

int odf_page_pool_fork(odf_page_pool* pool, int64_t seq, int64_t* child) {
    if (pool == nullptr || child == nullptr) return no_pool();
    Sequence* s = find(pool, seq);
    if (s == nullptr) return no_seq();
    return guarded([&] {
        Sequence copy = *s;
        const auto it = pool->seqs.emplace(pool->next_seq, std::move(copy)).first;
        for (int32_t id : it->second.pages) ++pool->refs[id];
        *child = pool->next_seq++;
        return ODF_OK;
    });
}

int odf_page_pool_extend(odf_page_pool* pool, int64_t seq, int64_t tokens, int32_t pair[2], int64_t* n_pairs) {
    if (pool == nullptr || pair == nullptr || n_pairs == nullptr) return no_pool();
    *n_pairs = 0;
    Sequence* s = find(pool, seq);
    if (s == nullptr) return no_seq();
    if (tokens < 0 || tokens > 0x7fffffffLL - s->tokens)
        return set_error(ODF_ERR_INVALID_ARG, "a sequence grows by 0 tokens or more, to at most 2^31 - 1");
    if (tokens == 0) return ODF_OK;
    const int64_t S = pool->page_size;
    const int64_t have = static_cast<int64_t>(s->pages.size());
    const int64_t need = (s->tokens + tokens + S - 1) / S - have;
    const bool own_last = s->tokens % S != 0 && pool->refs[s->pages.back()] > 1;
    if (need + (own_last ? 1 : 0) > static_cast<int64_t>(pool->free_ids.size()))
        return set_error(ODF_ERR_NO_PAGES, "not enough free pages");
    return guarded([&] {
        s->pages.reserve(static_cast<size_t>(have + need));
        if (own_last) {
            const int32_t old = s->pages.back();
            const int32_t fresh = pool->take();
            pool->drop(old);
            s->pages.back() = fresh;
            pair[0] = old;
            pair[1] = fresh;
            *n_pairs = 1;
        }
        for (int64_t i = 0; i < need; ++i) s->pages.push_back(pool->take());
        s->tokens += tokens;
        return ODF_OK;
    });
}

int odf_page_pool_truncate(odf_page_pool* pool, int64_t seq, int64_t length) {
    if (pool == nullptr) return no_pool();
    Sequence* s = find(pool, seq);
    if (s == nullptr) return no_seq();
    if (length < 0 || length > s->tokens)
        return set_error(ODF_ERR_INVALID_ARG, "a sequence is cut to between 0 and its own length");
    return guarded([&] {
        const size_t keep = static_cast<size_t>((length + pool->page_size - 1) / pool->page_size);
        while (s->pages.size() > keep) {
            pool->drop(s->pages.back());
            s->pages.pop_back();
        }
        s->tokens = length;
        return ODF_OK;
    });
}

int odf_page_pool_free(odf_page_pool* pool, int64_t seq) {
    if (pool == nullptr) return no_pool();
    Sequence* s = find(pool, seq);
    if (s == nullptr) return no_seq();
    return guarded([&] {
        for (int32_t id : s->pages) pool->drop(id);
        pool->seqs.erase(seq);
        return ODF_OK;
    });
}

int odf_page_pool_compact(odf_page_pool* pool, int32_t* pairs, int64_t room, int64_t* n_pairs) {
    if (pool == nullptr || n_pairs == nullptr || (pairs == nullptr && room > 0)) return no_pool();
    *n_pairs = 0;
    const int64_t total = static_cast<int64_t>(pool->refs.size());
    const int64_t used = total - static_cast<int64_t>(pool->free_ids.size());
    return guarded([&] {
        // used pages at or past `used` move into the free ids below it, lowest first
        std::vector<int32_t> move(static_cast<size_t>(total), -1);
        std::vector<int32_t> new_free;
        new_free.reserve(static_cast<size_t>(total));
        int64_t n = 0, hole = 0;
        for (int64_t id = used; id < total; ++id) {
            if (pool->refs[id] == 0) continue;
            while (pool->refs[hole] != 0) ++hole;
            move[id] = static_cast<int32_t>(hole++);
            ++n;
        }
        if (n > room) return set_error(ODF_ERR_INVALID_ARG, "the array of pairs is too small for the compaction");
        for (int64_t id = used; id < total; ++id) new_free.push_back(static_cast<int32_t>(id));  // sorted: a min-heap
        int64_t at = 0;
        for (int64_t id = used; id < total; ++id) {
            if (move[id] < 0) continue;
            pairs[2 * at] = static_cast<int32_t>(id);
            pairs[2 * at + 1] = move[id];
            ++at;
            pool->refs[move[id]] = pool->refs[id];
            pool->refs[id] = 0;
        }
        for (auto& entry : pool->seqs)
            for (int32_t& id : entry.second.pages)
                if (move[id] >= 0) id = move[id];
        pool->free_ids.swap(new_free);
        *n_pairs = n;
        return ODF_OK;
    });
}

int odf_page_pool_length(const odf_page_pool* pool, int64_t seq, int64_t* tokens, int64_t* pages) {
    if (pool == nullptr || tokens == nullptr || pages == nullptr) return no_pool();
    const auto it = pool->seqs.find(seq);
    if (it == pool->seqs.end()) return no_seq();
    *tokens = it->second.tokens;
    *pages = static_cast<int64_t>(it->second.pages.size());
    return ODF_OK;
}

int odf_page_pool_table(const odf_page_pool* pool, int64_t seq, int32_t* out, int64_t max_pages) {
    if (pool == nullptr || (out == nullptr && max_pages > 0)) return no_pool();
    const auto it = pool->seqs.find(seq);
    if (it == pool->seqs.end()) return no_seq();
    const std::vector<int32_t>& pages = it->second.pages;
    if (static_cast<int64_t>(pages.size()) > max_pages)
        return set_error(ODF_ERR_INVALID_ARG, "the sequence has more pages than the table has entries");
    std::copy(pages.begin(), pages.end(), out);
    std::fill(out + pages.size(), out + max_pages, -1);
    return ODF_OK;
}

int64_t odf_page_pool_free_pages(const odf_page_pool* pool) {
    return pool == nullptr ? 0 : static_cast<int64_t>(pool->free_ids.size());
}

}  // extern "C"
