// Page bookkeeping of a paged KV cache on the host (include/g4.h, g4_page_pool_*): who
// holds which page, copy-on-write of shared last pages, and compaction.  No GPU work; the
// copies and moves it asks for run through g4_paged_copy / g4_paged_compact.
#include <cstdint>
#include <exception>
#include <new>
#include <set>
#include <string>
#include <vector>

#include "g4.h"

namespace {

struct Seq {
  bool live = false;
  int rows = 0;
  std::vector<int32_t> pages;  // -1: given back (below the window)
};
struct Copy {
  int32_t src, dst, rows;
};

}  // namespace

struct g4_page_pool {
  int n_pages = 0, page_rows = 0;
  std::vector<int> users;    // sequences holding each page
  std::set<int32_t> free_pages;
  std::vector<Seq> seqs;
  std::vector<Copy> pending;  // copies asked for and not taken yet, in order
  std::string last_error;
};

namespace {

g4_status refuse(g4_page_pool* pool, g4_status code, const std::string& msg) {
  pool->last_error = msg;
  return code;
}
Seq* find(g4_page_pool* pool, int32_t seq) {
  if (seq < 0 || static_cast<size_t>(seq) >= pool->seqs.size() || !pool->seqs[seq].live) return nullptr;
  return &pool->seqs[seq];
}
void drop(g4_page_pool* pool, int32_t page) {
  if (page >= 0 && --pool->users[page] == 0) pool->free_pages.insert(page);
}
int32_t take(g4_page_pool* pool) {
  const int32_t page = *pool->free_pages.begin();
  pool->free_pages.erase(pool->free_pages.begin());
  pool->users[page] = 1;
  return page;
}
int32_t new_seq(g4_page_pool* pool) {
  for (size_t i = 0; i < pool->seqs.size(); ++i)
    if (!pool->seqs[i].live) return static_cast<int32_t>(i);
  pool->seqs.emplace_back();
  return static_cast<int32_t>(pool->seqs.size() - 1);
}
// No C++ exception may leave a C entry point: the only ones here are failed allocations.
template <class F>
g4_status guarded(g4_page_pool* pool, F&& body) {
  if (pool == nullptr) return G4_ERR_BAD_ARG;
  try {
    return body();
  } catch (const std::exception&) {
    return G4_ERR_TOO_LARGE;
  }
}

}  // namespace

extern "C" {

g4_status g4_page_pool_create(int n_pages, int page_rows, g4_page_pool** out) {
  if (out == nullptr) return G4_ERR_BAD_ARG;
  *out = nullptr;
  if (n_pages < 1 || n_pages > (1 << 24) || page_rows < 8 || page_rows > 65536 || page_rows % 8 != 0) return G4_ERR_BAD_ARG;
  g4_page_pool* pool = new (std::nothrow) g4_page_pool();
  const g4_status st = guarded(pool, [&] {
    pool->n_pages = n_pages;
    pool->page_rows = page_rows;
    pool->users.assign(n_pages, 0);
    for (int i = 0; i < n_pages; ++i) pool->free_pages.insert(pool->free_pages.end(), i);
    return G4_OK;
  });
  if (st != G4_OK) {
    delete pool;
    return G4_ERR_TOO_LARGE;
  }
  *out = pool;
  return G4_OK;
}

g4_status g4_page_pool_destroy(g4_page_pool* pool) {
  if (pool == nullptr) return G4_ERR_BAD_ARG;
  delete pool;
  return G4_OK;
}

const char* g4_page_pool_last_error(const g4_page_pool* pool) {
  return pool != nullptr ? pool->last_error.c_str() : "null page pool";
}

g4_status g4_page_pool_add(g4_page_pool* pool, int32_t* out_seq) {
  return guarded(pool, [&] {
    if (out_seq == nullptr) return refuse(pool, G4_ERR_BAD_ARG, "null sequence output");
    const int32_t id = new_seq(pool);
    pool->seqs[id] = Seq();
    pool->seqs[id].live = true;
    *out_seq = id;
    return G4_OK;
  });
}

g4_status g4_page_pool_extend(g4_page_pool* pool, int32_t seq, int n_rows) {
  return guarded(pool, [&] {
    Seq* s = find(pool, seq);
    if (s == nullptr) return refuse(pool, G4_ERR_BAD_ARG, "no such sequence");
    if (n_rows < 0) return refuse(pool, G4_ERR_BAD_ARG, "negative row count");
    const long long rows = static_cast<long long>(s->rows) + n_rows;
    const long long pages = (rows + pool->page_rows - 1) / pool->page_rows;
    if (rows > INT32_MAX || pages > pool->n_pages + static_cast<long long>(s->pages.size()))
      return refuse(pool, G4_ERR_TOO_LARGE, "more rows than the pool has pages for");
    const int used = s->rows % pool->page_rows;  // rows in the partly filled last page
    const bool own = n_rows > 0 && used != 0 && s->pages.back() >= 0 && pool->users[s->pages.back()] > 1;
    const size_t fresh = static_cast<size_t>(pages) - s->pages.size();
    if (fresh + (own ? 1 : 0) > pool->free_pages.size())
      return refuse(pool, G4_ERR_TOO_LARGE, "not enough free pages");
    // every allocation first, so that a failed one leaves the pool as it was
    s->pages.reserve(static_cast<size_t>(pages));
    if (own) pool->pending.reserve(pool->pending.size() + 1);
    if (own) {
      const int32_t shared = s->pages.back(), page = take(pool);
      drop(pool, shared);
      s->pages.back() = page;
      pool->pending.push_back({shared, page, used});
    }
    for (size_t i = 0; i < fresh; ++i) s->pages.push_back(take(pool));
    s->rows = static_cast<int>(rows);
    return G4_OK;
  });
}

g4_status g4_page_pool_fork(g4_page_pool* pool, int32_t seq, int32_t* out_child) {
  return guarded(pool, [&] {
    if (out_child == nullptr) return refuse(pool, G4_ERR_BAD_ARG, "null sequence output");
    if (find(pool, seq) == nullptr) return refuse(pool, G4_ERR_BAD_ARG, "no such sequence");
    Seq child = pool->seqs[seq];
    const int32_t id = new_seq(pool);  // (may move pool->seqs)
    for (const int32_t p : child.pages)
      if (p >= 0) ++pool->users[p];
    pool->seqs[id] = std::move(child);
    *out_child = id;
    return G4_OK;
  });
}

g4_status g4_page_pool_trim(g4_page_pool* pool, int32_t seq, int first_row) {
  return guarded(pool, [&] {
    Seq* s = find(pool, seq);
    if (s == nullptr) return refuse(pool, G4_ERR_BAD_ARG, "no such sequence");
    if (first_row < 0 || first_row > s->rows) return refuse(pool, G4_ERR_BAD_ARG, "row outside the sequence");
    for (int i = 0; i < first_row / pool->page_rows; ++i) {
      drop(pool, s->pages[i]);
      s->pages[i] = -1;
    }
    return G4_OK;
  });
}

g4_status g4_page_pool_free(g4_page_pool* pool, int32_t seq) {
  return guarded(pool, [&] {
    Seq* s = find(pool, seq);
    if (s == nullptr) return refuse(pool, G4_ERR_BAD_ARG, "no such sequence");
    for (const int32_t p : s->pages) drop(pool, p);
    *s = Seq();
    return G4_OK;
  });
}

g4_status g4_page_pool_compact(g4_page_pool* pool, int32_t* src, int32_t* dst, int32_t* page_map, int* out_n) {
  return guarded(pool, [&] {
    if (src == nullptr || dst == nullptr || page_map == nullptr || out_n == nullptr)
      return refuse(pool, G4_ERR_BAD_ARG, "null output");
    if (!pool->pending.empty()) return refuse(pool, G4_ERR_BAD_ARG, "page copies wait to be taken");
    const int used = pool->n_pages - static_cast<int>(pool->free_pages.size());
    std::set<int32_t> now_free;
    for (int p = used; p < pool->n_pages; ++p) now_free.insert(now_free.end(), p);
    for (int p = 0; p < pool->n_pages; ++p) page_map[p] = p;
    // the k-th page in use beyond the front goes to the k-th free page of the front: no page
    // is both left and filled, so the moves may run in any order
    int n = 0;
    auto hole = pool->free_pages.begin();
    for (int p = used; p < pool->n_pages; ++p) {
      if (pool->users[p] == 0) continue;
      src[n] = p;
      dst[n] = *hole++;
      page_map[p] = dst[n];
      ++n;
    }
    for (int i = 0; i < n; ++i) {
      pool->users[dst[i]] = pool->users[src[i]];
      pool->users[src[i]] = 0;
    }
    for (Seq& s : pool->seqs)
      for (int32_t& p : s.pages)
        if (p >= 0) p = page_map[p];
    pool->free_pages.swap(now_free);
    *out_n = n;
    return G4_OK;
  });
}

g4_status g4_page_pool_take_copies(g4_page_pool* pool, int32_t* src, int32_t* dst, int32_t* rows, int cap,
                                   int* out_n) {
  return guarded(pool, [&] {
    if (src == nullptr || dst == nullptr || rows == nullptr || out_n == nullptr || cap < 1)
      return refuse(pool, G4_ERR_BAD_ARG, "null output or no room");
    // a copy joins the group unless it fills a page the group reads or fills, or reads one it fills
    std::set<int32_t> read, filled;
    int n = 0;
    for (const Copy& c : pool->pending) {
      if (n == cap || read.count(c.dst) || filled.count(c.dst) || filled.count(c.src)) break;
      read.insert(c.src);
      filled.insert(c.dst);
      src[n] = c.src;
      dst[n] = c.dst;
      rows[n] = c.rows;
      ++n;
    }
    pool->pending.erase(pool->pending.begin(), pool->pending.begin() + n);
    *out_n = n;
    return G4_OK;
  });
}

g4_status g4_page_pool_table(const g4_page_pool* pool, int32_t seq, int32_t* table, int width, int* out_rows) {
  g4_page_pool* p = const_cast<g4_page_pool*>(pool);
  return guarded(p, [&] {
    const Seq* s = find(p, seq);
    if (s == nullptr) return refuse(p, G4_ERR_BAD_ARG, "no such sequence");
    if (out_rows == nullptr || width < 0 || (width > 0 && table == nullptr))
      return refuse(p, G4_ERR_BAD_ARG, "null output or negative width");
    *out_rows = s->rows;
    if (s->pages.size() > static_cast<size_t>(width)) return refuse(p, G4_ERR_TOO_LARGE, "table wider than its room");
    for (int i = 0; i < width; ++i) table[i] = i < static_cast<int>(s->pages.size()) ? s->pages[i] : -1;
    return G4_OK;
  });
}

g4_status g4_page_pool_free_pages(const g4_page_pool* pool, int* out_n) {
  if (pool == nullptr || out_n == nullptr) return G4_ERR_BAD_ARG;
  *out_n = static_cast<int>(pool->free_pages.size());
  return G4_OK;
}

}  // extern "C"
