// page_pool.cpp -- which sequence has which pages of a key/value cache: growing with copy on write, forking, trimming
// behind a window, closing and compacting.  Host memory only; the copies that a step asks for are made by
// aig_kv_copy_pages.  (Not in the reference.)
#include <limits.h>

#include <new>
#include <vector>

#include "aig_b200.h"

namespace {
struct Sequence {
  bool open = false;
  int length = 0;
  std::vector<int32_t> pages;  // -1: given up by trim
};
}  // namespace

struct aig_page_pool {
  int page_size = 0;
  std::vector<int> users;         // sequences that have the page
  std::vector<int32_t> free;      // taken from the back
  std::vector<Sequence> seqs;
};

namespace {

const Sequence* find(const aig_page_pool* p, int seq) {
  return p && seq >= 0 && seq < (int)p->seqs.size() && p->seqs[seq].open ? &p->seqs[seq] : nullptr;
}
Sequence* find(aig_page_pool* p, int seq) { return const_cast<Sequence*>(find(static_cast<const aig_page_pool*>(p), seq)); }

// A number for a new sequence; may throw before anything changes.
int slot_for(aig_page_pool* p) {
  for (size_t i = 0; i < p->seqs.size(); ++i)
    if (!p->seqs[i].open) return (int)i;
  p->seqs.emplace_back();
  return (int)p->seqs.size() - 1;
}

// (the list of free pages has room for all of them from the start)
void give_up(aig_page_pool* p, int32_t page) {
  if (page >= 0 && --p->users[page] == 0) p->free.push_back(page);
}

int32_t take(aig_page_pool* p) {
  const int32_t page = p->free.back();
  p->free.pop_back();
  p->users[page] = 1;
  return page;
}

}  // namespace

extern "C" {

int aig_page_pool_create(int num_pages, int page_size, aig_page_pool** out) {
  if (!out) return AIG_ERR_INVALID;
  *out = nullptr;
  if (num_pages <= 0 || page_size <= 0) return AIG_ERR_INVALID;
  aig_page_pool* p = nullptr;
  try {
    p = new aig_page_pool();
    p->page_size = page_size;
    p->users.assign(num_pages, 0);
    p->free.resize(num_pages);
    for (int i = 0; i < num_pages; ++i) p->free[i] = num_pages - 1 - i;
  } catch (const std::bad_alloc&) {
    delete p;
    return AIG_ERR_INVALID;
  }
  *out = p;
  return AIG_OK;
}

int aig_page_pool_destroy(aig_page_pool* p) {
  delete p;
  return AIG_OK;
}

int aig_page_pool_open(aig_page_pool* p, int* seq) {
  if (!p || !seq) return AIG_ERR_INVALID;
  try {
    const int s = slot_for(p);
    p->seqs[s].open = true;
    p->seqs[s].length = 0;
    p->seqs[s].pages.clear();
    *seq = s;
    return AIG_OK;
  } catch (const std::bad_alloc&) {
    return AIG_ERR_INVALID;
  }
}

int aig_page_pool_grow(aig_page_pool* p, int seq, int tokens, int32_t* copy_src, int32_t* copy_dst) {
  Sequence* s = find(p, seq);
  if (!s || tokens < 0 || !copy_src || !copy_dst || tokens > INT_MAX - p->page_size - s->length) return AIG_ERR_INVALID;
  *copy_src = *copy_dst = -1;
  if (tokens == 0) return AIG_OK;
  const size_t had = s->pages.size(), need = ((size_t)s->length + tokens + p->page_size - 1) / p->page_size;
  const bool own_copy = s->length % p->page_size != 0 && p->users[s->pages.back()] > 1;
  if (need - had + (own_copy ? 1 : 0) > p->free.size()) return AIG_ERR_NO_PAGES;
  try {
    s->pages.reserve(need);
  } catch (const std::bad_alloc&) {
    return AIG_ERR_INVALID;
  }
  if (own_copy) {
    *copy_src = s->pages.back();
    *copy_dst = take(p);
    --p->users[*copy_src];
    s->pages.back() = *copy_dst;
  }
  for (size_t i = had; i < need; ++i) s->pages.push_back(take(p));
  s->length += tokens;
  return AIG_OK;
}

int aig_page_pool_fork(aig_page_pool* p, int seq, int* new_seq) {
  if (!find(p, seq) || !new_seq) return AIG_ERR_INVALID;
  try {
    const int n = slot_for(p);  // (may move the sequences)
    p->seqs[n].pages = p->seqs[seq].pages;
    p->seqs[n].length = p->seqs[seq].length;
    p->seqs[n].open = true;
    for (int32_t page : p->seqs[n].pages)
      if (page >= 0) ++p->users[page];
    *new_seq = n;
    return AIG_OK;
  } catch (const std::bad_alloc&) {
    return AIG_ERR_INVALID;
  }
}

int aig_page_pool_trim(aig_page_pool* p, int seq, int window, int sinks) {
  Sequence* s = find(p, seq);
  if (!s || sinks < 0) return AIG_ERR_INVALID;
  if (window <= 0) return AIG_OK;  // everything stays visible
  const long long size = p->page_size, from = (sinks + size - 1) / size, to = ((long long)s->length - window) / size;
  for (long long i = from; i < to; ++i) {
    give_up(p, s->pages[i]);
    s->pages[i] = -1;
  }
  return AIG_OK;
}

int aig_page_pool_close(aig_page_pool* p, int seq) {
  Sequence* s = find(p, seq);
  if (!s) return AIG_ERR_INVALID;
  for (int32_t page : s->pages) give_up(p, page);
  s->pages.clear();
  s->length = 0;
  s->open = false;
  return AIG_OK;
}

int aig_page_pool_compact(aig_page_pool* p, int32_t* copy_src, int32_t* copy_dst, int capacity, int* pairs) {
  if (!p || !pairs || capacity < 0 || (capacity > 0 && (!copy_src || !copy_dst))) return AIG_ERR_INVALID;
  *pairs = 0;
  try {
    const int n = (int)p->users.size();
    std::vector<int32_t> now(n);
    for (int i = 0; i < n; ++i) now[i] = i;
    // the lowest free page takes the highest used one; the two meet, so no source is a destination
    int low = 0, high = n - 1, moved = 0;
    while (moved < capacity) {
      while (low < high && p->users[low] > 0) ++low;
      while (low < high && p->users[high] == 0) --high;
      if (low >= high) break;
      copy_src[moved] = high;
      copy_dst[moved++] = low;
      now[high] = low;
      p->users[low] = p->users[high];
      p->users[high] = 0;
    }
    for (Sequence& s : p->seqs)
      for (int32_t& page : s.pages)
        if (page >= 0) page = now[page];
    p->free.clear();
    for (int i = n - 1; i >= 0; --i)
      if (p->users[i] == 0) p->free.push_back(i);
    *pairs = moved;
    return AIG_OK;
  } catch (const std::bad_alloc&) {
    return AIG_ERR_INVALID;
  }
}

int aig_page_pool_table(const aig_page_pool* p, int seq, int32_t* out, int width) {
  const Sequence* s = find(p, seq);
  if (!s || width < 0 || (width > 0 && !out)) return AIG_ERR_INVALID;
  for (int i = 0; i < width; ++i) out[i] = i < (int)s->pages.size() ? s->pages[i] : -1;
  return (int)s->pages.size();
}

int aig_page_pool_length(const aig_page_pool* p, int seq) {
  const Sequence* s = find(p, seq);
  return s ? s->length : AIG_ERR_INVALID;
}

int aig_page_pool_free_pages(const aig_page_pool* p) { return p ? (int)p->free.size() : AIG_ERR_INVALID; }

int aig_page_pool_shared(const aig_page_pool* p, int page) {
  return p && page >= 0 && page < (int)p->users.size() ? p->users[page] : AIG_ERR_INVALID;
}

}  // extern "C"
