// Host (CPU) implementation of the pages of a paged cache.  It serves CPU ranks and defines the
// results that csrc/hip/pages.hip gives bit for bit (tests compare both).
#include "pages.h"

#include <string.h>

#include <algorithm>
#include <vector>

namespace tpi {

namespace {

void refuse(const tpi_pages& p, int code) {
  if (!p.header[TPI_PAGES_ERROR]) p.header[TPI_PAGES_ERROR] = code;
}

int64_t pages_of(const tpi_pages& p, int64_t tokens) { return (tokens + p.tokens - 1) / p.tokens; }

bool get(const uint32_t* bits, int64_t page) { return bits[page >> 5] >> (page & 31) & 1; }
void set(uint32_t* bits, int64_t page) { bits[page >> 5] |= 1u << (page & 31); }
void reset(uint32_t* bits, int64_t page) { bits[page >> 5] &= ~(1u << (page & 31)); }

bool slot_ok(const tpi_pages& p, int64_t s) { return s >= 0 && s < p.slots; }
bool page_ok(const tpi_pages& p, int64_t s) { return s >= 0 && s < p.pages; }

// Page `src` copied to page `dst` in every tensor, or `dst` cleared (src < 0).
void move_page(const tpi_pages& p, int64_t src, int64_t dst) {
  for (int c = 0; c < p.chunks; ++c) {
    const tpi_page_chunk& x = p.chunk[c];
    for (uint32_t r = 0; r < x.rows; ++r) {
      uint8_t* row = (uint8_t*)x.base + (int64_t)r * x.row_stride;
      if (src < 0) memset(row + dst * x.page_stride, 0, x.row_bytes);
      else memcpy(row + dst * x.page_stride, row + src * x.page_stride, x.row_bytes);
    }
  }
}

// The `total` lowest free pages, taken; empty (ESTATE) when the bits hold fewer.
std::vector<int32_t> take(const tpi_pages& p, int64_t total) {
  std::vector<int32_t> out;
  for (int64_t page = 0; page < p.pages && (int64_t)out.size() < total; ++page)
    if (get(p.free_bits, page)) {
      reset(p.free_bits, page);
      out.push_back((int32_t)page);
    }
  if ((int64_t)out.size() < total) {
    refuse(p, TPI_PAGES_ESTATE);
    out.clear();
  }
  return out;
}

// The largest code of any entry, as the kernel finds it.
struct Check {
  int error = 0;
  void at(int code) { error = std::max(error, code); }
};

}  // namespace

void pages_copy(const tpi_pages& p, const int64_t* src, const int64_t* dst, int64_t n) {
  for (int64_t i = 0; i < n; ++i) {
    if (!page_ok(p, src[i]) || !page_ok(p, dst[i])) {
      refuse(p, TPI_PAGES_EPAGE);
    } else if (src[i] != dst[i]) {
      move_page(p, src[i], dst[i]);
      if (get(p.free_bits, dst[i])) set(p.stale_bits, dst[i]);  // not known to be zero any more
    }
  }
}

void pages_fork(const tpi_pages& p, const int64_t* src, const int64_t* dst, int64_t n) {
  Check check;
  int64_t total = 0;
  std::vector<uint8_t> seen(p.slots, 0);
  for (int64_t i = 0; i < n; ++i) {
    if (!slot_ok(p, src[i]) || !slot_ok(p, dst[i])) {
      check.at(TPI_PAGES_ESLOT);
      continue;
    }
    if (src[i] == dst[i] || p.lengths[dst[i]] != 0) {
      check.at(TPI_PAGES_EBUSY);
      continue;
    }
    total += p.lengths[src[i]] % p.tokens != 0;
  }
  if (!check.error)
    for (int64_t i = 0; i < n; ++i) {
      if (seen[dst[i]]) check.at(TPI_PAGES_EDUPLICATE);
      seen[dst[i]] = 1;
    }
  if (total > p.header[TPI_PAGES_FREE]) check.at(TPI_PAGES_ENOSPACE);
  if (check.error) return refuse(p, check.error);
  const std::vector<int32_t> taken = take(p, total);
  if ((int64_t)taken.size() < total) return;
  std::vector<int32_t> length(n);
  for (int64_t i = 0; i < n; ++i) length[i] = p.lengths[src[i]];
  int64_t at = 0;
  for (int64_t i = 0; i < n; ++i) {
    const int32_t* from = p.table + src[i] * p.width;
    int32_t* to = p.table + dst[i] * p.width;
    const int64_t full = length[i] / p.tokens;
    for (int64_t k = 0; k < full; ++k) {
      to[k] = from[k];
      if (page_ok(p, to[k])) ++p.refs[to[k]];
    }
    if (length[i] % p.tokens) {
      to[full] = taken[at++];
      p.refs[to[full]] = 1;
      if (page_ok(p, from[full])) move_page(p, from[full], to[full]);
    }
    p.lengths[dst[i]] = length[i];
  }
  p.header[TPI_PAGES_FREE] -= (int32_t)total;
}

void pages_extend(const tpi_pages& p, const int64_t* slots, const int64_t* more, int64_t n) {
  Check check;
  int64_t total = 0;
  std::vector<uint8_t> seen(p.slots, 0);
  for (int64_t i = 0; i < n; ++i) {
    if (!slot_ok(p, slots[i])) {
      check.at(TPI_PAGES_ESLOT);
      continue;
    }
    const int64_t old = p.lengths[slots[i]];
    if (more[i] < 0) check.at(TPI_PAGES_ETOKENS);
    else if (more[i] > (int64_t)p.width * p.tokens - old || old + more[i] > 0x7fffffff)
      check.at(TPI_PAGES_EWIDTH);
    else total += pages_of(p, old + more[i]) - pages_of(p, old);
  }
  if (!check.error)
    for (int64_t i = 0; i < n; ++i) {
      if (seen[slots[i]]) check.at(TPI_PAGES_EDUPLICATE);
      seen[slots[i]] = 1;
    }
  if (total > p.header[TPI_PAGES_FREE]) check.at(TPI_PAGES_ENOSPACE);
  if (check.error) return refuse(p, check.error);
  const std::vector<int32_t> taken = take(p, total);
  if ((int64_t)taken.size() < total) return;
  int64_t at = 0;
  for (int64_t i = 0; i < n; ++i) {
    int32_t& length = p.lengths[slots[i]];
    const int64_t old = pages_of(p, length), now = pages_of(p, length + more[i]);
    for (int64_t k = old; k < now; ++k) {
      p.table[slots[i] * p.width + k] = taken[at];
      p.refs[taken[at++]] = 1;
    }
    length += (int32_t)more[i];
  }
  p.header[TPI_PAGES_FREE] -= (int32_t)total;
}

void pages_free(const tpi_pages& p, const int64_t* slots, int64_t n) {
  for (int64_t i = 0; i < n; ++i)
    if (!slot_ok(p, slots[i])) return refuse(p, TPI_PAGES_ESLOT);
  for (int64_t i = 0; i < n; ++i) {
    int32_t* row = p.table + slots[i] * p.width;
    const int64_t held = std::min<int64_t>(pages_of(p, p.lengths[slots[i]]), p.width);
    p.lengths[slots[i]] = 0;
    for (int64_t k = 0; k < held; ++k) {
      const int32_t page = row[k];
      row[k] = -1;
      if (!page_ok(p, page) || --p.refs[page] != 0) continue;
      set(p.free_bits, page);
      set(p.stale_bits, page);
      ++p.header[TPI_PAGES_FREE];
    }
  }
}

void pages_compact(const tpi_pages& p, bool clear) {
  const int64_t live = p.pages - p.header[TPI_PAGES_FREE];
  std::vector<int32_t> map(p.pages, -1);
  int64_t hole = 0, moves = 0, clears = 0;
  for (int64_t page = live; page < p.pages; ++page) {
    if (get(p.free_bits, page)) continue;
    while (hole < live && !get(p.free_bits, hole)) ++hole;
    if (hole == live) break;  // the count and the bits disagree
    move_page(p, page, hole);
    p.refs[hole] = p.refs[page];
    p.refs[page] = 0;
    map[page] = (int32_t)hole++;
    ++moves;
  }
  for (int64_t e = 0; e < (int64_t)p.slots * p.width; ++e)
    if (p.table[e] >= live && p.table[e] < p.pages) p.table[e] = map[p.table[e]];
  for (int64_t page = 0; page < p.pages; ++page) {
    if (page < live) {
      reset(p.free_bits, page);
      reset(p.stale_bits, page);
      continue;
    }
    const bool stale = get(p.stale_bits, page) || !get(p.free_bits, page);
    set(p.free_bits, page);
    if (stale && clear) {
      move_page(p, -1, page);
      ++clears;
    }
    if (stale && !clear) set(p.stale_bits, page);
    else reset(p.stale_bits, page);
  }
  p.header[TPI_PAGES_LIVE] = (int32_t)live;
  p.header[TPI_PAGES_MOVES] = (int32_t)moves;
  p.header[TPI_PAGES_CLEARS] = (int32_t)clears;
}

}  // namespace tpi
