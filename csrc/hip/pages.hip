// Pages of a paged cache: copying, forking, freeing and compacting (ops/paging.py).
//
// A pool is a set of tensors whose first dimension is the page (keys and values of every layer)
// and int32 bookkeeping on the device: table[slot][k] = page of tokens [k P, (k + 1) P) of the
// slot's sequence, refs[page] = table entries that name it, and a bit per page that has none.
// Nothing here waits for the host: numbers of pages to move are read on the device, so a step
// that forks and frees can be captured into a graph.
//
// Order: free pages are taken lowest number first, slots in the order they are asked for, and
// reference counts and bits are changed by integer atomics only, so that every result is the same
// on every run -- and on the host implementation (csrc/native/pages.cpp).
//
//  k_reserve      one workgroup: checks a fork or an extension as a whole, then takes its pages
//                 from the free bits (1024 words at a time: popcount, prefix sum);
//                 k_reserve_few the same in registers
//  k_fork         table rows of the forks, and their partial pages' bytes
//  k_free         a workgroup per slot; k_free_check before it for many
//  k_plan         one workgroup: holes and movers of a compaction, and the pages to clear
//  k_compact      table entries, moved pages' bytes
//  k_clear        free pages' bytes
//  k_copy         pages named by the caller
//
// What bounds them: moved bytes at the rate of a large copy (5 TB/s), cleared ones at 5.8; the plans
// by dependent loads and barriers: 5.4 to 5.7 us for 128 forks or 192 extensions, 5.2 for a compaction
// of 4096 pages and 8.4 of 8192 that clears, 409 of a million (one workgroup, 32768 pages a pass).
#include <hip/hip_runtime.h>

#include "internal.h"
#include "tpi_hip.h"

namespace {

constexpr int kBlock = 256;   // threads that move bytes
constexpr int kPlan = 1024;   // threads of the one-workgroup kernels
constexpr int kSpread = 256 * 32;  // workgroups that take pages of an unknown number
constexpr int kRowSpan = 1024;  // table entries of a row that one workgroup of k_fork takes

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// scratch: [pages] x 4, [slots] x 5
__device__ static inline int32_t* list(const tpi_pages& p, int i) {
  return p.scratch + (int64_t)i * p.pages;
}
__device__ static inline int32_t* slot_list(const tpi_pages& p, int i) {
  return p.scratch + 4 * (int64_t)p.pages + (int64_t)i * p.slots;
}
enum { TAKEN = 0, HOLES = 0, MOVERS = 1, CLEARS = 2, MAP = 3 };            // list()
enum { MARK = 0, OFFSET = 1, LENGTH = 2, PAIR_SRC = 3, PAIR_DST = 4 };     // slot_list()

__device__ static inline int64_t number(const void* a, int64_t i, bool wide) {
  return wide ? ((const int64_t*)a)[i] : ((const int32_t*)a)[i];
}

__device__ static inline void refuse(const tpi_pages& p, int code) {
  atomicCAS(&p.header[TPI_PAGES_ERROR], 0, code);
}

__device__ static inline int32_t pages_of(int64_t tokens, int32_t per) {
  return (int32_t)((tokens + per - 1) / per);
}

// ---- moving bytes ------------------------------------------------------------------------------

// A unit is one 16-byte access of any alignment (the GPU's need none).  A run whose bytes are no
// multiple of 16 ends with a unit that begins 16 bytes before its end, so two units write the
// same bytes there; one of less than 16 bytes moves byte by byte.
typedef u32x4 u32x4_any __attribute__((aligned(1)));

struct Unit {
  int64_t at;      // byte offset from the chunk's base
  uint32_t bytes;  // 16, less in a short run, 0: behind the chunk's end
};

__device__ static inline Unit unit_of(const tpi_page_chunk& c, uint32_t u) {
  uint32_t row = 0, col = u;
  if (c.rows > 1) {
    row = u / c.row_units;
    col = u - row * c.row_units;
  }
  if (row >= c.rows || col >= c.row_units) return Unit{0, 0};
  const int64_t base = (int64_t)row * c.row_stride;
  if (c.row_bytes < 16) return Unit{base, c.row_bytes};
  const uint32_t at = col * 16, last = c.row_bytes - 16;
  return Unit{base + (at < last ? at : last), 16};
}

constexpr int kUnits = TPI_PAGE_UNITS / kBlock;  // of a thread

// All of a thread's loads first, then its stores: 16 KB of a workgroup in flight.  Measured with
// 1024 pages of 32 KB in 16 tensors: 214 us (5.0 TB/s, what a large copy reaches), 290 with half
// of it and a lookup of the tensor before the first load.  Nontemporal stores leave the caches to
// the pages that are read: 256 MB of 16 KB pages 36 us instead of 39.
__device__ static inline void copy_chunk(const tpi_page_chunk& c, int64_t src, int64_t dst) {
  const uint8_t* s = (const uint8_t*)c.base + src * c.page_stride;
  uint8_t* d = (uint8_t*)c.base + dst * c.page_stride;
  Unit unit[kUnits];
  u32x4 v[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    unit[k] = unit_of(c, k * kBlock + threadIdx.x);
    if (unit[k].bytes == 16) v[k] = *(const u32x4_any*)(s + unit[k].at);
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    if (unit[k].bytes == 16) {
      __builtin_nontemporal_store(v[k], (u32x4_any*)(d + unit[k].at));
    } else {
      for (uint32_t b = 0; b < unit[k].bytes; ++b) d[unit[k].at + b] = s[unit[k].at + b];
    }
  }
}

__device__ static inline void zero_chunk(const tpi_page_chunk& c, int64_t page) {
  uint8_t* d = (uint8_t*)c.base + page * c.page_stride;
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const Unit unit = unit_of(c, k * kBlock + threadIdx.x);
    if (unit.bytes == 16) {
      *(u32x4_any*)(d + unit.at) = u32x4{0, 0, 0, 0};
    } else {
      for (uint32_t b = 0; b < unit.bytes; ++b) d[unit.at + b] = 0;
    }
  }
}

// Workgroups (chunk, pair): nothing to look up or divide before the first load.  A free page that is
// written is not known to be zero any more.
__global__ __launch_bounds__(kBlock) void k_copy(tpi_pages p, const void* src, const void* dst,
                                                 int64_t n, bool wide) {
  for (int64_t i = blockIdx.y; i < n; i += gridDim.y) {
    const int64_t s = number(src, i, wide), d = number(dst, i, wide);
    if (s < 0 || s >= p.pages || d < 0 || d >= p.pages) {
      if (threadIdx.x == 0) refuse(p, TPI_PAGES_EPAGE);
      continue;
    }
    // looked at before the bytes move, by the wave that has least to move: 777 pages of 2886 bytes
    // in 6 tensors took 14.5 us with a look behind them
    const uint32_t bit = 1u << (d & 31);
    uint32_t fresh = 0;
    if (blockIdx.x == 0 && threadIdx.x == kBlock - 1 && s != d)
      fresh = p.free_bits[d >> 5] & ~p.stale_bits[d >> 5] & bit;
    copy_chunk(p.chunk[blockIdx.x], s, d);
    if (fresh) atomicOr(&p.stale_bits[d >> 5], bit);
  }
}

// ---- one-workgroup helpers ---------------------------------------------------------------------

// Exclusive prefix sum over the kPlan threads of the workgroup; `total` = the sum.
__device__ static inline int scan(int v, int* total) {
  __shared__ int waves[kPlan / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the last scan's sums have been read
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kPlan / 64; ++w) {
    if (w < wave) before += waves[w];
    sum += waves[w];
  }
  *total = sum;
  return before + x - v;
}

// A pass of the workgroup over kPlan words of bits: thread t has `bits` of word base + t, whose
// first set bit has rank `rank`.  Writes the numbers of the set bits with ranks below `limit` to
// out[rank].  A thread per bit, 32 words apart (one per word would store up to 32 numbers one
// after the other: 10 us of a compaction's plan instead of 6).
struct Words {
  uint32_t bits[kPlan];
  int rank[kPlan];
};

__device__ static inline void emit(Words& lds, uint32_t bits, int rank, int base, int words,
                                   int limit, int32_t* out) {
  __syncthreads();  // the last pass has been read
  lds.bits[threadIdx.x] = bits;
  lds.rank[threadIdx.x] = rank;
  __syncthreads();
  const int n = 32 * (words - base < kPlan ? words - base : kPlan);
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const uint32_t w = lds.bits[i >> 5], bit = 1u << (i & 31);
    if (!(w & bit)) continue;
    const int r = lds.rank[i >> 5] + __popc(w & (bit - 1));
    if (r < limit) out[r] = 32 * base + i;
  }
}

// `bits` without its lowest n set ones.
__device__ static inline uint32_t without_lowest(uint32_t bits, int n) {
  for (; n > 0 && bits; --n) bits &= bits - 1;
  return bits;
}

// Pages of slot entry i that a fork / an extension takes.
template <bool FORK>
__device__ static inline int32_t needed(const tpi_pages& p, const void* a, int64_t i, bool wide) {
  const int32_t len = slot_list(p, LENGTH)[i];
  if (FORK) return len % p.tokens != 0;
  return pages_of(len, p.tokens) - pages_of(p.lengths[number(a, i, wide)], p.tokens);
}

template <bool FORK>
__global__ __launch_bounds__(kPlan) void k_reserve(tpi_pages p, const void* a, const void* b,
                                                   int n, bool wide, const void* more,
                                                   bool more_wide, int64_t each) {
  __shared__ int s_error;
  __shared__ unsigned long long s_total;
  __shared__ Words lds;
  const int tid = threadIdx.x;
  int32_t* mark = slot_list(p, MARK);
  int32_t* offset = slot_list(p, OFFSET);
  int32_t* length = slot_list(p, LENGTH);
  if (tid == 0) {
    s_error = 0;
    s_total = 0;
  }
  __syncthreads();
  // 1. every entry by itself, and what all of them take
  for (int i = tid; i < n; i += kPlan) {
    const int64_t s = number(a, i, wide), d = FORK ? number(b, i, wide) : s;
    int error = 0;
    int64_t len = 0;
    if (s < 0 || s >= p.slots || d < 0 || d >= p.slots) {
      error = TPI_PAGES_ESLOT;
    } else {
      const int64_t old = p.lengths[s];
      if (FORK) {
        len = old;
        if (s == d || p.lengths[d] != 0) error = TPI_PAGES_EBUSY;
      } else {
        const int64_t m = more ? number(more, i, more_wide) : each;
        if (m < 0) {
          error = TPI_PAGES_ETOKENS;
        } else if (m > (int64_t)p.width * p.tokens - old || old + m > 0x7fffffff) {
          error = TPI_PAGES_EWIDTH;
        } else {
          len = old + m;
        }
      }
      mark[d] = i;  // of entries that name one slot, one stays
    }
    if (error) {
      atomicMax(&s_error, error);
      continue;
    }
    length[i] = (int32_t)len;
    const int32_t need = FORK ? len % p.tokens != 0
                              : pages_of(len, p.tokens) - pages_of(p.lengths[s], p.tokens);
    if (need) atomicAdd(&s_total, (unsigned long long)need);
  }
  __syncthreads();
  const bool sound = !s_error;
  __syncthreads();  // every wave has read it before the first reason below is written
  if (sound)
    for (int i = tid; i < n; i += kPlan)
      if (mark[FORK ? number(b, i, wide) : number(a, i, wide)] != i)
        atomicMax(&s_error, TPI_PAGES_EDUPLICATE);
  if (tid == 0 && s_total > (unsigned long long)p.header[TPI_PAGES_FREE])
    atomicMax(&s_error, TPI_PAGES_ENOSPACE);
  __syncthreads();
  if (s_error) {
    if (tid == 0) refuse(p, s_error);
    if (FORK)
      for (int i = tid; i < n; i += kPlan) length[i] = -1;  // nothing for k_fork
    return;
  }
  const int total = (int)s_total;
  // 2. where each entry's pages begin among those taken
  for (int base = 0, carry = 0; base < n; base += kPlan) {
    int sum;
    const int i = base + tid;
    const int before = scan(i < n ? needed<FORK>(p, a, i, wide) : 0, &sum);
    if (i < n) offset[i] = carry + before;
    carry += sum;
  }
  // 3. the lowest free pages
  const int words = (p.pages + 31) / 32;
  int found = 0;
  for (int base = 0; base < words && found < total; base += kPlan) {
    int sum;
    const int w = base + tid;
    const uint32_t bits = w < words ? p.free_bits[w] : 0;
    const int rank = found + scan(__popc(bits), &sum);
    if (bits && rank < total) p.free_bits[w] = without_lowest(bits, total - rank);
    emit(lds, bits, rank, base, words, total, list(p, TAKEN));
    found += sum;
  }
  __syncthreads();
  if (found < total) {  // the count and the bits disagree: not a state that these kernels leave
    if (tid == 0) refuse(p, TPI_PAGES_ESTATE);
    if (FORK)
      for (int i = tid; i < n; i += kPlan) length[i] = -1;
    return;
  }
  // 4. to the entries
  const int32_t* taken = list(p, TAKEN);
  if (FORK) {
    for (int i = tid; i < n; i += kPlan) {
      const int64_t s = number(a, i, wide);
      int32_t from = -1, to = -1;
      if (length[i] % p.tokens) {
        from = p.table[s * p.width + length[i] / p.tokens];
        to = taken[offset[i]];
        p.refs[to] = 1;
      }
      slot_list(p, PAIR_SRC)[i] = from;
      slot_list(p, PAIR_DST)[i] = to;
    }
  } else {
    for (int r = tid; r < total; r += kPlan) {
      int lo = 0, hi = n - 1;  // the last entry that begins at or before r
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (offset[mid] <= r) lo = mid; else hi = mid - 1;
      }
      const int64_t s = number(a, lo, wide);
      p.table[s * p.width + pages_of(p.lengths[s], p.tokens) + (r - offset[lo])] = taken[r];
      p.refs[taken[r]] = 1;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kPlan) p.lengths[number(a, i, wide)] = length[i];
  }
  if (tid == 0) p.header[TPI_PAGES_FREE] -= total;
}

// k_reserve for few entries in a pool of ordinary size: an entry stays in its thread's registers,
// slots named twice are found in a bitmap in LDS, and the pages taken stay there too, so that three
// loads follow one another instead of nine: 128 forks 5.7 us instead of 7.3, 192 extensions 5.4
// instead of 8.1.  The limits: a thread per entry, 8 KB of bitmap, sums of pages below 2^31.
constexpr int kFewSlots = 1 << 16, kFewPages = 1 << 20, kFewTaken = 4096;

template <bool FORK>
__global__ __launch_bounds__(kPlan) void k_reserve_few(tpi_pages p, const void* a, const void* b,
                                                       int n, bool wide, const void* more,
                                                       bool more_wide, int64_t each) {
  __shared__ Words lds;
  __shared__ uint32_t s_seen[kFewSlots / 32];
  __shared__ int32_t s_taken[kFewTaken], s_offset[kPlan];
  __shared__ int64_t s_row[kPlan];
  __shared__ int s_error, s_twice, s_most;
  const int tid = threadIdx.x, words = (p.pages + 31) / 32;
  const int64_t s = tid < n ? number(a, tid, wide) : 0;
  const int64_t d = FORK && tid < n ? number(b, tid, wide) : s;
  uint32_t bits = tid < words ? p.free_bits[tid] : 0;
  const int free = p.header[TPI_PAGES_FREE];
  for (int i = tid; i < (p.slots + 31) / 32; i += kPlan) s_seen[i] = 0;
  if (tid == 0) s_error = s_twice = s_most = 0;
  const bool mine = tid < n && s >= 0 && s < p.slots && d >= 0 && d < p.slots;
  int error = tid < n && !mine ? TPI_PAGES_ESLOT : 0;
  const int32_t old = mine ? p.lengths[s] : 0;
  int64_t len = old;
  if (mine && FORK) {
    if (s == d || p.lengths[d] != 0) error = TPI_PAGES_EBUSY;
  } else if (mine) {
    const int64_t m = more ? number(more, tid, more_wide) : each;
    if (m < 0) error = TPI_PAGES_ETOKENS;
    else if (m > (int64_t)p.width * p.tokens - old || old + m > 0x7fffffff)
      error = TPI_PAGES_EWIDTH;
    else len = old + m;
  }
  const int32_t had = pages_of(old, p.tokens);
  int need = !mine || error ? 0 : FORK ? old % p.tokens != 0 : pages_of(len, p.tokens) - had;
  const bool full = need > free;  // and their sum stays below 2^31 without such
  if (full) need = 0;
  int32_t from = -1;
  if (FORK && need) from = p.table[s * p.width + old / p.tokens];
  __syncthreads();
  if (mine && (atomicOr(&s_seen[d >> 5], 1u << (d & 31)) >> (d & 31) & 1)) s_twice = 1;
  if (error) atomicMax(&s_error, error);
  if (need > 1) atomicMax(&s_most, need);
  int total;
  const int offset = scan(need, &total);  // (its barriers order the shared words, too)
  if (full) atomicMax(&s_error, TPI_PAGES_ENOSPACE);
  __syncthreads();
  const int why = s_error > TPI_PAGES_ENOSPACE ? s_error : s_twice ? TPI_PAGES_EDUPLICATE
                  : s_error || total > free ? TPI_PAGES_ENOSPACE : 0;
  if (why) {
    if (tid == 0) refuse(p, why);
    if (FORK && tid < n) slot_list(p, LENGTH)[tid] = -1;  // nothing for k_fork
    return;
  }
  const bool near = total <= kFewTaken;
  int found = 0;
  for (int base = 0; base < words && found < total; base += kPlan) {
    int sum;
    const int w = base + tid;
    if (base) bits = w < words ? p.free_bits[w] : 0;
    const int rank = found + scan(__popc(bits), &sum);
    if (bits && rank < total) p.free_bits[w] = without_lowest(bits, total - rank);
    if (near) emit(lds, bits, rank, base, words, total, s_taken);
    else emit(lds, bits, rank, base, words, total, list(p, TAKEN));
    found += sum;
  }
  if (!FORK) {
    s_offset[tid] = tid < n ? offset : total;
    s_row[tid] = s * p.width + had;
  }
  __syncthreads();
  if (found < total) {
    if (tid == 0) refuse(p, TPI_PAGES_ESTATE);
    if (FORK && tid < n) slot_list(p, LENGTH)[tid] = -1;
    return;
  }
  const int32_t* far = list(p, TAKEN);
  if (FORK) {
    if (tid < n) {
      const int32_t to = need ? near ? s_taken[offset] : far[offset] : -1;
      slot_list(p, LENGTH)[tid] = old;
      slot_list(p, PAIR_SRC)[tid] = from;
      slot_list(p, PAIR_DST)[tid] = to;
      if (need) p.refs[to] = 1;
    }
  } else {
    if (s_most <= 1) {
      if (need) {
        const int32_t page = near ? s_taken[offset] : far[offset];
        p.table[s * p.width + had] = page;
        p.refs[page] = 1;
      }
    } else {
      for (int r = tid; r < total; r += kPlan) {
        int lo = 0, hi = n - 1;  // the last entry that begins at or before r
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (s_offset[mid] <= r) lo = mid; else hi = mid - 1;
        }
        const int32_t page = near ? s_taken[r] : far[r];
        p.table[s_row[lo] + (r - s_offset[lo])] = page;
        p.refs[page] = 1;
      }
    }
    if (tid < n) p.lengths[s] = (int32_t)len;
  }
  if (tid == 0) p.header[TPI_PAGES_FREE] = free - total;
}

// Workgroups (j, entry): the first `spans` of an entry take its table row, the others a chunk of
// its partial page each.
__global__ __launch_bounds__(kBlock) void k_fork(tpi_pages p, const void* src, const void* dst,
                                                 int64_t n, bool wide, int spans) {
  const int j = blockIdx.x;
  for (int64_t i = blockIdx.y; i < n; i += gridDim.y) {
    const int32_t len = slot_list(p, LENGTH)[i];
    if (len < 0) return;  // refused
    const int32_t from = slot_list(p, PAIR_SRC)[i], to = slot_list(p, PAIR_DST)[i];
    if (j >= spans) {
      if (from >= 0 && from < p.pages && to >= 0) copy_chunk(p.chunk[j - spans], from, to);
      continue;
    }
    const int64_t s = number(src, i, wide), d = number(dst, i, wide);
    const int32_t full = len / p.tokens;
    for (int64_t k = (int64_t)j * kRowSpan + threadIdx.x; k < (j + 1ll) * kRowSpan && k < full;
         k += kBlock) {
      const int32_t page = p.table[s * p.width + k];
      p.table[d * p.width + k] = page;
      if (page >= 0 && page < p.pages) atomicAdd(&p.refs[page], 1);
    }
    if (j == 0 && threadIdx.x == 0) {
      if (to >= 0) p.table[d * p.width + full] = to;
      p.lengths[d] = len;
    }
  }
}

// A free of many slots: whether one is out of range, for all of k_free's workgroups.
__global__ __launch_bounds__(kPlan) void k_free_check(tpi_pages p, const void* slots, int64_t n,
                                                      bool wide) {
  __shared__ int s_bad;
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < n; i += kPlan) {
    const int64_t s = number(slots, i, wide);
    if (s < 0 || s >= p.slots) s_bad = 1;
  }
  __syncthreads();
  if (threadIdx.x == 0) p.header[TPI_PAGES_BAD] = s_bad;
}

__global__ __launch_bounds__(kBlock) void k_free(tpi_pages p, const void* slots, int64_t n,
                                                 bool wide, bool checked) {
  __shared__ int s_bad, s_len, s_count;
  if (threadIdx.x == 0) {
    s_bad = checked ? p.header[TPI_PAGES_BAD] : 0;
    s_count = 0;
  }
  __syncthreads();
  if (!checked)
    for (int64_t i = threadIdx.x; i < n; i += kBlock) {  // every workgroup comes to the same end
      const int64_t s = number(slots, i, wide);
      if (s < 0 || s >= p.slots) s_bad = 1;
    }
  __syncthreads();
  if (s_bad) {
    if (threadIdx.x == 0) refuse(p, TPI_PAGES_ESLOT);
    return;
  }
  const int64_t s = number(slots, blockIdx.x, wide);
  if (threadIdx.x == 0) s_len = atomicExch(&p.lengths[s], 0);  // named twice: empty by then
  __syncthreads();
  int32_t held = pages_of(s_len, p.tokens);
  if (held > p.width) held = p.width;
  for (int32_t k = threadIdx.x; k < held; k += kBlock) {
    const int32_t page = p.table[s * p.width + k];
    p.table[s * p.width + k] = -1;
    if (page < 0 || page >= p.pages) continue;
    if (atomicSub(&p.refs[page], 1) == 1) {
      const uint32_t bit = 1u << (page & 31);
      atomicOr(&p.free_bits[page >> 5], bit);
      atomicOr(&p.stale_bits[page >> 5], bit);
      atomicAdd(&s_count, 1);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && s_count) atomicAdd(&p.header[TPI_PAGES_FREE], s_count);
}

// Bits of word w whose page is below `page`.
__device__ static inline uint32_t bits_below(int w, int page) {
  const int64_t n = (int64_t)page - 32ll * w;
  return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
}

__global__ __launch_bounds__(kPlan) void k_plan(tpi_pages p, bool clear) {
  __shared__ Words lds;
  const int tid = threadIdx.x;
  const int live = p.pages - p.header[TPI_PAGES_FREE];
  const int words = (p.pages + 31) / 32;
  int holes = 0, movers = 0, clears = 0;
  for (int base = 0; base < words; base += kPlan) {
    int sum;
    const int w = base + tid;
    uint32_t hole = 0, mover = 0, stale = 0;
    if (w < words) {
      const uint32_t free = p.free_bits[w], low = bits_below(w, live);
      const uint32_t freed = bits_below(w, p.pages) & ~low;  // the free pages afterwards
      hole = free & low;
      mover = ~free & freed;
      stale = (p.stale_bits[w] | mover) & freed;  // a mover's old page is stale
      p.free_bits[w] = freed;
      p.stale_bits[w] = clear ? 0 : stale;
    }
    // both counts of a pass (at most 32 kPlan = 32768) in one sum
    const uint32_t before = scan(__popc(hole) | __popc(mover) << 16, &sum);
    emit(lds, hole, holes + (int)(before & 0xffff), base, words, p.pages, list(p, HOLES));
    emit(lds, mover, movers + (int)(before >> 16), base, words, p.pages, list(p, MOVERS));
    holes += sum & 0xffff;
    movers += (uint32_t)sum >> 16;
    if (!clear) continue;
    const int c = scan(__popc(stale), &sum);
    emit(lds, stale, clears + c, base, words, p.pages, list(p, CLEARS));
    clears += sum;
  }
  __syncthreads();
  // as many holes below `live` as live pages at or above it, if the counts are in order
  const int moves = holes < movers ? holes : movers;
  for (int i = tid; i < moves; i += kPlan) {
    const int32_t from = list(p, MOVERS)[i], to = list(p, HOLES)[i];
    p.refs[to] = p.refs[from];
    p.refs[from] = 0;
    list(p, MAP)[from] = to;
  }
  if (tid == 0) {
    p.header[TPI_PAGES_LIVE] = live;
    p.header[TPI_PAGES_MOVES] = moves;
    p.header[TPI_PAGES_CLEARS] = clears;
  }
}

// Workgroups (x, chunk): neighbours take neighbouring pages of one tensor, so that reads and
// writes run through it (neighbours in different tensors measure the same).  The first `spans`
// of every chunk take the table, the others the moved pages x - spans, x - spans + their number, ...
__global__ __launch_bounds__(kBlock) void k_compact(tpi_pages p, int spans) {
  const int x = blockIdx.x;
  if (x < spans) {
    const int live = p.header[TPI_PAGES_LIVE];
    const int64_t entries = (int64_t)p.slots * p.width;
    for (int64_t e = ((int64_t)x * gridDim.y + blockIdx.y) * kBlock + threadIdx.x; e < entries;
         e += (int64_t)spans * gridDim.y * kBlock) {
      const int32_t page = p.table[e];
      if (page >= live && page < p.pages) p.table[e] = list(p, MAP)[page];
    }
    return;
  }
  const int moves = p.header[TPI_PAGES_MOVES];
  for (int c = blockIdx.y; c < p.chunks; c += gridDim.y)
    for (int i = x - spans; i < moves; i += gridDim.x - spans)
      copy_chunk(p.chunk[c], list(p, MOVERS)[i], list(p, HOLES)[i]);
}

__global__ __launch_bounds__(kBlock) void k_clear(tpi_pages p) {
  const int clears = p.header[TPI_PAGES_CLEARS];
  for (int c = blockIdx.y; c < p.chunks; c += gridDim.y)
    for (int i = blockIdx.x; i < clears; i += gridDim.x)
      zero_chunk(p.chunk[c], list(p, CLEARS)[i]);
}

constexpr int64_t kMaxY = 32768;  // of a grid; the loops over entries take the rest

uint32_t rows_of(int64_t n) { return (uint32_t)(n < kMaxY ? n : kMaxY); }

// Workgroups per chunk for an unknown number of pages: enough to fill the GPU several times, so
// that few of them wait for a last one.
uint32_t spread(const tpi_pages* p) {
  const int64_t per = kSpread / p->chunks + 1;
  return (uint32_t)(per < p->pages ? per : p->pages);
}

bool few(const tpi_pages* p, int64_t n) {
  return n <= kPlan && p->slots <= kFewSlots && p->pages <= kFewPages;
}

}  // namespace

extern "C" {

int tpi_pages_copy(const tpi_pages* p, const void* src, const void* dst, int64_t n, int wide,
                   uint64_t stream) {
  if (n <= 0) return 0;
  TPI_HIP(tpi_launch(k_copy, dim3(p->chunks, rows_of(n)), kBlock, (hipStream_t)stream, *p, src, dst, n,
                     wide & 1));
  return 0;
}

int tpi_pages_fork(const tpi_pages* p, const void* src, const void* dst, int64_t n, int wide,
                   uint64_t stream) {
  if (n <= 0) return 0;
  if (n > p->slots) return tpi_fail("fork: more destinations than slots");
  hipStream_t s = (hipStream_t)stream;
  const auto reserve = few(p, n) ? k_reserve_few<true> : k_reserve<true>;
  TPI_HIP(tpi_launch(reserve, 1, kPlan, s, *p, src, dst, (int)n, wide & 1, nullptr, false, 0));
  const int spans = (p->width + kRowSpan - 1) / kRowSpan;
  TPI_HIP(tpi_launch(k_fork, dim3(spans + p->chunks, rows_of(n)), kBlock, s, *p, src, dst, n, wide & 1,
                     spans));
  return 0;
}

int tpi_pages_extend(const tpi_pages* p, const void* slots, int64_t n, int wide,
                     const void* more, int64_t each, uint64_t stream) {
  if (n <= 0) return 0;
  if (n > p->slots) return tpi_fail("extend: more sequences than slots");
  const auto reserve = few(p, n) ? k_reserve_few<false> : k_reserve<false>;
  TPI_HIP(tpi_launch(reserve, 1, kPlan, (hipStream_t)stream, *p, slots, nullptr, (int)n, wide & 1, more,
                     (wide & 2) != 0, each));
  return 0;
}

int tpi_pages_free(const tpi_pages* p, const void* slots, int64_t n, int wide, uint64_t stream) {
  if (n <= 0) return 0;
  if (n > p->slots) return tpi_fail("free: more sequences than slots");
  hipStream_t s = (hipStream_t)stream;
  const bool many = n > kPlan;  // up to here a workgroup's own look at all slots is 4 loads a thread
  if (many) {
    TPI_HIP(tpi_launch(k_free_check, 1, kPlan, s, *p, slots, n, wide & 1));
  }
  TPI_HIP(tpi_launch(k_free, (uint32_t)n, kBlock, s, *p, slots, n, wide & 1, many));
  return 0;
}

int tpi_pages_compact(const tpi_pages* p, int clear, uint64_t stream) {
  hipStream_t s = (hipStream_t)stream;
  TPI_HIP(tpi_launch(k_plan, 1, kPlan, s, *p, clear != 0));
  const int64_t table = ((int64_t)p->slots * p->width + 4 * kBlock - 1) / (4 * kBlock);
  const int chunks = (int)rows_of(p->chunks);
  const int spans = (int)(((table < 256 ? table : 256) + chunks - 1) / chunks);
  TPI_HIP(tpi_launch(k_compact, dim3(spans + spread(p), chunks), kBlock, s, *p, spans));
  if (clear) {
    TPI_HIP(tpi_launch(k_clear, dim3(spread(p), chunks), kBlock, s, *p));
  }
  return 0;
}

}  // extern "C"
