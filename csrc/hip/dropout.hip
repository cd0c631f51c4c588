// Dropout from a counter-based generator, forward and (the same kernel) backward.
//
//   out[e] = (kept(seed, draw, n(e)) ? x[e] * scale : 0) + residual[e]
//
// with n(e) the element's index in the whole tensor (csrc/common/philox.h): nothing of the mask
// is stored, the backward pass draws it again.  The arithmetic is in 32 bits, one multiplication
// and one addition, each rounded by itself (the host implementation gives the same bits), and
// one rounding to the output's type.  A dropped element is 0 whatever x holds (NaN, infinity).
//
//  k_dropout_rows     rows of unit stride, however they lie (a contiguous tensor is one row).  A
//                     thread owns the 8 elements of a generator block: one 16-byte access (two for
//                     fp32) each way.
//  k_dropout_tiles    views whose index runs across memory (transposed, channels last): a thread
//                     owns the 8 x 8 elements of 8 generator blocks, 8 neighbours in memory each.
//  k_dropout_strided  anything else: one thread per element, which draws a block of its own.
#include <hip/hip_runtime.h>

#include "../common/philox.h"
#include "internal.h"
#include "tpi_hip.h"

#pragma clang fp contract(off)

namespace {

constexpr int kThreads = 256;

template <int TYPE> struct Elem;
template <> struct Elem<TPI_F32> { typedef float type; };
template <> struct Elem<TPI_F16> { typedef _Float16 type; };
template <> struct Elem<TPI_BF16> { typedef __bf16 type; };

// Division of a number below 2^31 by a constant: (n + high word of n * mul) >> shift, with
// mul = floor(2^32 (2^shift - d) / d) + 1 and shift the least with 2^shift >= d.
struct Divider {
  uint32_t mul, shift;
};

// A dimension of rows: how many, and the steps from one to the next.
struct Outer {
  int64_t size, sx, sr, so, si;  // elements
  Divider by;                    // by size
};

struct RowArgs {
  const void* x;
  const void* residual;
  void* out;
  const uint64_t* state;
  uint64_t* used;
  uint64_t seed, draw, first;
  int64_t rows, cols;
  uint64_t per_row;  // generator blocks per row
  Divider by_row;    // by per_row
  int32_t outer;     // dimensions of rows
  bool narrow;       // every quotient and divisor is below 2^31
  Outer dim[TPI_MAX_DIMS - 1];  // the innermost first
  tpi_keep keep;
  float scale;
};

__device__ static inline int64_t quotient(int64_t n, int64_t d, Divider by, bool narrow) {
  if (!narrow) return n / d;
  return (__umulhi((uint32_t)n, by.mul) + (uint32_t)n) >> by.shift;
}

// Offsets of a row in the operands and in the index; returns its place in the innermost dimension.
// That one is taken first, from a fixed place in the arguments: most views have no other.
template <bool RES>
__device__ static inline int64_t walk(const RowArgs& a, int64_t row, int64_t& sx, int64_t& sr,
                                      int64_t& so, uint64_t& start) {
  int64_t inner = row;
  if (a.outer > 1) {
    int64_t rest = quotient(row, a.dim[0].size, a.dim[0].by, a.narrow);
    inner = row - rest * a.dim[0].size;
    for (int k = 1; k < a.outer; ++k) {
      const Outer& d = a.dim[k];
      const int64_t q = k + 1 < a.outer ? quotient(rest, d.size, d.by, a.narrow) : 0;
      const int64_t i = rest - q * d.size;
      sx += i * d.sx;
      if (RES) sr += i * d.sr;
      so += i * d.so;
      start += (uint64_t)(i * d.si);
      rest = q;
    }
  }
  sx += inner * a.dim[0].sx;
  if (RES) sr += inner * a.dim[0].sr;
  so += inner * a.dim[0].so;
  start += (uint64_t)(inner * a.dim[0].si);
  return inner;
}

// The draw's seed and number: from the call, or from device memory at the time the kernel runs.
struct Key {
  uint64_t seed, draw;
};

__device__ static inline Key read_key(const uint64_t* state, uint64_t* used, uint64_t seed,
                                      uint64_t draw) {
  Key k{seed, draw};
  if (state) {
    k.seed = state[0];
    k.draw = state[1] + draw;
  }
  if (used && blockIdx.x == 0 && threadIdx.x == 0) {
    used[0] = k.seed;
    used[1] = k.draw;
  }
  return k;
}

// One element.  The compiler may join an fp32 operation with a conversion to fp16 (a mixed
// fma that rounds once, where two roundings are meant): the empty asm keeps them apart.
template <int OUT, bool RES>
__device__ static inline typename Elem<OUT>::type apply(float x, float residual, bool kept,
                                                        float scale) {
  float v = kept ? x * scale : 0.0f;
  if (RES) v = v + residual;
  if (OUT == TPI_F16) asm("" : "+v"(v));
  return (typename Elem<OUT>::type)v;
}

// Whether a half-word of the block equals keep.high.
__device__ static inline bool ties(const tpi_philox_words& p, tpi_keep keep) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const uint32_t both = keep.high | keep.high << 16;
  u16x2 least = {1, 1};  // 0 where some half-word is equal
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const u16x2 off = __builtin_bit_cast(u16x2, p.w[k] ^ both);
    least = __builtin_elementwise_min(least, off);
  }
  return __builtin_bit_cast(uint32_t, least) != 0x00010001u;
}

// 8 elements that may begin at any element: the GPU's vector accesses need no alignment.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
  T e[8];
};

template <typename T>
__device__ static inline Eight<T> load8(const T* p) {
  return *(const Eight<T>*)p;
}

// Elements of 2 bytes are one 16-byte access, stored nontemporally: the caches keep what is read
// (16M bf16 elements with a residual 18.5 us instead of 19.6, 8M 10.4 instead of 11.1; loading them
// so too costs what the last kernel left there: 14.4 us instead of 13.5 without a residual).  Those of
// 4 bytes are two, each half of what a line's lanes write: nontemporal they cost 99 us, not 92.
template <typename T>
__device__ static inline void store8(T* p, Eight<T> v) {
  if constexpr (sizeof(T) == 2) {
    typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(2)));
    __builtin_nontemporal_store(__builtin_bit_cast(raw, v), (raw*)p);
  } else {
    *(Eight<T>*)p = v;
  }
}

// A thread takes one block of the generator (two or four, with all loads in flight first, are 6
// to 20 % slower: fewer waves than accesses to hide).  Its 20 products are a quarter of what the
// memory leaves time for: with one round instead of 10 the kernel is 4 % faster.
// ONE: a single row, without the walk (5 % of a contiguous tensor's time).
template <int IN, int OUT, bool RES, bool ONE>
__global__ __launch_bounds__(kThreads) void k_dropout_rows(RowArgs a) {
  typedef typename Elem<IN>::type TI;
  typedef typename Elem<OUT>::type TO;
  const Key key = read_key(a.state, a.used, a.seed, a.draw);
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  int64_t row = 0;
  if (!ONE) row = quotient(t, (int64_t)a.per_row, a.by_row, a.narrow);
  if (!ONE && row >= a.rows) return;
  const int64_t b = t - row * (int64_t)a.per_row;
  uint64_t start = a.first;  // index of the row's first element
  int64_t sx = 0, sr = 0, so = 0;
  if (!ONE) walk<RES>(a, row, sx, sr, so, start);
  const uint64_t block = (start >> 3) + (uint64_t)b;
  const int64_t c0 = b * 8 - (int64_t)(start & 7);  // column of the block's element 0
  if (c0 >= a.cols) return;
  const TI* x = (const TI*)a.x + sx + c0;
  const TO* r = RES ? (const TO*)a.residual + sr + c0 : nullptr;
  TO* o = (TO*)a.out + so + c0;
  const bool whole = c0 >= 0 && c0 + 8 <= a.cols;
  Eight<TI> in;
  Eight<TO> add;
  if (whole) {
    in = load8(x);
    if (RES) add = load8(r);
  }
  const tpi_philox_words p = tpi_philox(block, key.draw, 0, key.seed);
  if (whole && !ties(p, a.keep)) {
    Eight<TO> out;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      out.e[j] = apply<OUT, RES>((float)in.e[j], RES ? (float)add.e[j] : 0.0f,
                                 tpi_philox_half(p, j) < a.keep.high, a.scale);
    store8(o, out);
    return;
  }
  // a row's ends, and blocks that need their second number (one in 8192): element by element
  const uint32_t kept = tpi_kept_bits(p, block, key.draw, key.seed, a.keep);
#pragma unroll 1
  for (int j = 0; j < 8; ++j)
    if (c0 + j >= 0 && c0 + j < a.cols)
      o[j] = apply<OUT, RES>((float)x[j], RES ? (float)r[j] : 0.0f, kept >> j & 1, a.scale);
}

struct TileArgs {
  RowArgs row;                 // rows, per_row and outer: of tiles across `along`
  int64_t along, across;       // sizes: of the index's dimension, of memory's
  int64_t ax, ar, ao, ai;      // steps of the three operands along, of the index across
};

// Tiles of 8 elements along the index, which are one generator block, by 8 across it, which are
// neighbours in memory.  Every block of the view is whole or cut at the dimension's end (the
// host has checked: all steps of the index but this one are multiples of 8).  Lanes lie across,
// so that their accesses join to whole lines.  16M bf16 elements, channels last: 15.6 us, 123 with
// a thread and a block of the generator per element (contiguous: 13.2).
template <int IN, int OUT, bool RES>
__global__ __launch_bounds__(kThreads) void k_dropout_tiles(TileArgs t) {
  typedef typename Elem<IN>::type TI;
  typedef typename Elem<OUT>::type TO;
  const RowArgs& a = t.row;
  const Key key = read_key(a.state, a.used, a.seed, a.draw);
  const int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t line = quotient(g, (int64_t)a.per_row, a.by_row, a.narrow);
  if (line >= a.rows) return;
  const int64_t b0 = (g - line * (int64_t)a.per_row) * 8;  // across
  uint64_t start = a.first;
  int64_t sx = 0, sr = 0, so = 0;
  const int64_t a0 = 8 * walk<RES>(a, line, sx, sr, so, start);  // along
  const int na = (int)(t.along - a0 < 8 ? t.along - a0 : 8);
  const int nb = (int)(t.across - b0 < 8 ? t.across - b0 : 8);
  uint64_t kept = 0;  // bit 8 j + i: element i along, j across
  for (int j = 0; j < nb; ++j)
    kept |= (uint64_t)tpi_draw_block((start + (uint64_t)((b0 + j) * t.ai)) >> 3, key.draw, key.seed,
                                     a.keep) << (8 * j);
  const TI* x = (const TI*)a.x + sx + b0;
  const TO* r = RES ? (const TO*)a.residual + sr + b0 : nullptr;
  TO* o = (TO*)a.out + so + b0;
  for (int i = 0; i < na; ++i, x += t.ax, r += RES ? t.ar : 0, o += t.ao, kept >>= 1) {
    if (nb == 8) {
      const Eight<TI> in = load8(x);
      Eight<TO> out;
      if (RES) out = load8(r);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        out.e[j] = apply<OUT, RES>((float)in.e[j], RES ? (float)out.e[j] : 0.0f,
                                   kept >> (8 * j) & 1, a.scale);
      store8(o, out);
    } else {
      for (int j = 0; j < nb; ++j)
        o[j] = apply<OUT, RES>((float)x[j], RES ? (float)r[j] : 0.0f, kept >> (8 * j) & 1, a.scale);
    }
  }
}

template <int IN, int OUT, bool RES>
__global__ __launch_bounds__(kThreads) void k_dropout_strided(tpi_dropout_args a, uint64_t total) {
  typedef typename Elem<IN>::type TI;
  typedef typename Elem<OUT>::type TO;
  const Key key = read_key((const uint64_t*)a.state, (uint64_t*)a.used, a.seed, a.draw);
  const tpi_keep keep = tpi_keep_below(a.threshold);
  for (uint64_t e = (uint64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
       e += (uint64_t)gridDim.x * kThreads) {
    uint64_t rest = e, n = a.first;
    int64_t x = 0, r = 0, o = 0;
    for (int d = a.ndim - 1; d >= 0; --d) {
      const uint64_t size = (uint64_t)a.sizes[d], q = rest / size;
      const int64_t i = (int64_t)(rest - q * size);
      x += i * a.sx[d];
      if (RES) r += i * a.sr[d];
      o += i * a.so[d];
      n += (uint64_t)(i * a.si[d]);
      rest = q;
    }
    const uint32_t kept = tpi_draw_block(n >> 3, key.draw, key.seed, keep);
    ((TO*)a.out)[o] = apply<OUT, RES>((float)((const TI*)a.x)[x],
                                      RES ? (float)((const TO*)a.residual)[r] : 0.0f,
                                      kept >> (n & 7) & 1, a.scale);
  }
}

Divider divider(uint64_t d) {
  Divider by{0, 0};
  if (d >> 31) return by;  // not used
  while ((1ull << by.shift) < d) ++by.shift;
  by.mul = (uint32_t)((((1ull << by.shift) - d) << 32) / d + 1);
  return by;
}

RowArgs common(const tpi_dropout_args& a) {
  RowArgs k{};
  k.x = (const void*)a.x;
  k.residual = (const void*)a.residual;
  k.out = (void*)a.out;
  k.state = (const uint64_t*)a.state;
  k.used = (uint64_t*)a.used;
  k.seed = a.seed;
  k.draw = a.draw;
  k.keep = tpi_keep_below(a.threshold);
  k.first = a.first;
  k.scale = a.scale;
  k.rows = 1;
  k.narrow = true;
  return k;
}

void add_outer(RowArgs& k, int64_t size, int64_t sx, int64_t sr, int64_t so, int64_t si) {
  k.dim[k.outer++] = Outer{size, sx, sr, so, si, divider((uint64_t)size)};
  k.rows *= size;
  k.narrow = k.narrow && size >> 31 == 0;
}

// Workgroups for per_row threads in each of the rows; 0: more than a launch has (2^32 threads, 34e9
// elements of rows).
uint32_t finish(RowArgs& k) {
  k.by_row = divider(k.per_row);
  const uint64_t threads = k.per_row * (uint64_t)k.rows;
  // the last workgroup's threads behind the last block are divided, too
  k.narrow = k.narrow && k.per_row >> 31 == 0 && (threads + kThreads) >> 31 == 0;
  const uint64_t grid = (threads + kThreads - 1) / kThreads;
  return grid * kThreads >> 32 ? 0 : (uint32_t)grid;
}

template <int IN, int OUT, bool RES>
int launch_rows(const tpi_dropout_args& a, hipStream_t stream) {
  const int last = a.ndim - 1;
  RowArgs k = common(a);
  k.cols = a.sizes[last];
  uint64_t lead = a.first % 8;  // of a row's first element in its block; 7: of some row
  for (int d = last - 1; d >= 0; --d) {
    add_outer(k, a.sizes[d], a.sx[d], a.sr[d], a.so[d], a.si[d]);
    if (a.si[d] % 8) lead = 7;
  }
  k.per_row = ((uint64_t)k.cols + lead + 7) / 8;
  const uint32_t grid = finish(k);
  if (!grid) return tpi_fail("dropout: tensor too large");
  const auto kernel = last ? k_dropout_rows<IN, OUT, RES, false> : k_dropout_rows<IN, OUT, RES, true>;
  TPI_HIP(tpi_launch(kernel, grid, kThreads, stream, k));
  return 0;
}

// `along`: the dimension that the index runs along, `across`: the one that memory does.
template <int IN, int OUT, bool RES>
int launch_tiles(const tpi_dropout_args& a, int along, int across, hipStream_t stream) {
  TileArgs t{};
  t.row = common(a);
  t.along = a.sizes[along];
  t.across = a.sizes[across];
  t.ax = a.sx[along];
  t.ar = a.sr[along];
  t.ao = a.so[along];
  t.ai = a.si[across];
  add_outer(t.row, (t.along + 7) / 8, 8 * t.ax, 8 * t.ar, 8 * t.ao, 8);
  for (int d = a.ndim - 1; d >= 0; --d)
    if (d != along && d != across)
      add_outer(t.row, a.sizes[d], a.sx[d], a.sr[d], a.so[d], a.si[d]);
  t.row.per_row = (uint64_t)(t.across + 7) / 8;
  const uint32_t grid = finish(t.row);
  if (!grid) return tpi_fail("dropout: tensor too large");
  const auto kernel = k_dropout_tiles<IN, OUT, RES>;
  TPI_HIP(tpi_launch(kernel, grid, kThreads, stream, t));
  return 0;
}

template <int IN, int OUT, bool RES>
int launch(const tpi_dropout_args& a, hipStream_t stream) {
  const auto unit = [&](int d) {
    return a.sx[d] == 1 && a.so[d] == 1 && (!RES || a.sr[d] == 1);
  };
  const int last = a.ndim - 1;
  if (unit(last) && a.si[last] == 1) return launch_rows<IN, OUT, RES>(a, stream);
  int along = -1, across = -1;
  bool whole = a.first % 8 == 0;  // every block begins with an element of the view
  for (int d = 0; d < a.ndim; ++d) {
    if (a.si[d] == 1) along = d;
    else if (a.si[d] % 8) whole = false;
    if (unit(d)) across = d;
  }
  if (whole && along >= 0 && across >= 0 && along != across)
    return launch_tiles<IN, OUT, RES>(a, along, across, stream);
  uint64_t total = 1;
  for (int d = 0; d < a.ndim; ++d) total *= (uint64_t)a.sizes[d];
  const uint64_t want = (total + kThreads - 1) / kThreads;
  const uint32_t grid = (uint32_t)(want < 65536 ? want : 65536);
  const auto kernel = k_dropout_strided<IN, OUT, RES>;
  TPI_HIP(tpi_launch(kernel, grid, kThreads, stream, a, total));
  return 0;
}

template <int IN, int OUT>
int launch(const tpi_dropout_args& a, hipStream_t s) {
  if (!a.residual) return launch<IN, OUT, false>(a, s);
  // the residual stream and its gradient may be wider than the activations, not narrower
  if constexpr (OUT == IN || OUT == TPI_F32) return launch<IN, OUT, true>(a, s);
  return tpi_fail("dropout: unsupported types");
}

}  // namespace

extern "C" int tpi_capture_id(uint64_t stream, uint64_t* id) {
  *id = 0;
  if (!stream) return 0;  // the default stream is never captured
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long number = 0;
  TPI_HIP(hipStreamGetCaptureInfo((hipStream_t)stream, &status, &number));
  if (status != hipStreamCaptureStatusNone) *id = number + 1;  // whatever the first one's is
  return 0;
}

extern "C" int tpi_dropout(const tpi_dropout_args* args, uint64_t stream) {
  const tpi_dropout_args& a = *args;
  if (a.ndim < 1 || a.ndim > TPI_MAX_DIMS) return tpi_fail("dropout: bad number of dimensions");
  for (int d = 0; d < a.ndim; ++d)
    if (a.sizes[d] < 1) return tpi_fail("dropout: empty dimension");
  if (a.threshold > 1ull << 32) return tpi_fail("dropout: bad threshold");
  hipStream_t s = (hipStream_t)stream;
  switch (a.in_type * 3 + a.out_type) {
    case TPI_F32 * 3 + TPI_F32: return launch<TPI_F32, TPI_F32>(a, s);
    case TPI_F16 * 3 + TPI_F16: return launch<TPI_F16, TPI_F16>(a, s);
    case TPI_BF16 * 3 + TPI_BF16: return launch<TPI_BF16, TPI_BF16>(a, s);
    case TPI_F16 * 3 + TPI_F32: return launch<TPI_F16, TPI_F32>(a, s);
    case TPI_BF16 * 3 + TPI_F32: return launch<TPI_BF16, TPI_F32>(a, s);
    case TPI_F32 * 3 + TPI_F16: return launch<TPI_F32, TPI_F16>(a, s);
    case TPI_F32 * 3 + TPI_BF16: return launch<TPI_F32, TPI_BF16>(a, s);
    default: return tpi_fail("dropout: unsupported types");
  }
}
