// Dropout from a counter-based generator, forward and (the same kernel) backward.
//
//   out[e] = (kept(seed, draw, n(e)) ? x[e] * scale : 0) + residual[e]
//
// with n(e) the element's index in the whole tensor (csrc/common/philox.h): nothing of the mask
// is stored, the backward pass draws it again.  The arithmetic is in 32 bits, one multiplication
// and one addition, each rounded by itself (the host implementation gives the same bits), and
// one rounding to the output's type.  A dropped element is 0 whatever x holds (NaN, infinity).
//
//  k_dropout_rows     rows of unit stride (a contiguous tensor is one row).  A thread owns the 8
//                     elements of one generator block.
//  k_dropout_strided  anything else, one thread per element: its own block of the generator.
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

struct RowArgs {
  const void* x;
  const void* residual;
  void* out;
  const uint64_t* state;
  uint64_t* used;
  uint64_t seed, draw, threshold, first;
  int64_t rows, cols, sx, sr, so, si;  // elements
  uint64_t per_row;                    // generator blocks (threads) per row
  float scale;
};

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

// VEC: every row starts on a block of the generator and on 16 bytes in memory, so a thread's 8
// elements move as vectors; otherwise element by element, the block's ends cut at the row's.
template <int IN, int OUT, bool RES, bool VEC>
__global__ __launch_bounds__(kThreads) void k_dropout_rows(RowArgs a) {
  typedef typename Elem<IN>::type TI;
  typedef typename Elem<OUT>::type TO;
  typedef TI vin __attribute__((ext_vector_type(8)));
  typedef TO vout __attribute__((ext_vector_type(8)));
  const Key key = read_key(a.state, a.used, a.seed, a.draw);
  const uint64_t t = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t row = a.rows == 1 ? 0 : (int64_t)(t / a.per_row);
  if (row >= a.rows) return;
  const uint64_t b = t - (uint64_t)row * a.per_row;
  if (b >= a.per_row) return;
  const TI* x = (const TI*)a.x + row * a.sx;
  const TO* r = RES ? (const TO*)a.residual + row * a.sr : nullptr;
  TO* o = (TO*)a.out + row * a.so;
  const uint64_t start = a.first + (uint64_t)row * (uint64_t)a.si;
  const int64_t c0 = (int64_t)(b * 8) - (int64_t)(start & 7);  // column of the block's lane 0
  if (c0 >= a.cols) return;
  const uint32_t kept = tpi_draw_block((start >> 3) + b, key.draw, key.seed, a.threshold);
  if (VEC && c0 + 8 <= a.cols) {
    const vin v = *(const vin*)(x + c0);
    vout w;
    if (RES) w = *(const vout*)(r + c0);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      w[j] = apply<OUT, RES>((float)v[j], RES ? (float)w[j] : 0.0f, kept >> j & 1, a.scale);
    *(vout*)(o + c0) = w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t c = c0 + j;
    if (c >= 0 && c < a.cols)
      o[c] = apply<OUT, RES>((float)x[c], RES ? (float)r[c] : 0.0f, kept >> j & 1, a.scale);
  }
}

template <int IN, int OUT, bool RES>
__global__ __launch_bounds__(kThreads) void k_dropout_strided(tpi_dropout_args a, uint64_t total) {
  typedef typename Elem<IN>::type TI;
  typedef typename Elem<OUT>::type TO;
  const Key key = read_key((const uint64_t*)a.state, (uint64_t*)a.used, a.seed, a.draw);
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
    const uint32_t kept = tpi_draw_block(n >> 3, key.draw, key.seed, a.threshold);
    ((TO*)a.out)[o] = apply<OUT, RES>((float)((const TI*)a.x)[x],
                                      RES ? (float)((const TO*)a.residual)[r] : 0.0f,
                                      kept >> (n & 7) & 1, a.scale);
  }
}

int64_t elem_bytes(int type) { return type == TPI_F32 ? 4 : 2; }

template <int IN, int OUT, bool RES>
int launch(const tpi_dropout_args& a, hipStream_t stream) {
  uint64_t total = 1;
  bool rows = a.ndim <= 2;
  for (int d = 0; d < a.ndim; ++d) total *= (uint64_t)a.sizes[d];
  const int last = a.ndim - 1;
  rows = rows && a.sx[last] == 1 && a.so[last] == 1 && a.si[last] == 1 &&
         (!RES || a.sr[last] == 1);
  if (!rows) {
    const uint64_t want = (total + kThreads - 1) / kThreads;
    const uint32_t grid = (uint32_t)(want < 65536 ? want : 65536);
    k_dropout_strided<IN, OUT, RES><<<grid, kThreads, 0, stream>>>(a, total);
    TPI_HIP(hipGetLastError());
    return 0;
  }
  RowArgs k{};
  k.x = (const void*)a.x;
  k.residual = (const void*)a.residual;
  k.out = (void*)a.out;
  k.state = (const uint64_t*)a.state;
  k.used = (uint64_t*)a.used;
  k.seed = a.seed;
  k.draw = a.draw;
  k.threshold = a.threshold;
  k.first = a.first;
  k.scale = a.scale;
  k.cols = a.sizes[last];
  k.rows = a.ndim == 2 ? a.sizes[0] : 1;
  if (a.ndim == 2) {
    k.sx = a.sx[0];
    k.sr = RES ? a.sr[0] : 0;
    k.so = a.so[0];
    k.si = a.si[0];
  }
  const auto on16 = [](uint64_t ptr, int64_t stride, int64_t bytes) {
    return ptr % 16 == 0 && stride * bytes % 16 == 0;
  };
  const bool vec = a.first % 8 == 0 && k.si % 8 == 0 && on16(a.x, k.sx, elem_bytes(IN)) &&
                   on16(a.out, k.so, elem_bytes(OUT)) &&
                   (!RES || on16(a.residual, k.sr, elem_bytes(OUT)));
  // a row that starts inside a block touches up to one more of them
  k.per_row = vec ? (uint64_t)(k.cols + 7) / 8 : (uint64_t)(k.cols + 14) / 8;
  const uint64_t threads = k.per_row * (uint64_t)k.rows;
  const uint64_t grid = (threads + kThreads - 1) / kThreads;
  if (grid > 0x7fffffffull) return tpi_fail("dropout: tensor too large");
  if (vec)
    k_dropout_rows<IN, OUT, RES, true><<<(uint32_t)grid, kThreads, 0, stream>>>(k);
  else
    k_dropout_rows<IN, OUT, RES, false><<<(uint32_t)grid, kThreads, 0, stream>>>(k);
  TPI_HIP(hipGetLastError());
  return 0;
}

template <int IN, int OUT>
int launch(const tpi_dropout_args& a, hipStream_t s) {
  return a.residual ? launch<IN, OUT, true>(a, s) : launch<IN, OUT, false>(a, s);
}

}  // namespace

extern "C" int tpi_dropout(const tpi_dropout_args* args, uint64_t stream) {
  const tpi_dropout_args& a = *args;
  if (a.ndim < 1 || a.ndim > TPI_MAX_DIMS) return tpi_fail("dropout: bad number of dimensions");
  for (int d = 0; d < a.ndim; ++d)
    if (a.sizes[d] < 1) return tpi_fail("dropout: empty dimension");
  if (a.threshold > 1ull << 32) return tpi_fail("dropout: bad threshold");
  hipStream_t s = (hipStream_t)stream;
  // the residual stream and its gradient may be wider than the activations
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
