// Counter-based random bits shared by the host library and the HIP kernels: Philox4x32 with
// 10 rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw: "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011).  A draw is a function of (seed, draw number, element index) alone:
//
//   element n of a tensor belongs to block n / 8; the block's counter is
//       (block lo, block hi, draw lo, draw hi | level << 31),  key (seed lo, seed hi),
//   and its four words hold eight half-words, low half first: element n has half-word n % 8.
//   The element's 32-bit uniform number is level 0's half-word (high) joined with level 1's
//   (low).  It is below a threshold of 32 bits exactly when level 0's half-word is below the
//   threshold's high half, or equal to it and level 1's is below the low half: level 1 decides
//   one element in 65536, so that eight elements cost one block of the generator, not two,
//   at a probability that is exact to 2^-32.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define TPI_PHD __host__ __device__
#else
#define TPI_PHD
#endif

#define TPI_PHILOX_M0 0xD2511F53u
#define TPI_PHILOX_M1 0xCD9E8D57u
#define TPI_PHILOX_W0 0x9E3779B9u
#define TPI_PHILOX_W1 0xBB67AE85u
#define TPI_PHILOX_ROUNDS 10
#define TPI_DRAW_LANES 8  // elements of one block

struct tpi_philox_words {
  uint32_t w[4];
};

TPI_PHD static inline uint32_t tpi_xor3(uint32_t a, uint32_t b, uint32_t c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);  // one instruction
#else
  return a ^ b ^ c;
#endif
}

TPI_PHD static inline tpi_philox_words tpi_philox(uint64_t block, uint64_t draw, uint32_t level,
                                                  uint64_t seed) {
  uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32);
  uint32_t c = (uint32_t)draw, d = (uint32_t)(draw >> 32) | level << 31;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma GCC unroll 10
  for (int r = 0; r < TPI_PHILOX_ROUNDS; ++r) {
    const uint64_t p = (uint64_t)TPI_PHILOX_M0 * a, q = (uint64_t)TPI_PHILOX_M1 * c;
    a = tpi_xor3((uint32_t)(q >> 32), b, k0);
    b = (uint32_t)q;
    c = tpi_xor3((uint32_t)(p >> 32), d, k1);
    d = (uint32_t)p;
    k0 += TPI_PHILOX_W0;
    k1 += TPI_PHILOX_W1;
  }
  return tpi_philox_words{{a, b, c, d}};
}

// Half-word `lane` (0..7) of a block.
TPI_PHD static inline uint32_t tpi_philox_half(const tpi_philox_words& p, int lane) {
  return (p.w[lane >> 1] >> (16 * (lane & 1))) & 0xffffu;
}

// A threshold of 0 .. 2^32 (the share kept * 2^32) as two halves that a half-word is compared
// with: kept below `high`, and at `high` if level 1's half-word is below `low`.  All kept (2^32)
// is "at 0xffff, any": `high` stays a half-word.
struct tpi_keep {
  uint32_t high, low;
};

TPI_PHD static inline tpi_keep tpi_keep_below(uint64_t threshold) {
  if (threshold >> 32) return tpi_keep{0xffffu, 0x10000u};
  return tpi_keep{(uint32_t)(threshold >> 16), (uint32_t)threshold & 0xffffu};
}

// Bit j: element j of the block is kept.  `p` is level 0 of the block.
TPI_PHD static inline uint32_t tpi_kept_bits(const tpi_philox_words& p, uint64_t block,
                                             uint64_t draw, uint64_t seed, tpi_keep keep) {
  uint32_t kept = 0, tie = 0;
  for (int j = 0; j < TPI_DRAW_LANES; ++j) {
    const uint32_t h = tpi_philox_half(p, j);
    kept |= (uint32_t)(h < keep.high) << j;
    tie |= (uint32_t)(h == keep.high) << j;
  }
  if (tie) {
    const tpi_philox_words q = tpi_philox(block, draw, 1, seed);
    for (int j = 0; j < TPI_DRAW_LANES; ++j)
      kept |= (tie >> j & 1u & (uint32_t)(tpi_philox_half(q, j) < keep.low)) << j;
  }
  return kept;
}

TPI_PHD static inline uint32_t tpi_draw_block(uint64_t block, uint64_t draw, uint64_t seed,
                                              tpi_keep keep) {
  return tpi_kept_bits(tpi_philox(block, draw, 0, seed), block, draw, seed, keep);
}
