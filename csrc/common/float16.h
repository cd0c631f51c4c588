// fp16 and bf16 <-> fp32 on the host, rounding to nearest even as the GPU's conversions do.
#pragma once
#include <stdint.h>
#include <string.h>

static inline float tpi_f32_of_bits(uint32_t u) {
  float f;
  memcpy(&f, &u, 4);
  return f;
}

static inline uint32_t tpi_bits_of_f32(float f) {
  uint32_t u;
  memcpy(&u, &f, 4);
  return u;
}

static inline float tpi_bf16_to_f32(uint16_t h) { return tpi_f32_of_bits((uint32_t)h << 16); }

static inline uint16_t tpi_f32_to_bf16(float f) {
  const uint32_t u = tpi_bits_of_f32(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)(u >> 16 | 0x40);  // NaN stays NaN
  return (uint16_t)((u + 0x7fffu + (u >> 16 & 1)) >> 16);
}

static inline float tpi_f16_to_f32(uint16_t h) {
  const uint32_t sign = (uint32_t)(h & 0x8000) << 16, exp = h >> 10 & 31, man = h & 0x3ff;
  if (exp == 31) return tpi_f32_of_bits(sign | 0x7f800000u | man << 13);
  if (exp) return tpi_f32_of_bits(sign | (exp + 112) << 23 | man << 13);
  const float v = (float)man * 0x1p-24f;  // subnormal or zero: exact
  return sign ? -v : v;
}

static inline uint16_t tpi_f32_to_f16(float f) {
  const uint32_t u = tpi_bits_of_f32(f), a = u & 0x7fffffffu;
  const uint16_t sign = (uint16_t)(u >> 16 & 0x8000);
  if (a > 0x7f800000u) return sign | 0x7e00;
  if (a >= 0x477ff000u) return sign | 0x7c00;  // 65520 and more round to infinity
  if (a < 0x38800000u) {  // below 2^-14: a multiple of 2^-24, rounded by an exact scaling
    const float m = tpi_f32_of_bits(a) * 0x1p24f;
    uint32_t q = (uint32_t)m;
    const float rest = m - (float)q;
    if (rest > 0.5f || (rest == 0.5f && (q & 1))) ++q;
    return (uint16_t)(sign | q);
  }
  return (uint16_t)(sign | (a - 0x38000000u + 0xfffu + (a >> 13 & 1)) >> 13);
}
