// Host-side helpers: element conversions for the quantisers of data in host
// memory, and a launch's grid.
#ifndef QIK_HOST_H
#define QIK_HOST_H

#include <stdint.h>
#include <string.h>
#include <cmath>

#include "qik_fp8.h"

namespace qik_host {

// exact fp32 value of element i of a bf16 / fp16 / fp32 host array
inline float host_elem(const void* w, int32_t dtype, int64_t i) {
  if (dtype == QIK_DTYPE_FP32) return static_cast<const float*>(w)[i];
  const uint16_t h = static_cast<const uint16_t*>(w)[i];
  uint32_t bits;
  if (dtype == QIK_DTYPE_BF16) {
    bits = (uint32_t)h << 16;
  } else {
    // binary16: 1 sign, 5 exponent bits (bias 15), 10 mantissa bits
    const uint32_t sign = (uint32_t)(h & 0x8000u) << 16;
    const uint32_t e = (h >> 10) & 0x1fu, m = h & 0x3ffu;
    if (e == 0x1f) {
      bits = sign | 0x7f800000u | (m << 13);
    } else if (e != 0) {
      bits = sign | ((e + 112u) << 23) | (m << 13);
    } else {
      // zero or subnormal: m * 2^-24, exact in fp32
      const float f = (float)m * 5.9604644775390625e-8f;
      memcpy(&bits, &f, 4);
      bits |= sign;
    }
  }
  float f;
  memcpy(&f, &bits, 4);
  return f;
}

// e4m3fn code of q (|q| <= 448 or NaN), round to nearest even; NaN keeps its
// sign bit (0x7f / 0xff), and a magnitude that rounds past 448 is NaN (the
// format has no infinity)
inline unsigned char host_e4m3fn(float q) {
  uint32_t u;
  memcpy(&u, &q, 4);
  const unsigned char sign = (unsigned char)((u >> 24) & 0x80u);
  const uint32_t a = u & 0x7fffffffu;
  if (a >= 0x43e80000u) return sign | 0x7f;  // NaN, or |q| >= 464 (= 448 + half a step)
  if (a < 0x3c800000u) {
    // below 2^-6: subnormal codes m * 2^-9, m = round_even(|q| * 512) (exact scaling)
    float fa;
    memcpy(&fa, &a, 4);
    return sign | (unsigned char)std::nearbyint(fa * 512.0f);
  }
  // normal: keep 3 mantissa bits with round-to-nearest-even at bit 20, then
  // move the exponent from bias 127 to bias 7
  const uint32_t r = a + 0x7ffffu + ((a >> 20) & 1u);
  return sign | (unsigned char)((r >> 20) - (120u << 3));
}

// `workgroups` of `threads` as a grid of x * y workgroups, less than y of them
// surplus, with fewer than 2^32 threads in x (a launch's limit) and y at most
// 65535; false where no such grid holds them.
inline bool split_grid(int64_t workgroups, int threads, unsigned* x, unsigned* y) {
  const int64_t most = UINT32_MAX / threads;  // workgroups in x
  const int64_t rows = (workgroups + most - 1) / most;
  if (workgroups < 1 || rows > 65535) return false;
  *x = (unsigned)((workgroups + rows - 1) / rows);
  *y = (unsigned)rows;
  return true;
}

}  // namespace qik_host

#endif  // QIK_HOST_H
