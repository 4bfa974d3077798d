// Eight elements of a row, and the block of 32 that a quad of lanes holds: what
// the microscaled quantisers share.
#ifndef QIK_MX_BLOCK_H
#define QIK_MX_BLOCK_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qik_mx.h"

namespace qik_mx {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((__vector_size__(2 * sizeof(__bf16))));
typedef _Float16 f16x2 __attribute__((__vector_size__(2 * sizeof(_Float16))));

// ---------------------------------------------------------------------------
// Eight elements of a row
// ---------------------------------------------------------------------------

template <int DT>
constexpr int elem_bytes() {
  return DT == QIK_DTYPE_FP32 ? 4 : 2;
}

// 8 elements as they lie in memory
template <int DT>
struct Raw8 {
  u32x4 w[DT == QIK_DTYPE_FP32 ? 2 : 1];
};

typedef u32x4 u32x4_u __attribute__((aligned(2)));  // any alignment of an element (gfx950 loads and stores it in one access)

// 8 elements at p: ALIGNED says p is a multiple of 16 bytes
template <int DT, bool ALIGNED>
__device__ __forceinline__ Raw8<DT> load8(const char* p) {
  Raw8<DT> r;
#pragma unroll
  for (int i = 0; i < elem_bytes<DT>() / 2; ++i)
    r.w[i] = ALIGNED ? *reinterpret_cast<const u32x4*>(p + 16 * i) : (u32x4)*reinterpret_cast<const u32x4_u*>(p + 16 * i);
  return r;
}
template <int DT, bool ALIGNED>
__device__ __forceinline__ void store8(char* p, const Raw8<DT>& r) {
#pragma unroll
  for (int i = 0; i < elem_bytes<DT>() / 2; ++i) {
    if constexpr (ALIGNED) *reinterpret_cast<u32x4*>(p + 16 * i) = r.w[i];
    else *reinterpret_cast<u32x4_u*>(p + 16 * i) = r.w[i];
  }
}
typedef u32x2 u32x2_u __attribute__((aligned(2)));
typedef unsigned u32_u __attribute__((aligned(2)));

// The first n < 8 elements at p, the rest zero, in pieces of 4, 2 and 1: a wave
// issues each piece of a row's end for one lane of it, and element by element
// they cost a tenth of the call (fp16 9001 x 1111 13.4 us, in pieces 11.8).
template <int DT>
__device__ __forceinline__ Raw8<DT> load_part(const char* p, int n) {
  constexpr int EB = elem_bytes<DT>();
  const bool h4 = (n & 4) != 0, h2 = (n & 2) != 0, h1 = (n & 1) != 0;
  Raw8<DT> r = {};
  if constexpr (DT == QIK_DTYPE_FP32) {
    u32x4 a = {};
    u32x2 b = {};
    unsigned c = 0u;
    if (h4) a = *reinterpret_cast<const u32x4_u*>(p);
    if (h2) b = *reinterpret_cast<const u32x2_u*>(p + (n & 4) * EB);
    if (h1) c = *reinterpret_cast<const unsigned*>(p + (n & 6) * EB);
    const u32x4 rest = h2 ? u32x4{b.x, b.y, c, 0u} : u32x4{c, 0u, 0u, 0u};
    r.w[0] = h4 ? a : rest;
    r.w[1] = h4 ? rest : u32x4{};
  } else {
    u32x2 a = {};
    unsigned b = 0u, c = 0u;
    if (h4) a = *reinterpret_cast<const u32x2_u*>(p);
    if (h2) b = *reinterpret_cast<const u32_u*>(p + (n & 4) * EB);
    if (h1) c = *reinterpret_cast<const unsigned short*>(p + (n & 6) * EB);
    const u32x2 rest = h2 ? u32x2{b, c} : u32x2{c, 0u};
    r.w[0] = h4 ? u32x4{a.x, a.y, rest.x, rest.y} : u32x4{rest.x, rest.y, 0u, 0u};
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void store_part(char* p, const Raw8<DT>& r, int n) {
  constexpr int EB = elem_bytes<DT>();
  const bool h4 = (n & 4) != 0, h2 = (n & 2) != 0;
  if constexpr (DT == QIK_DTYPE_FP32) {
    const u32x4 rest = h4 ? r.w[1] : r.w[0];
    if (h4) *reinterpret_cast<u32x4_u*>(p) = r.w[0];
    if (h2) *reinterpret_cast<u32x2_u*>(p + (n & 4) * EB) = u32x2{rest.x, rest.y};
    if (n & 1) *reinterpret_cast<unsigned*>(p + (n & 6) * EB) = h2 ? rest.z : rest.x;
  } else {
    const u32x2 rest = h4 ? u32x2{r.w[0].z, r.w[0].w} : u32x2{r.w[0].x, r.w[0].y};
    if (h4) *reinterpret_cast<u32x2_u*>(p) = u32x2{r.w[0].x, r.w[0].y};
    if (h2) *reinterpret_cast<u32_u*>(p + (n & 4) * EB) = rest.x;
    if (n & 1) *reinterpret_cast<unsigned short*>(p + (n & 6) * EB) = (unsigned short)(h2 ? rest.y : rest.x);
  }
}

template <int DT>
__device__ __forceinline__ void unpack8(const Raw8<DT>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == QIK_DTYPE_FP32) {
      f[2 * i] = __uint_as_float(r.w[i / 2][2 * i % 4]);
      f[2 * i + 1] = __uint_as_float(r.w[i / 2][2 * i % 4 + 1]);
    } else if constexpr (DT == QIK_DTYPE_FP16) {
      const unsigned w = r.w[0][i];
      const f16x2 h = __builtin_bit_cast(f16x2, w);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    } else {
      f[2 * i] = __uint_as_float(r.w[0][i] << 16);
      f[2 * i + 1] = __uint_as_float(r.w[0][i] & 0xffff0000u);
    }
  }
}
// round to nearest even into the element type.  The empty asm pins each value
// as an fp32 one: otherwise the fp16 conversion of a sum or product is folded
// into a mixed-precision fma, which rounds the exact value once instead of
// the fp32 one.
template <int DT>
__device__ __forceinline__ Raw8<DT> pack8(const float (&f)[8]) {
  Raw8<DT> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = f[2 * i], b = f[2 * i + 1];
    if constexpr (DT == QIK_DTYPE_FP32) {
      r.w[i / 2][2 * i % 4] = __float_as_uint(a);
      r.w[i / 2][2 * i % 4 + 1] = __float_as_uint(b);
    } else if constexpr (DT == QIK_DTYPE_FP16) {
      asm volatile("" : "+v"(a), "+v"(b));
      const f16x2 h = {(_Float16)a, (_Float16)b};
      r.w[0][i] = __builtin_bit_cast(unsigned, h);
    } else {
      const bf16x2 h = {(__bf16)a, (__bf16)b};
      r.w[0][i] = __builtin_bit_cast(unsigned, h);
    }
  }
  return r;
}

// ---------------------------------------------------------------------------
// A block of 32 in the four lanes of a quad
// ---------------------------------------------------------------------------

template <int FMT>
constexpr unsigned emax() {
  return FMT == QIK_MXFP4 ? 2u : 8u;
}

// quad_perm {1, 0, 3, 2} and {2, 3, 0, 1}
__device__ __forceinline__ unsigned quad_max(unsigned m) {
  m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));
  return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));
}

// the 8 codes of this lane's share of a block: 4 bytes of MXFP4 (w0) or 8 of
// MXFP8; returns the block's scale byte.  All four lanes of the quad are active.
template <int FMT>
__device__ __forceinline__ unsigned block_codes(const float (&f)[8], unsigned& w0, unsigned& w1) {
#pragma clang fp contract(off)
  unsigned m = 0;  // |x| as bits: unsigned order is |x| order, every NaN above +inf
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  const unsigned E = quad_max(m) >> 23;
  const unsigned byte = E == 255u ? 255u : (E > emax<FMT>() ? E - emax<FMT>() : 0u);
  const float mul = __uint_as_float((254u - (byte == 255u ? 127u : byte)) << 23);  // 2^(127 - byte), normal
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = f[i] * mul;
  w0 = w1 = 0u;
  if constexpr (FMT == QIK_MXFP4) {  // the conversion saturates at 6
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w0, q[0], q[1], 1.0f, 0);
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w0, q[2], q[3], 1.0f, 1);
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w0, q[4], q[5], 1.0f, 2);
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w0, q[6], q[7], 1.0f, 3);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = fminf(fmaxf(q[i], -448.0f), 448.0f);
    w0 = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], (int)w0, false);
    w0 = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], (int)w0, true);
    w1 = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], (int)w1, false);
    w1 = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], (int)w1, true);
  }
  if (byte == 255u) w0 = w1 = 0u;
  return byte;
}

// the v-th 8 codes of a row
template <int FMT>
__device__ __forceinline__ void store_codes(unsigned char* row, int v, unsigned w0, unsigned w1) {
  if constexpr (FMT == QIK_MXFP4) reinterpret_cast<unsigned*>(row)[v] = w0;
  else reinterpret_cast<u32x2*>(row)[v] = u32x2{w0, w1};
}

}  // namespace qik_mx

#endif  // QIK_MX_BLOCK_H
