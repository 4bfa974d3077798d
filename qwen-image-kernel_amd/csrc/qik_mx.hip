// Microscaled (MX) byte movers on MI355X (gfx950): the quantiser to MXFP4 and
// MXFP8, its inverse, and the residual add + RMSNorm whose output is in the
// element type or microscaled.
//
// All three are HBM-bound: a thread moves 8 elements of a row per step, so the
// 32 elements of a block are in the four lanes of a quad, whose largest
// magnitude takes two cross-lane moves, and the elements are converted by
// gfx950's packed fp4 / fp8 conversions.  Contraction is off, so every fp32
// operation rounds on its own and a plain restatement reproduces every bit (the
// norm's but for the order of its fp64 sum, norm_kernel).

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include <limits.h>
#include <algorithm>
#include <cmath>
#include <thread>
#include <vector>

#include "qik_host.h"
#include "qik_mx.h"
#include "qik_mx_block.h"

namespace qik_mx {

inline bool aligned_to(const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) % a) == 0; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// a launch's workgroups in order: a grid of 2^32 threads or more has rows (launch)
__device__ __forceinline__ int64_t block_index() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// byte offset of (row, block) in the scales; C = ceil(K / 256)
__device__ __forceinline__ int64_t scale_at(int64_t row, int block, int C) {
  return ((row >> 5) * C + (block >> 3)) * 256 + (row & 31) * 8 + (block & 7);
}

// ---------------------------------------------------------------------------
// Quantiser and its inverse
// ---------------------------------------------------------------------------

constexpr int QT = 256;  // threads per workgroup
constexpr int MAX_K = 262144;

struct QuantParams {
  const char* x;       // dequantiser: unused
  char* out;           // dequantiser only
  unsigned char* codes;
  unsigned char* scales;
  int64_t M, ldx;
  int64_t units;       // rows (quantiser: padded to 32) x C
  int K, C;
  unsigned magic;      // ceil(2^32 / C)
};

// Row and chunk of the unit `local` units after the workgroup's first.  The
// row of the first is a 64-bit division of uniform values; the rest is below C
// + 16, where the product with ceil(2^32 / C) is exact (C <= 1024).
__device__ __forceinline__ void unit_at(const QuantParams& p, int64_t first, int local, int64_t& row, int& c) {
  const int64_t r0 = first / p.C;
  const unsigned off = (unsigned)(first - r0 * p.C) + (unsigned)local;
  const unsigned q = p.C == 1 ? off : __umulhi(off, p.magic);
  row = r0 + q;
  c = (int)(off - q * (unsigned)p.C);
}

// 32 threads take a unit, one row's 256 elements (8 blocks, 8 scale bytes in a
// row), QU units one after the other, all loads ahead of the first conversion.
// Padding rows and blocks read nothing and get a scale of 0.  Bound by HBM:
// from memory bf16 4352 x 4096 to MXFP4 13.1 us (3.4 TB/s; 10.4 where the 256 MB
// cache holds a part), fp32 12288 x 4096 41.6 us (5.5 TB/s).
// One unit keeps the small calls short (bf16 203 x 12288 3.0 us against 3.3 with
// two and 3.9 with four), two do better on long 16-bit ones (16000 x 3200 26.5
// against 28.5; with four 32.0), one on fp32 (41.1, 43.4, 45.2).
template <int DT, int FMT, bool ALIGNED, int QU>
__global__ void __launch_bounds__(QT) quant_kernel(const QuantParams p) {
  constexpr int HW = QT / 32;
  const int hw = threadIdx.x >> 5, t = threadIdx.x & 31;
  const int64_t first = block_index() * (HW * QU);
  Raw8<DT> raw[QU];
  int64_t row[QU];
  int v[QU];  // 8-element vector within the row
#pragma unroll
  for (int u = 0; u < QU; ++u) {
    int c;
    unit_at(p, first, u * HW + hw, row[u], c);
    v[u] = c * 32 + t;
    raw[u] = Raw8<DT>{};
    if (row[u] < p.M && v[u] * 8 < p.K)
      raw[u] = load8<DT, ALIGNED>(p.x + (row[u] * p.ldx + v[u] * 8) * elem_bytes<DT>());
  }
#pragma unroll
  for (int u = 0; u < QU; ++u) {
    float f[8];
    unpack8<DT>(raw[u], f);
    unsigned w0, w1;
    const unsigned byte = block_codes<FMT>(f, w0, w1);
    if (first + u * HW + hw >= p.units) continue;
    const bool real = row[u] < p.M && v[u] * 8 < p.K;
    if (real) store_codes<FMT>(p.codes + row[u] * (FMT == QIK_MXFP4 ? p.K / 2 : p.K), v[u], w0, w1);
    if ((t & 3) == 0) p.scales[scale_at(row[u], v[u] >> 2, p.C)] = (unsigned char)(real ? byte : 0u);
  }
}

// the values of 8 codes of MXFP4 (w0) or MXFP8 times s: exact in fp32 (a product
// below the normals, 2^-136 at least, is a subnormal with bits to spare) up to
// its overflow
template <int FMT>
__device__ __forceinline__ void values8(unsigned w0, unsigned w1, float s, float (&f)[8]) {
  f32x2 d[4];
  if constexpr (FMT == QIK_MXFP4) {
    d[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w0, 1.0f, 0);
    d[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w0, 1.0f, 1);
    d[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w0, 1.0f, 2);
    d[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w0, 1.0f, 3);
  } else {
    d[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w0, false);
    d[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w0, true);
    d[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w1, false);
    d[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w1, true);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = d[i][0] * s;
    f[2 * i + 1] = d[i][1] * s;
  }
}

// 2^(byte - 127): 0 gives the subnormal 2^-127, 255 a NaN
__device__ __forceinline__ float scale_value(unsigned byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}

// The quantiser's units over the rows themselves, each read and written whole
// (MXFP4 of 4352 x 4096 to bf16 12.2 us from memory, 3.7 TB/s; 9.3 where the 256 MB
// cache holds a part).
template <int DT, int FMT, int QU>
__global__ void __launch_bounds__(QT) dequant_kernel(const QuantParams p) {
  constexpr int HW = QT / 32;
  const int hw = threadIdx.x >> 5, t = threadIdx.x & 31;
  const int64_t first = block_index() * (HW * QU);
  unsigned w0[QU], w1[QU], byte[QU];
  int64_t at[QU];  // element offset, or -1
#pragma unroll
  for (int u = 0; u < QU; ++u) {
    int64_t row;
    int c;
    unit_at(p, first, u * HW + hw, row, c);
    const int v = c * 32 + t;
    at[u] = row < p.M && v * 8 < p.K ? row * p.K + v * 8 : -1;
    w0[u] = w1[u] = byte[u] = 0u;
    if (at[u] >= 0) {
      if constexpr (FMT == QIK_MXFP4) {
        w0[u] = *reinterpret_cast<const unsigned*>(p.codes + at[u] / 2);
      } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(p.codes + at[u]);
        w0[u] = w.x;
        w1[u] = w.y;
      }
      byte[u] = p.scales[scale_at(row, v >> 2, p.C)];
    }
  }
#pragma unroll
  for (int u = 0; u < QU; ++u) {
    if (at[u] < 0) continue;
    float f[8];
    values8<FMT>(w0[u], w1[u], scale_value(byte[u]), f);
    store8<DT, true>(p.out + at[u] * elem_bytes<DT>(), pack8<DT>(f));
  }
}

// ---------------------------------------------------------------------------
// Residual add + RMSNorm
// ---------------------------------------------------------------------------

struct NormParams {
  const char* x;
  const char* residual;
  const char* weight;
  bool weight_fp32;       // else in the element type
  char* sum;
  char* out;              // elements, or the codes
  unsigned char* scales;
  int64_t M, ldx, ldr;
  int D, C;
  double eps;
};

// v of the lane that DPP control CTRL names (0.0 where there is none, or where
// ROWS masks this lane's row of 16 off)
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_move(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)u, CTRL, ROWS, 0xf, true);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(u >> 32), CTRL, ROWS, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// the sum of v over the LANES (16 or 64) lanes of a group, in each of them:
// rotations within rows of 16, then rows 0 -> 1 and 2 -> 3, then 1 -> 2 and 3
template <int LANES>
__device__ __forceinline__ double lane_sum(double v) {
  v += dpp_move<0x128, 0xf>(v);  // row_ror:8
  v += dpp_move<0x124, 0xf>(v);
  v += dpp_move<0x122, 0xf>(v);
  v += dpp_move<0x121, 0xf>(v);
  if constexpr (LANES == 64) {
    v += dpp_move<0x142, 0xa>(v);  // row_bcast:15
    v += dpp_move<0x143, 0xc>(v);  // row_bcast:31
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)u, 63);
    const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(u >> 32), 63);
    v = __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  }
  return v;
}

// LPR threads per row, VPT vectors of 8 elements per thread: the row is read
// once and stays in registers, packed, between the sum of squares and the
// output.  The squares are summed in fp64: each is exact there, and the sum off
// by some sixty roundings of 2^-53 at most, so another order changes r only where 1
// / sqrt lies that close to the middle of two fp32 numbers, and then by one step
// of fp32.  Bound by HBM: operands from memory, bf16 4352 x 4096 with a residual
// 29.0 us (4.9 TB/s), to MXFP8 28.0 (4.5), to MXFP4 26.2 (4.4); rows at odd
// addresses go slower (fp16 9001 x 1111 15.2 us, 2.6 TB/s; 1112 wide 13.1, 3.1).
template <int DT, int FMT, bool RES, bool ALIGNED, int LPR, int VPT>
__global__ void __launch_bounds__(LPR < 256 ? 256 : LPR) norm_kernel(const NormParams p) {
#pragma clang fp contract(off)
  constexpr int NT = LPR < 256 ? 256 : LPR;
  constexpr int EB = elem_bytes<DT>();
  const int t = threadIdx.x % LPR;
  const int64_t row = block_index() * (NT / LPR) + threadIdx.x / LPR;
  if constexpr (FMT != QIK_MX_NONE) {
    // scales of padding rows (up to 32 ceil(M / 32)) and padding blocks
    if (row >= ((p.M + 31) & ~(int64_t)31)) return;
    for (int b = (row < p.M ? p.D / 32 : 0) + t; b < 8 * p.C; b += LPR) p.scales[scale_at(row, b, p.C)] = 0;
  }
  if (row >= p.M) return;  // a whole row's threads: with LPR > 64 the whole workgroup

  const char* xr = p.x + row * p.ldx * EB;
  const char* rr = RES ? p.residual + row * p.ldr * EB : nullptr;
  Raw8<DT> h[VPT];
  Raw8<DT> res[RES ? VPT : 1];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = (i * LPR + t) * 8;
    h[i] = Raw8<DT>{};
    if (e + 8 <= p.D) {
      h[i] = load8<DT, ALIGNED>(xr + e * EB);
      if constexpr (RES) res[i] = load8<DT, ALIGNED>(rr + e * EB);
    } else if (e < p.D) {
      h[i] = load_part<DT>(xr + e * EB, p.D - e);
      if constexpr (RES) res[i] = load_part<DT>(rr + e * EB, p.D - e);
    } else if constexpr (RES) {
      res[i] = Raw8<DT>{};
    }
  }
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float f[8];
    unpack8<DT>(h[i], f);
    if constexpr (RES) {
      float g[8];
      unpack8<DT>(res[i], g);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = f[k] + g[k];
      h[i] = pack8<DT>(f);
      const int e = (i * LPR + t) * 8;
      char* sr = p.sum + (row * p.D + e) * EB;
      if (e + 8 <= p.D) store8<DT, ALIGNED>(sr, h[i]);
      else if (e < p.D) store_part<DT>(sr, h[i], p.D - e);
      unpack8<DT>(h[i], f);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = __builtin_fma((double)f[k], (double)f[k], ss);
  }
  ss = lane_sum<(LPR < 64 ? LPR : 64)>(ss);
  if constexpr (LPR > 64) {
    __shared__ double part[LPR / 64];
    if ((t & 63) == 0) part[t >> 6] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int k = 0; k < LPR / 64; ++k) ss += part[k];
  }
  const float r = (float)(1.0 / sqrt(ss / (double)p.D + p.eps));

#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = (i * LPR + t) * 8;
    float f[8], w[8];
    unpack8<DT>(h[i], f);
    if (p.weight_fp32) {
      Raw8<QIK_DTYPE_FP32> raw = {};
      if (e + 8 <= p.D) raw = load8<QIK_DTYPE_FP32, ALIGNED>(p.weight + e * 4);
      else if (e < p.D) raw = load_part<QIK_DTYPE_FP32>(p.weight + e * 4, p.D - e);
      unpack8<QIK_DTYPE_FP32>(raw, w);
    } else {
      Raw8<DT> raw = {};
      if (e + 8 <= p.D) raw = load8<DT, ALIGNED>(p.weight + e * EB);
      else if (e < p.D) raw = load_part<DT>(p.weight + e * EB, p.D - e);
      unpack8<DT>(raw, w);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f[k] = f[k] * r;
      f[k] = f[k] * w[k];
    }
    if constexpr (FMT != QIK_MX_NONE) {
      // D is a multiple of 32, so a quad is all inside the row or all outside
      unsigned w0, w1;
      const unsigned byte = block_codes<FMT>(f, w0, w1);
      if (e < p.D) {
        store_codes<FMT>(reinterpret_cast<unsigned char*>(p.out) + row * (FMT == QIK_MXFP4 ? p.D / 2 : p.D), e / 8, w0, w1);
        if ((t & 3) == 0) p.scales[scale_at(row, e / 32, p.C)] = (unsigned char)byte;
      }
    } else {
      char* o = p.out + (row * p.D + e) * EB;
      const Raw8<DT> y = pack8<DT>(f);
      if (e + 8 <= p.D) store8<DT, ALIGNED>(o, y);
      else if (e < p.D) store_part<DT>(o, y, p.D - e);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

inline bool known_dtype(int32_t d) { return d == QIK_DTYPE_BF16 || d == QIK_DTYPE_FP16 || d == QIK_DTYPE_FP32; }
inline int dtype_bytes(int32_t d) { return d == QIK_DTYPE_FP32 ? 4 : 2; }
inline bool known_format(int32_t f) { return f == QIK_MXFP4 || f == QIK_MXFP8; }
inline int64_t scales_bytes(int64_t M, int64_t K) { return cdiv(M, 32) * cdiv(K, 256) * 256; }

int validate_quant(const qik_mx_quant_args* a) {
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  if (a->abi_version != QIK_ABI_VERSION || a->reserved0 != 0) return QIK_ERR_ABI_VERSION;
  if (!known_dtype(a->dtype) || !known_format(a->format)) return QIK_ERR_DTYPE;
  if (a->M < 0 || a->M > INT_MAX || a->K < 32 || a->K > MAX_K || a->K % 32 != 0) return QIK_ERR_SHAPE;
  if (a->ldx < a->K || a->ldx > ((int64_t)1 << 40)) return QIK_ERR_SHAPE;
  if (a->M == 0) return QIK_OK;
  if (a->x == nullptr || a->codes == nullptr || a->scales == nullptr) return QIK_ERR_NULL_ARG;
  if (!aligned_to(a->x, dtype_bytes(a->dtype)) || !aligned_to(a->codes, 16) || !aligned_to(a->scales, 4))
    return QIK_ERR_ALIGN;
  return QIK_OK;
}

int validate_dequant(const qik_mx_dequant_args* a) {
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  if (a->abi_version != QIK_ABI_VERSION || a->reserved0 != 0) return QIK_ERR_ABI_VERSION;
  if (!known_dtype(a->dtype) || !known_format(a->format)) return QIK_ERR_DTYPE;
  if (a->M < 0 || a->M > INT_MAX || a->K < 32 || a->K > MAX_K || a->K % 32 != 0) return QIK_ERR_SHAPE;
  if (a->M == 0) return QIK_OK;
  if (a->codes == nullptr || a->scales == nullptr || a->out == nullptr) return QIK_ERR_NULL_ARG;
  if (!aligned_to(a->codes, 16) || !aligned_to(a->scales, 4) || !aligned_to(a->out, 16)) return QIK_ERR_ALIGN;
  return QIK_OK;
}

int validate_norm(const qik_residual_rms_norm_args* a) {
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  if (a->abi_version != QIK_ABI_VERSION) return QIK_ERR_ABI_VERSION;
  if (!known_dtype(a->dtype) || (a->format != QIK_MX_NONE && !known_format(a->format))) return QIK_ERR_DTYPE;
  if (a->weight_dtype != QIK_DTYPE_FP32 && a->weight_dtype != a->dtype) return QIK_ERR_DTYPE;
  if (a->M < 0 || a->M > INT_MAX || a->D < 1 || a->D > 32768) return QIK_ERR_SHAPE;
  if (a->format != QIK_MX_NONE && a->D % 32 != 0) return QIK_ERR_SHAPE;
  if (a->ldx < a->D || a->ldx > ((int64_t)1 << 40)) return QIK_ERR_SHAPE;
  if ((a->residual == nullptr) != (a->sum == nullptr)) return QIK_ERR_NULL_ARG;
  if (a->residual != nullptr && (a->ldr < a->D || a->ldr > ((int64_t)1 << 40))) return QIK_ERR_SHAPE;
  if (a->M == 0) return QIK_OK;
  if (a->x == nullptr || a->weight == nullptr || a->out == nullptr) return QIK_ERR_NULL_ARG;
  if (a->format != QIK_MX_NONE && a->scales == nullptr) return QIK_ERR_NULL_ARG;
  const int eb = dtype_bytes(a->dtype);
  if (!aligned_to(a->x, eb) || !aligned_to(a->residual, eb) || !aligned_to(a->sum, eb) ||
      !aligned_to(a->weight, dtype_bytes(a->weight_dtype)))
    return QIK_ERR_ALIGN;
  if (!aligned_to(a->out, a->format == QIK_MX_NONE ? eb : 16) || !aligned_to(a->scales, 4)) return QIK_ERR_ALIGN;
  return QIK_OK;
}

int launch(const void* fn, int64_t grid, int threads, void* params, hipStream_t s) {
  unsigned gx, gy;  // the surplus workgroups are behind the last row of the data
  if (!qik_host::split_grid(grid, threads, &gx, &gy)) return QIK_ERR_SHAPE;
  void* args[] = {params};
  return hipLaunchKernel(fn, dim3(gx, gy), dim3((unsigned)threads), args, 0, s) == hipSuccess ? QIK_OK : QIK_ERR_LAUNCH;
}

QuantParams unit_params(int64_t M, int64_t K, int64_t rows) {
  QuantParams p;
  memset(&p, 0, sizeof(p));
  p.M = M;
  p.K = (int)K;
  p.C = (int)cdiv(K, 256);
  p.units = rows * p.C;
  p.magic = p.C == 1 ? 0u : (unsigned)((((uint64_t)1 << 32) + p.C - 1) / p.C);
  return p;
}

// units from which a half wave takes two (quant_kernel)
constexpr int64_t TWO_UNITS = 65536;

template <int DT, int FMT>
const void* quant_fn(bool al, int qu) {
  if (DT != QIK_DTYPE_FP32 && qu == 2)
    return al ? (const void*)quant_kernel<DT, FMT, true, 2> : (const void*)quant_kernel<DT, FMT, false, 2>;
  return al ? (const void*)quant_kernel<DT, FMT, true, 1> : (const void*)quant_kernel<DT, FMT, false, 1>;
}

template <int DT>
int launch_quant(const qik_mx_quant_args* a, hipStream_t s) {
  QuantParams p = unit_params(a->M, a->K, cdiv(a->M, 32) * 32);
  p.x = static_cast<const char*>(a->x);
  p.codes = static_cast<unsigned char*>(a->codes);
  p.scales = static_cast<unsigned char*>(a->scales);
  p.ldx = a->ldx;
  const bool al = aligned_to(a->x, 16) && (a->M == 1 || a->ldx * elem_bytes<DT>() % 16 == 0);
  const int qu = DT != QIK_DTYPE_FP32 && p.units >= TWO_UNITS ? 2 : 1;
  const void* fn = a->format == QIK_MXFP4 ? quant_fn<DT, QIK_MXFP4>(al, qu) : quant_fn<DT, QIK_MXFP8>(al, qu);
  return launch(fn, cdiv(p.units, QT / 32 * qu), QT, &p, s);
}

template <int DT>
int launch_dequant(const qik_mx_dequant_args* a, hipStream_t s) {
  QuantParams p = unit_params(a->M, a->K, a->M);
  p.codes = static_cast<unsigned char*>(const_cast<void*>(a->codes));
  p.scales = static_cast<unsigned char*>(const_cast<void*>(a->scales));
  p.out = static_cast<char*>(a->out);
  const bool two = p.units >= TWO_UNITS;
  const void* fn = a->format == QIK_MXFP4
                       ? (two ? (const void*)dequant_kernel<DT, QIK_MXFP4, 2> : (const void*)dequant_kernel<DT, QIK_MXFP4, 1>)
                       : (two ? (const void*)dequant_kernel<DT, QIK_MXFP8, 2> : (const void*)dequant_kernel<DT, QIK_MXFP8, 1>);
  return launch(fn, cdiv(p.units, QT / 32 * (two ? 2 : 1)), QT, &p, s);
}

template <int DT, int FMT, bool RES, bool ALIGNED, int LPR, int VPT>
int launch_norm_shape(const NormParams& p0, hipStream_t s) {
  NormParams p = p0;
  const int64_t rows = FMT == QIK_MX_NONE ? p.M : cdiv(p.M, 32) * 32;
  constexpr int NT = LPR < 256 ? 256 : LPR;
  return launch((const void*)norm_kernel<DT, FMT, RES, ALIGNED, LPR, VPT>, cdiv(rows, NT / LPR), NT, &p, s);
}

// The fewest lanes that hold a row in at most 64 bytes a lane of x (a wave of
// its own needs no barrier; fp32 2048 wide 26.5 us with 256 lanes of one vector
// against 30.5 with 64 of four, 5000 rows; bf16 4096 wide 29.1 with 256 of two
// against 33.6 with 64 of eight), 16 of a wave for rows up to 256 (16384 rows of
// 128 4.9 us against 10.3 with a wave each).
template <int DT, int FMT, bool RES, bool ALIGNED>
int launch_norm(const NormParams& p, hipStream_t s) {
  if (p.D <= 128) return launch_norm_shape<DT, FMT, RES, ALIGNED, 16, 1>(p, s);
  if (p.D <= 256) return launch_norm_shape<DT, FMT, RES, ALIGNED, 16, 2>(p, s);
  if (p.D <= 512) return launch_norm_shape<DT, FMT, RES, ALIGNED, 64, 1>(p, s);
  if (p.D <= 1024) return launch_norm_shape<DT, FMT, RES, ALIGNED, 64, 2>(p, s);
  if constexpr (DT != QIK_DTYPE_FP32) {
    if (p.D <= 1536) return launch_norm_shape<DT, FMT, RES, ALIGNED, 64, 3>(p, s);
    if (p.D <= 2048) return launch_norm_shape<DT, FMT, RES, ALIGNED, 64, 4>(p, s);
  } else {
    if (p.D <= 2048) return launch_norm_shape<DT, FMT, RES, ALIGNED, 256, 1>(p, s);
  }
  if (p.D <= 4096) return launch_norm_shape<DT, FMT, RES, ALIGNED, 256, 2>(p, s);
  if (p.D <= 6144) return launch_norm_shape<DT, FMT, RES, ALIGNED, 256, 3>(p, s);
  if (p.D <= 8192) return launch_norm_shape<DT, FMT, RES, ALIGNED, 256, 4>(p, s);
  return launch_norm_shape<DT, FMT, RES, ALIGNED, 1024, 4>(p, s);
}

template <int DT>
int launch_norm_format(const qik_residual_rms_norm_args* a, hipStream_t s) {
  NormParams p;
  memset(&p, 0, sizeof(p));
  p.x = static_cast<const char*>(a->x);
  p.residual = static_cast<const char*>(a->residual);
  p.weight = static_cast<const char*>(a->weight);
  p.weight_fp32 = a->weight_dtype == QIK_DTYPE_FP32;
  p.sum = static_cast<char*>(a->sum);
  p.out = static_cast<char*>(a->out);
  p.scales = static_cast<unsigned char*>(a->scales);
  p.M = a->M;
  p.ldx = a->ldx;
  p.ldr = a->ldr;
  p.D = (int)a->D;
  p.C = (int)cdiv(a->D, 256);
  p.eps = a->eps;
  // every row of x, residual, sum and an out of elements, and the weight, starts at a multiple of 16 bytes
  const int EB = elem_bytes<DT>();
  auto rows_aligned = [&](const void* ptr, int64_t ld) {
    return aligned_to(ptr, 16) && (a->M == 1 || ld * EB % 16 == 0);
  };
  const bool al = rows_aligned(a->x, a->ldx) && aligned_to(a->weight, 16) &&
                  (a->residual == nullptr || (rows_aligned(a->residual, a->ldr) && rows_aligned(a->sum, a->D))) &&
                  (a->format != QIK_MX_NONE || rows_aligned(a->out, a->D));
  const bool res = a->residual != nullptr;
  switch (a->format) {
    case QIK_MX_NONE:
      if (al) return res ? launch_norm<DT, QIK_MX_NONE, true, true>(p, s) : launch_norm<DT, QIK_MX_NONE, false, true>(p, s);
      return res ? launch_norm<DT, QIK_MX_NONE, true, false>(p, s) : launch_norm<DT, QIK_MX_NONE, false, false>(p, s);
    case QIK_MXFP4:
      if (!al) return QIK_ERR_ALIGN;
      return res ? launch_norm<DT, QIK_MXFP4, true, true>(p, s) : launch_norm<DT, QIK_MXFP4, false, true>(p, s);
    default:
      if (!al) return QIK_ERR_ALIGN;
      return res ? launch_norm<DT, QIK_MXFP8, true, true>(p, s) : launch_norm<DT, QIK_MXFP8, false, true>(p, s);
  }
}

// ---------------------------------------------------------------------------
// Quantiser of rows in host memory (no device involved)
// ---------------------------------------------------------------------------

// E2M1 code of q (|q| below 8), round to nearest even, saturated at 6.  The
// magnitude's grid is 0.5 below 2, 1 below 4, 2 above.
inline unsigned host_e2m1(float q) {
  uint32_t u;
  memcpy(&u, &q, 4);
  const unsigned sign = (u >> 28) & 8u;
  const float a = std::min(std::fabs(q), 6.0f);
  const float step = a < 2.0f ? 0.5f : a < 4.0f ? 1.0f : 2.0f;
  const int h = (int)(std::nearbyint(a / step) * step * 2.0f);  // twice the magnitude: 0 1 2 3 4 6 8 12
  return sign | (unsigned)(h < 4 ? h : h < 8 ? 2 + h / 2 : 4 + h / 4);
}

void host_rows(const qik_mx_quant_args* a, int64_t m0, int64_t m1) {
  const int64_t C = cdiv(a->K, 256);
  const char* x = static_cast<const char*>(a->x);
  unsigned char* codes = static_cast<unsigned char*>(a->codes);
  unsigned char* scales = static_cast<unsigned char*>(a->scales);
  const bool fp4 = a->format == QIK_MXFP4;
  for (int64_t m = m0; m < m1; ++m) {
    const void* row = x + m * a->ldx * dtype_bytes(a->dtype);
    unsigned char* out = codes + m * (fp4 ? a->K / 2 : a->K);
    for (int64_t b = 0; b < a->K / 32; ++b) {
      float f[32];
      uint32_t top = 0;
      for (int i = 0; i < 32; ++i) {
        f[i] = qik_host::host_elem(row, a->dtype, b * 32 + i);
        uint32_t u;
        memcpy(&u, &f[i], 4);
        top = std::max(top, u & 0x7fffffffu);
      }
      const uint32_t E = top >> 23, em = fp4 ? 2 : 8;
      const uint32_t byte = E == 255 ? 255 : E > em ? E - em : 0;
      scales[((m / 32) * C + b / 8) * 256 + (m % 32) * 8 + b % 8] = (unsigned char)byte;
      for (int i = 0; i < 32; ++i) {
        unsigned code = 0;
        if (byte != 255) {
          const float q = std::ldexp(f[i], 127 - (int)byte);
          code = fp4 ? host_e2m1(q) : qik_host::host_e4m3fn(std::min(std::max(q, -448.0f), 448.0f));
        }
        if (!fp4) out[b * 32 + i] = (unsigned char)code;
        else if (i % 2 == 0) out[b * 16 + i / 2] = (unsigned char)code;
        else out[b * 16 + i / 2] |= (unsigned char)(code << 4);
      }
    }
  }
}

}  // namespace qik_mx

extern "C" {

int qik_mx_scales_size(int64_t M, int64_t K, int64_t* bytes) {
  if (bytes == nullptr) return QIK_ERR_NULL_ARG;
  *bytes = 0;
  if (M < 0 || M > INT_MAX || K < 32 || K % 32 != 0 || K > qik_mx::MAX_K) return QIK_ERR_SHAPE;
  *bytes = qik_mx::scales_bytes(M, K);
  return QIK_OK;
}

int qik_mx_quantize(const qik_mx_quant_args* a, void* stream) {
  using namespace qik_mx;
  const int st = validate_quant(a);
  if (st != QIK_OK || a->M == 0) return st;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case QIK_DTYPE_BF16: return launch_quant<QIK_DTYPE_BF16>(a, s);
    case QIK_DTYPE_FP16: return launch_quant<QIK_DTYPE_FP16>(a, s);
    default: return launch_quant<QIK_DTYPE_FP32>(a, s);
  }
}

int qik_mx_quantize_host(const qik_mx_quant_args* a, int32_t threads) {
  using namespace qik_mx;
  const int st = validate_quant(a);
  if (st != QIK_OK || a->M == 0) return st;
  memset(a->scales, 0, (size_t)scales_bytes(a->M, a->K));
  // rows that share a 32-row group of scales write different bytes of it
  const int64_t nt = std::max<int64_t>(1, std::min<int64_t>({(int64_t)threads, a->M, a->M * a->K / 65536 + 1}));
  try {
    std::vector<std::thread> pool;
    for (int64_t t = 1; t < nt; ++t) {
      try {
        pool.emplace_back(host_rows, a, a->M * t / nt, a->M * (t + 1) / nt);
      } catch (...) {  // no thread to be had: this one does its rows
        host_rows(a, a->M * t / nt, a->M * (t + 1) / nt);
      }
    }
    host_rows(a, 0, a->M / nt);
    for (auto& th : pool) th.join();
  } catch (...) {
    return QIK_ERR_LAUNCH;
  }
  return QIK_OK;
}

int qik_mx_dequantize(const qik_mx_dequant_args* a, void* stream) {
  using namespace qik_mx;
  const int st = validate_dequant(a);
  if (st != QIK_OK || a->M == 0) return st;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case QIK_DTYPE_BF16: return launch_dequant<QIK_DTYPE_BF16>(a, s);
    case QIK_DTYPE_FP16: return launch_dequant<QIK_DTYPE_FP16>(a, s);
    default: return launch_dequant<QIK_DTYPE_FP32>(a, s);
  }
}

int qik_residual_rms_norm(const qik_residual_rms_norm_args* a, void* stream) {
  using namespace qik_mx;
  const int st = validate_norm(a);
  if (st != QIK_OK || a->M == 0) return st;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case QIK_DTYPE_BF16: return launch_norm_format<QIK_DTYPE_BF16>(a, s);
    case QIK_DTYPE_FP16: return launch_norm_format<QIK_DTYPE_FP16>(a, s);
    default: return launch_norm_format<QIK_DTYPE_FP32>(a, s);
  }
}

}  // extern "C"
