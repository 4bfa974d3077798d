// Product of microscaled operands on MI355X (gfx950): A in MXFP4 or MXFP8, W in
// MXFP4, on the scaled matrix instructions v_mfma_scale_f32_*_f8f6f4, which
// multiply each block of 32 by its two power-of-two scales as they sum it.
//
// Few rows (`rows_kernel`): every wave takes 16 weight rows and a share of K,
// loads the codes straight into registers and meets the others of its
// workgroup in LDS.  It is bound by the weight's bytes.

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include <limits.h>
#include <algorithm>

#include "qik_mx.h"

namespace qik_mx {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int FMT_E4M3 = 0, FMT_E2M1 = 4;  // the instruction's operand formats

struct MxGemmParams {
  const unsigned char* a;
  const unsigned char* as;
  const unsigned char* w;
  const unsigned char* ws;
  const char* bias;
  char* out;
  int M, N, K, C;  // C = ceil(K / 256)
  int64_t lda, ldw, ldc;
};

template <bool FP16>
__device__ __forceinline__ unsigned short round16(float f) {
  asm volatile("" : "+v"(f));  // an fp32 value: no mixed-precision fma rounds it
  if constexpr (FP16) return __builtin_bit_cast(unsigned short, (_Float16)f);
  else return __builtin_bit_cast(unsigned short, (__bf16)f);
}
template <bool FP16>
__device__ __forceinline__ float widen16(unsigned short h) {
  if constexpr (FP16) return (float)__builtin_bit_cast(_Float16, h);
  else return __uint_as_float((unsigned)h << 16);
}

__device__ __forceinline__ i32x8 operand(u32x4 lo, u32x4 hi) {
  return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// ---------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------
//
// 16x16x128: lane l of the wave holds row l % 16 of an operand.  Of an E2M1
// operand it holds k = 32 (l / 16) .. + 31 of the step; of an E4M3 operand k =
// 16 (l / 16) .. + 15 and 64 + 16 (l / 16) .. + 15; in both its scale is that
// of block l / 16 of the step.  W is the first operand, so a lane's 4 sums are
// 4 consecutive columns n of row m = l % 16.

constexpr int RK = 4;  // waves of a workgroup, each with its share of the 256-k chunks

template <bool A8, int MB, int NB, bool FP16>
__global__ void __launch_bounds__(64 * RK) rows_kernel(const MxGemmParams p) {
  __shared__ f32x4 red[RK][NB * MB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * NB), m0 = blockIdx.y * (16 * MB);

  // rows past the end repeat the last one; their sums are not stored
  const unsigned char* wr[NB];
  const unsigned char* wsr[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int n = min(n0 + j * 16 + r, p.N - 1);
    wr[j] = p.w + n * p.ldw;
    wsr[j] = p.ws + (int64_t)(n >> 5) * p.C * 256 + (n & 31) * 8;
  }
  const unsigned char* ar[MB];
  const unsigned char* asr[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int m = min(m0 + i * 16 + r, p.M - 1);
    ar[i] = p.a + m * p.lda;
    asr[i] = p.as + (int64_t)(m >> 5) * p.C * 256 + (m & 31) * 8;
  }

  f32x4 acc[NB][MB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int c0 = p.C * wave / RK, c1 = p.C * (wave + 1) / RK;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int c = c0; c < c1; ++c) {
    u32x2 wsc[NB], asc[MB];
    u32x4 wf[2][NB], af[2][MB][A8 ? 2 : 1];
#pragma unroll
    for (int j = 0; j < NB; ++j) wsc[j] = *reinterpret_cast<const u32x2*>(wsr[j] + c * 256);
#pragma unroll
    for (int i = 0; i < MB; ++i) asc[i] = *reinterpret_cast<const u32x2*>(asr[i] + c * 256);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      // a lane's blocks past K are zeros (loaded from the row's start, then cleared)
      const int k = c * 256 + s * 128 + g * 32;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(wr[j] + (k < p.K ? k / 2 : 0));
        wf[s][j] = k < p.K ? v : zero;
      }
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        if constexpr (A8) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int ka = c * 256 + s * 128 + h * 64 + g * 16;
            const u32x4 v = *reinterpret_cast<const u32x4*>(ar[i] + (ka < p.K ? ka : 0));
            af[s][i][h] = ka < p.K ? v : zero;
          }
        } else {
          const u32x4 v = *reinterpret_cast<const u32x4*>(ar[i] + (k < p.K ? k / 2 : 0));
          af[s][i][0] = k < p.K ? v : zero;
        }
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
          acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              operand(wf[s][j], zero), operand(af[s][i][0], A8 ? af[s][i][A8 ? 1 : 0] : zero), acc[j][i], FMT_E2M1,
              A8 ? FMT_E4M3 : FMT_E2M1, 0, (int)(wsc[j][s] >> (8 * g)), 0, (int)(asc[i][s] >> (8 * g)));
  }
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) red[wave][j * MB + i][lane] = acc[j][i];
  __syncthreads();
  for (int e = threadIdx.x; e < NB * MB * 256; e += 64 * RK) {
    const int nl = e % (16 * NB), ml = e / (16 * NB);
    const int n = n0 + nl, m = m0 + ml;
    if (n >= p.N || m >= p.M) continue;
    const int tile = (nl / 16) * MB + ml / 16, ln = (nl % 16) / 4 * 16 + ml % 16;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < RK; ++k) y += red[k][tile][ln][nl % 4];  // the shares in order
    if (p.bias != nullptr) y += widen16<FP16>(reinterpret_cast<const unsigned short*>(p.bias)[n]);
    reinterpret_cast<unsigned short*>(p.out)[m * p.ldc + n] = round16<FP16>(y);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

inline bool aligned_to(const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) % a) == 0; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// with_a: a, a_scales and lda are checked too
int validate_gemm(const qik_mx_gemm_args* a, bool with_a) {
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  if (a->abi_version != QIK_ABI_VERSION || a->reserved0 != 0) return QIK_ERR_ABI_VERSION;
  if (a->out_dtype != QIK_DTYPE_BF16 && a->out_dtype != QIK_DTYPE_FP16) return QIK_ERR_DTYPE;
  if (a->a_format != QIK_MXFP4 && a->a_format != QIK_MXFP8) return QIK_ERR_DTYPE;
  if (a->M < 0 || a->M > INT_MAX || a->N < 1 || a->N > INT_MAX) return QIK_ERR_SHAPE;
  if (a->K < 32 || a->K > 262144 || a->K % 32 != 0) return QIK_ERR_SHAPE;
  const int64_t row_a = a->a_format == QIK_MXFP4 ? a->K / 2 : a->K;
  // a tile's rows must be addressable by a 31-bit buffer offset
  if (a->ldw < a->K / 2 || a->ldw > INT_MAX / 256 || a->ldc < a->N || a->ldc > ((int64_t)1 << 40)) return QIK_ERR_SHAPE;
  if (with_a && (a->lda < row_a || a->lda > INT_MAX / 256)) return QIK_ERR_SHAPE;
  if (a->M == 0) return QIK_OK;
  if (a->w == nullptr || a->w_scales == nullptr || a->out == nullptr) return QIK_ERR_NULL_ARG;
  if (!aligned_to(a->w, 16) || !aligned_to(a->w_scales, 16) || a->ldw % 16 != 0) return QIK_ERR_ALIGN;
  if (!aligned_to(a->out, 2) || !aligned_to(a->bias, 2)) return QIK_ERR_ALIGN;
  if (with_a) {
    if (a->a == nullptr || a->a_scales == nullptr) return QIK_ERR_NULL_ARG;
    if (!aligned_to(a->a, 16) || !aligned_to(a->a_scales, 16) || a->lda % 16 != 0) return QIK_ERR_ALIGN;
  }
  return QIK_OK;
}

int validate_linear(const qik_mx_linear_args* a) {
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  const int st = validate_gemm(&a->g, false);
  if (st != QIK_OK) return st;
  if (a->reserved0 != 0) return QIK_ERR_ABI_VERSION;
  if (a->x_dtype != QIK_DTYPE_BF16 && a->x_dtype != QIK_DTYPE_FP16 && a->x_dtype != QIK_DTYPE_FP32) return QIK_ERR_DTYPE;
  if (a->ldx < a->g.K || a->ldx > ((int64_t)1 << 40)) return QIK_ERR_SHAPE;
  if (a->g.M == 0) return QIK_OK;
  if (a->x == nullptr) return QIK_ERR_NULL_ARG;
  return aligned_to(a->x, a->x_dtype == QIK_DTYPE_FP32 ? 4 : 2) ? QIK_OK : QIK_ERR_ALIGN;
}

MxGemmParams gemm_params(const qik_mx_gemm_args* a) {
  MxGemmParams p;
  memset(&p, 0, sizeof(p));
  p.a = static_cast<const unsigned char*>(a->a);
  p.as = static_cast<const unsigned char*>(a->a_scales);
  p.w = static_cast<const unsigned char*>(a->w);
  p.ws = static_cast<const unsigned char*>(a->w_scales);
  p.bias = static_cast<const char*>(a->bias);
  p.out = static_cast<char*>(a->out);
  p.M = (int)a->M;
  p.N = (int)a->N;
  p.K = (int)a->K;
  p.C = (int)cdiv(a->K, 256);
  p.lda = a->lda;
  p.ldw = a->ldw;
  p.ldc = a->ldc;
  return p;
}

template <bool A8, bool FP16>
int launch_rows(MxGemmParams& p, hipStream_t s) {
  const int64_t gy = cdiv(p.M, 16);
  if (gy > 65535) return QIK_ERR_SHAPE;
  void* args[] = {&p};
  return hipLaunchKernel((const void*)rows_kernel<A8, 1, 1, FP16>, dim3((unsigned)cdiv(p.N, 16), (unsigned)gy),
                         dim3(64 * RK), args, 0, s) == hipSuccess
             ? QIK_OK
             : QIK_ERR_LAUNCH;
}

int launch_gemm(const qik_mx_gemm_args* a, hipStream_t s) {
  MxGemmParams p = gemm_params(a);
  const bool fp16 = a->out_dtype == QIK_DTYPE_FP16;
  if (a->a_format == QIK_MXFP8) return fp16 ? launch_rows<true, true>(p, s) : launch_rows<true, false>(p, s);
  return fp16 ? launch_rows<false, true>(p, s) : launch_rows<false, false>(p, s);
}

inline int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// bytes of x's codes and scales in a linear's workspace
int64_t code_bytes(const qik_mx_gemm_args* g) { return round256(g->M * (g->a_format == QIK_MXFP4 ? g->K / 2 : g->K)); }
int64_t scale_bytes(const qik_mx_gemm_args* g) { return cdiv(g->M, 32) * cdiv(g->K, 256) * 256; }

}  // namespace qik_mx

extern "C" {

int qik_mx_gemm_workspace_size(const qik_mx_gemm_args* a, int64_t* bytes) {
  if (bytes == nullptr) return QIK_ERR_NULL_ARG;
  *bytes = 0;
  return qik_mx::validate_gemm(a, true);
}

int qik_mx_gemm(const qik_mx_gemm_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace qik_mx;
  const int st = validate_gemm(a, true);
  if (st != QIK_OK || a->M == 0) return st;
  (void)workspace;
  (void)workspace_bytes;
  return launch_gemm(a, static_cast<hipStream_t>(stream));
}

int qik_mx_linear_workspace_size(const qik_mx_linear_args* a, int64_t* bytes) {
  using namespace qik_mx;
  if (bytes == nullptr) return QIK_ERR_NULL_ARG;
  *bytes = 0;
  const int st = validate_linear(a);
  if (st != QIK_OK) return st;
  *bytes = code_bytes(&a->g) + scale_bytes(&a->g);
  return QIK_OK;
}

int qik_mx_linear(const qik_mx_linear_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace qik_mx;
  const int st = validate_linear(a);
  if (st != QIK_OK || a->g.M == 0) return st;
  int64_t need = 0;
  qik_mx_linear_workspace_size(a, &need);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 256))) return QIK_ERR_WORKSPACE;
  qik_mx_gemm_args g = a->g;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  g.a = ws;
  g.a_scales = ws + code_bytes(&g);
  g.lda = g.a_format == QIK_MXFP4 ? g.K / 2 : g.K;
  qik_mx_quant_args q;
  memset(&q, 0, sizeof(q));
  q.abi_version = QIK_ABI_VERSION;
  q.dtype = a->x_dtype;
  q.format = g.a_format;
  q.x = a->x;
  q.codes = ws;
  q.scales = ws + code_bytes(&g);
  q.M = g.M;
  q.K = g.K;
  q.ldx = a->ldx;
  const int qs = qik_mx_quantize(&q, stream);
  if (qs != QIK_OK) return qs;
  return launch_gemm(&g, static_cast<hipStream_t>(stream));
}

}  // extern "C"
