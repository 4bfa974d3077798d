// RMSNorm over each head and the rotation by positions on several axes, of a
// layer's Q and K in one launch, and its gradient (include/qik_rope.h).
//
// A byte mover: every row is read and written once.  What it must not do is
// take a sine per element: the D / 2 angles of a token are the same for all its
// heads, in Q and in K.  So rows are numbered token by token, the heads of Q and
// then those of K; a workgroup takes a run of rows, its threads first issue the
// loads of all of them, then compute the cosines and sines of the few tokens
// that the run touches into LDS, and then turn the rows.  D / 8 lanes hold a row,
// a lane the pairs 4t .. 4t + 3: eight neighbouring elements, or four of each half.

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include <limits.h>
#include <algorithm>

#include "qik_rope.h"
#include "qik_mx_block.h"
#include "qik_attn_launch.h"

namespace qik_rope {

using qik_mx::Raw8;
using qik_mx::u32x2;
using qik_mx::u32x4;

constexpr int THREADS = 256;
constexpr int UNITS = 4;            // rows of a lane group, their loads issued together
// backward: workgroups at most, each with a [2, D] sum of dw in the workspace
constexpr int BWD_GRID = 512;

struct Tensor {
  const char* x;
  const char* dy;
  char* out;                        // y, or dx
  const float* w;
  int64_t sx[3], so[3], sdy[3];     // b, s, h in bytes
  int H;
  float eps;
};

struct Params {
  Tensor t[2];
  const double* pos;
  const double* freq;
  const int32_t* axis;
  int64_t pos_b, pos_a;
  float* part;                      // backward: [grid][2][D]
  int rows;                         // B * S * (H of both)
  int S, heads;
  int runs;                         // runs of rows: workgroups of the forward launch
};

template <int D>
constexpr int run_rows() { return THREADS / (D / 8) * UNITS; }

// the lane's eight elements of a row: pairs 4t .. 4t + 3, in order
template <int D, bool FP16, bool HALVES>
__device__ __forceinline__ u32x4 load_pairs(const char* row, int t) {
  if constexpr (HALVES) {
    const u32x2 a = *reinterpret_cast<const u32x2*>(row + t * 8);
    const u32x2 b = *reinterpret_cast<const u32x2*>(row + D + t * 8);
    return u32x4{a.x, a.y, b.x, b.y};
  } else {
    return *reinterpret_cast<const u32x4*>(row + t * 16);
  }
}
template <int D, bool HALVES>
__device__ __forceinline__ void store_pairs(char* row, int t, u32x4 v) {
  if constexpr (HALVES) {
    *reinterpret_cast<u32x2*>(row + t * 8) = u32x2{v.x, v.y};
    *reinterpret_cast<u32x2*>(row + D + t * 8) = u32x2{v.z, v.w};
  } else {
    *reinterpret_cast<u32x4*>(row + t * 16) = v;
  }
}
// where element e of the lane (0 .. 7, as load_pairs gives them) lies in the row
template <int D, bool HALVES>
__device__ __forceinline__ int element_of(int t, int e) {
  return HALVES ? (e < 4 ? 4 * t + e : D / 2 + 4 * t + e - 4) : 8 * t + e;
}
// the two elements of the lane's pair i
template <bool HALVES>
constexpr int first_of(int i) { return HALVES ? i : 2 * i; }
template <bool HALVES>
constexpr int second_of(int i) { return HALVES ? i + 4 : 2 * i + 1; }

template <int TPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int k = TPR / 2; k >= 1; k >>= 1) v += __shfl_xor(v, k);
  return v;
}

// a row of the run: its tensor, and where it lies
struct Row {
  int which, token, b, s, h;
};
__device__ __forceinline__ Row row_of(const Params& p, int row) {
  Row r;
  r.token = (int)((unsigned)row / (unsigned)p.heads);
  const int h = row - r.token * p.heads;
  r.which = h >= p.t[0].H ? 1 : 0;
  r.h = r.which ? h - p.t[0].H : h;
  r.b = (int)((unsigned)r.token / (unsigned)p.S);
  r.s = r.token - r.b * p.S;
  return r;
}

// cosines and sines of the tokens [first, first + n) into cs [n][D / 2]
template <int D>
__device__ __forceinline__ void turn_table(const Params& p, int first, int n, float2* cs) {
  for (int i = (int)threadIdx.x; i < n * (D / 2); i += THREADS) {
    const int pair = i % (D / 2), token = first + i / (D / 2);
    const int b = (int)((unsigned)token / (unsigned)p.S), s = token - b * p.S;
    const double turns = p.pos[b * p.pos_b + p.axis[pair] * p.pos_a + s] * p.freq[pair];
    float sn, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &c);
    cs[i] = make_float2(c, sn);
  }
}

template <int D, bool FP16, bool HALVES, bool NORM>
__global__ void __launch_bounds__(THREADS) axial_rope_kernel(const Params p) {
  constexpr int DT = FP16 ? QIK_DTYPE_FP16 : QIK_DTYPE_BF16;
  constexpr int TPR = D / 8, RPB = THREADS / TPR;
  extern __shared__ float2 cs[];
  const int t = (int)threadIdx.x % TPR;
  const int row0 = (int)blockIdx.x * run_rows<D>() + (int)threadIdx.x / TPR;
  const int first = (int)((unsigned)((int)blockIdx.x * run_rows<D>()) / (unsigned)p.heads);
  const int last = (int)((unsigned)min((int)blockIdx.x * run_rows<D>() + run_rows<D>() - 1, p.rows - 1) / (unsigned)p.heads);
  u32x4 raw[UNITS];
  Row r[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    r[u] = row_of(p, min(row0 + u * RPB, p.rows - 1));
    const Tensor& x = p.t[r[u].which];
    raw[u] = load_pairs<D, FP16, HALVES>(x.x + r[u].b * x.sx[0] + r[u].s * x.sx[1] + r[u].h * x.sx[2], t);
  }
  turn_table<D>(p, first, last - first + 1, cs);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    float x[8];
    qik_mx::unpack8<DT>(Raw8<DT>{{raw[u]}}, x);
    const Tensor& tn = p.t[r[u].which];
    if constexpr (NORM) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(x[e], x[e], ss);
      const float rs = 1.0f / sqrtf(row_sum<TPR>(ss) * (1.0f / D) + tn.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (x[e] * rs) * tn.w[element_of<D, HALVES>(t, e)];
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 c = cs[(r[u].token - first) * (D / 2) + 4 * t + i];
      const float a = x[first_of<HALVES>(i)], b = x[second_of<HALVES>(i)];
      y[first_of<HALVES>(i)] = a * c.x - b * c.y;
      y[second_of<HALVES>(i)] = a * c.y + b * c.x;
    }
    if (row0 + u * RPB < p.rows)
      store_pairs<D, HALVES>(tn.out + r[u].b * tn.so[0] + r[u].s * tn.so[1] + r[u].h * tn.so[2], t, qik_mx::pack8<DT>(y).w[0]);
  }
}

// The gradient: as above with dy beside x; a workgroup takes every gridDim.x-th
// run and keeps its rows' sums of dw in registers, which become one [2, D] sum in
// the workspace at its end.
template <int D, bool FP16, bool HALVES, bool NORM>
__global__ void __launch_bounds__(THREADS) axial_rope_bwd_kernel(const Params p) {
  constexpr int DT = FP16 ? QIK_DTYPE_FP16 : QIK_DTYPE_BF16;
  constexpr int TPR = D / 8, RPB = THREADS / TPR;
  extern __shared__ float2 cs[];
  const int t = (int)threadIdx.x % TPR;
  float dw[2][8] = {};
  for (int run = (int)blockIdx.x; run < p.runs; run += (int)gridDim.x) {
    const int base = run * run_rows<D>();
    const int row0 = base + (int)threadIdx.x / TPR;
    const int first = (int)((unsigned)base / (unsigned)p.heads);
    const int last = (int)((unsigned)min(base + run_rows<D>() - 1, p.rows - 1) / (unsigned)p.heads);
    u32x4 raw[UNITS], gr[UNITS];
    Row r[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      r[u] = row_of(p, min(row0 + u * RPB, p.rows - 1));
      const Tensor& x = p.t[r[u].which];
      gr[u] = load_pairs<D, FP16, HALVES>(x.dy + r[u].b * x.sdy[0] + r[u].s * x.sdy[1] + r[u].h * x.sdy[2], t);
      if constexpr (NORM) raw[u] = load_pairs<D, FP16, HALVES>(x.x + r[u].b * x.sx[0] + r[u].s * x.sx[1] + r[u].h * x.sx[2], t);
    }
    __syncthreads();  // the last run's table has been read
    turn_table<D>(p, first, last - first + 1, cs);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const bool live = row0 + u * RPB < p.rows;
      float g[8], dn[8];
      qik_mx::unpack8<DT>(Raw8<DT>{{gr[u]}}, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 c = cs[(r[u].token - first) * (D / 2) + 4 * t + i];
        const float a = g[first_of<HALVES>(i)], b = g[second_of<HALVES>(i)];
        dn[first_of<HALVES>(i)] = a * c.x + b * c.y;
        dn[second_of<HALVES>(i)] = b * c.x - a * c.y;
      }
      const Tensor& tn = p.t[r[u].which];
      if constexpr (NORM) {
        float x[8];
        qik_mx::unpack8<DT>(Raw8<DT>{{raw[u]}}, x);
        float ss = 0.0f, dot = 0.0f;
        float wd[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          wd[e] = dn[e] * tn.w[element_of<D, HALVES>(t, e)];
          ss = __builtin_fmaf(x[e], x[e], ss);
          dot = __builtin_fmaf(x[e], wd[e], dot);
        }
        const float rs = 1.0f / sqrtf(row_sum<TPR>(ss) * (1.0f / D) + tn.eps);
        const float pull = row_sum<TPR>(dot) * (1.0f / D) * rs * rs;  // mean(x w dn) r^2
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float add = live ? dn[e] * (x[e] * rs) : 0.0f;
          dw[0][e] += r[u].which ? 0.0f : add;
          dw[1][e] += r[u].which ? add : 0.0f;
          dn[e] = rs * __builtin_fmaf(-x[e], pull, wd[e]);
        }
      }
      if (live)
        store_pairs<D, HALVES>(tn.out + r[u].b * tn.so[0] + r[u].s * tn.so[1] + r[u].h * tn.so[2], t, qik_mx::pack8<DT>(dn).w[0]);
    }
  }
  if constexpr (NORM) {
    // the lane groups' sums, through LDS, in group order
    float* const red = reinterpret_cast<float*>(cs);  // [RPB][D]
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) red[((int)threadIdx.x / TPR) * D + element_of<D, HALVES>(t, e)] = dw[w][e];
      __syncthreads();
      for (int d = (int)threadIdx.x; d < D; d += THREADS) {
        float v = 0.0f;
#pragma unroll
        for (int g = 0; g < RPB; ++g) v += red[g * D + d];
        p.part[((int64_t)blockIdx.x * 2 + w) * D + d] = v;
      }
    }
  }
}

// dw [2][D] from the workgroups' sums [n][2][D]: a workgroup takes 32 columns,
// its 8 lane groups every 8th sum, added in group order at the end
struct SumParams {
  const float* part;
  float* dw[2];
  int n, D;
};
__global__ void __launch_bounds__(THREADS) rope_dw_kernel(const SumParams p) {
  __shared__ float red[8][32];
  const int c = (int)threadIdx.x % 32, g = (int)threadIdx.x / 32;
  const int col = (int)blockIdx.x * 32 + c;  // of 2 D
  float v = 0.0f;
  for (int i = g; i < p.n; i += 8) v += p.part[(int64_t)i * 2 * p.D + col];
  red[g][c] = v;
  __syncthreads();
  if (g != 0) return;
  for (int i = 1; i < 8; ++i) v += red[i][c];
  const int w = col >= p.D ? 1 : 0;
  if (p.dw[w] != nullptr) p.dw[w][col - w * p.D] = v;
}

typedef void (*rope_fn)(Params);

template <int D, bool BWD>
rope_fn pick(bool fp16, bool halves, bool norm) {
#define QIK_ROPE_PICK(F, H, N) (BWD ? axial_rope_bwd_kernel<D, F, H, N> : axial_rope_kernel<D, F, H, N>)
  if (fp16) {
    if (halves) return norm ? QIK_ROPE_PICK(true, true, true) : QIK_ROPE_PICK(true, true, false);
    return norm ? QIK_ROPE_PICK(true, false, true) : QIK_ROPE_PICK(true, false, false);
  }
  if (halves) return norm ? QIK_ROPE_PICK(false, true, true) : QIK_ROPE_PICK(false, true, false);
  return norm ? QIK_ROPE_PICK(false, false, true) : QIK_ROPE_PICK(false, false, false);
#undef QIK_ROPE_PICK
}
template <bool BWD>
rope_fn pick(int64_t D, bool fp16, bool halves, bool norm) {
  switch (D) {
    case 32: return pick<32, BWD>(fp16, halves, norm);
    case 64: return pick<64, BWD>(fp16, halves, norm);
    case 128: return pick<128, BWD>(fp16, halves, norm);
    default: return pick<256, BWD>(fp16, halves, norm);
  }
}

bool strides_ok(const int64_t st[3], const qik_axial_rope_args* a, int64_t H) {
  return qik::stride_ok(st, a->B, a->S, H, 8);
}

// Checks; rows = B * S * (H of both), norm whether the tensors have weights.
int validate(const qik_axial_rope_args* a, bool bwd, int64_t* rows, bool* norm) {
  *rows = 0;
  *norm = false;
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  if (a->abi_version != QIK_ABI_VERSION || a->t[0].reserved0 != 0 || a->t[1].reserved0 != 0) return QIK_ERR_ABI_VERSION;
  if (a->dtype != QIK_DTYPE_BF16 && a->dtype != QIK_DTYPE_FP16) return QIK_ERR_DTYPE;
  if (a->D != 32 && a->D != 64 && a->D != 128 && a->D != 256) return QIK_ERR_HEAD_DIM;
  const int64_t lim = INT_MAX;
  if (a->B < 0 || a->S < 0 || a->B > lim || a->S > lim || a->naxes < 1 || a->halves < 0 || a->halves > 1) return QIK_ERR_SHAPE;
  int64_t heads = 0;
  for (int i = 0; i < 2; ++i) {
    if (a->t[i].H < 0 || a->t[i].H > lim) return QIK_ERR_SHAPE;
    heads += a->t[i].H;
  }
  if (a->B == 0 || a->S == 0 || heads == 0) return QIK_OK;
  // (a run past the last row is still an int)
  if (a->B > lim / a->S || a->B * a->S > (lim - 4096) / heads) return QIK_ERR_SHAPE;
  if (a->positions == nullptr || a->freq == nullptr || a->axis == nullptr) return QIK_ERR_NULL_ARG;
  bool with = false, without = false;
  for (int i = 0; i < 2; ++i) {
    const qik_rope_tensor& t = a->t[i];
    if (t.H == 0) continue;
    (t.weight != nullptr ? with : without) = true;
    void* const out = bwd ? t.dx : t.out;
    if (out == nullptr || (!bwd || t.weight != nullptr ? t.x == nullptr : false)) return QIK_ERR_NULL_ARG;
    if (bwd && (t.dy == nullptr || (t.weight != nullptr && t.dw == nullptr))) return QIK_ERR_NULL_ARG;
    if (!qik::aligned_to(t.x, 16) || !qik::aligned_to(out, 16) || !qik::aligned_to(t.weight, 16) ||
        (bwd && !qik::aligned_to(t.dy, 16)))
      return QIK_ERR_ALIGN;
    if (!strides_ok(t.stride_x, a, t.H) || !strides_ok(t.stride_out, a, t.H) || (bwd && !strides_ok(t.stride_dy, a, t.H)))
      return QIK_ERR_ALIGN;
  }
  if (with && without) return QIK_ERR_NULL_ARG;  // both have a weight, or neither
  *rows = a->B * a->S * heads;
  *norm = with;
  return QIK_OK;
}

void fill(const qik_axial_rope_args* a, bool bwd, int64_t rows, int run, Params* p) {
  memset(p, 0, sizeof(*p));
  for (int i = 0; i < 2; ++i) {
    const qik_rope_tensor& t = a->t[i];
    Tensor& d = p->t[i];
    d.x = static_cast<const char*>(t.x);
    d.dy = static_cast<const char*>(t.dy);
    d.out = static_cast<char*>(bwd ? t.dx : t.out);
    d.w = t.weight;
    for (int k = 0; k < 3; ++k) {
      d.sx[k] = t.stride_x[k] * 2;
      d.so[k] = t.stride_out[k] * 2;
      d.sdy[k] = t.stride_dy[k] * 2;
    }
    d.H = (int)t.H;
    d.eps = t.eps;
    p->heads += d.H;
  }
  p->pos = a->positions;
  p->freq = a->freq;
  p->axis = a->axis;
  p->pos_b = a->stride_pos_b;
  p->pos_a = a->stride_pos_a;
  p->rows = (int)rows;
  p->S = (int)a->S;
  p->runs = (int)((rows + run - 1) / run);
}

// rows of a run, and bytes of its tokens' table: a run touches at most (run -
// 2) / heads + 2 tokens, and never more than its rows
int run_of(int64_t D) { return THREADS / (int)(D / 8) * UNITS; }
size_t table_bytes(int64_t D, int run, int heads) {
  return (size_t)std::min((run - 2) / heads + 2, run) * (size_t)(D / 2) * sizeof(float2);
}

int bwd_grid(int runs) { return std::min(runs, BWD_GRID); }

}  // namespace qik_rope

extern "C" {

int qik_axial_rope(const qik_axial_rope_args* a, void* stream) {
  using namespace qik_rope;
  int64_t rows;
  bool norm;
  const int st = validate(a, false, &rows, &norm);
  if (st != QIK_OK || rows == 0) return st;
  Params p;
  const int run = run_of(a->D);
  fill(a, false, rows, run, &p);
  void* kargs[] = {&p};
  const rope_fn fn = pick<false>(a->D, a->dtype == QIK_DTYPE_FP16, a->halves != 0, norm);
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(fn), dim3((unsigned)p.runs), dim3(THREADS), kargs,
                                       table_bytes(a->D, run, p.heads), static_cast<hipStream_t>(stream));
  return e == hipSuccess ? QIK_OK : QIK_ERR_LAUNCH;
}

int qik_axial_rope_bwd_workspace_size(const qik_axial_rope_args* a, int64_t* bytes) {
  using namespace qik_rope;
  if (bytes == nullptr) return QIK_ERR_NULL_ARG;
  *bytes = 0;
  int64_t rows;
  bool norm;
  const int st = validate(a, true, &rows, &norm);
  if (st != QIK_OK || rows == 0 || !norm) return st;
  const int64_t run = run_of(a->D);
  *bytes = (int64_t)bwd_grid((int)((rows + run - 1) / run)) * 2 * a->D * 4;
  return QIK_OK;
}

int qik_axial_rope_bwd(const qik_axial_rope_args* a, void* ws, int64_t ws_bytes, void* stream) {
  using namespace qik_rope;
  int64_t rows;
  bool norm;
  int st = validate(a, true, &rows, &norm);
  if (st != QIK_OK || rows == 0) return st;
  Params p;
  const int run = run_of(a->D);
  fill(a, true, rows, run, &p);
  const int grid = bwd_grid(p.runs);
  if (norm && (ws == nullptr || !qik::aligned_to(ws, 16) || ws_bytes < (int64_t)grid * 2 * a->D * 4)) return QIK_ERR_WORKSPACE;
  p.part = static_cast<float*>(ws);
  void* kargs[] = {&p};
  const rope_fn fn = pick<true>(a->D, a->dtype == QIK_DTYPE_FP16, a->halves != 0, norm);
  const size_t lds = std::max(table_bytes(a->D, run, p.heads), (size_t)(THREADS / (a->D / 8) * a->D * 4));
  if (hipLaunchKernel(reinterpret_cast<const void*>(fn), dim3((unsigned)grid), dim3(THREADS), kargs, lds,
                      static_cast<hipStream_t>(stream)) != hipSuccess)
    return QIK_ERR_LAUNCH;
  if (!norm) return QIK_OK;
  SumParams s = {p.part, {a->t[0].H > 0 ? a->t[0].dw : nullptr, a->t[1].H > 0 ? a->t[1].dw : nullptr}, grid, (int)a->D};
  void* sargs[] = {&s};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(rope_dw_kernel), dim3((unsigned)(2 * a->D / 32)), dim3(THREADS),
                                       sargs, 0, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? QIK_OK : QIK_ERR_LAUNCH;
}

}  // extern "C"
