// RMSNorm over each head and the rotation by positions on several axes, of a
// layer's Q and K in one launch, and its gradient (include/qik_rope.h).
//
// A byte mover (every row is read and written once) that computes nearly as long
// as it moves, so the arithmetic is kept to what a row needs:
//   * the D / 2 angles of a token are the same for all its heads, in Q and in K: a
//     workgroup takes some tokens, computes their cosines and sines into LDS, and
//     turns their rows of Q and then those of K, so that what belongs to a tensor
//     (addresses, strides, the weight) is one for the whole workgroup.  With rows
//     of both in a run and a choice for each, 4352 tokens x 48 heads x 128 took
//     28.0 us, so 17.4 (22.6, 4.7 TB/s, with its operands from memory; the gradient
//     36, 4.4 TB/s);
//   * D / 8 lanes hold a row, a lane the pairs 4t .. 4t + 3: eight neighbouring
//     elements, or four of each half.  Sums over a row go by DPP;
//   * rows are found by multiplications with the host's reciprocals.

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
constexpr int UNITS = 2;            // rows of a lane group, their loads issued together
constexpr int ROWS_AIM = 96;        // rows of the larger tensor that a workgroup takes at once
constexpr int TABLE_BYTES = 32768;  // of cosines and sines at most
// backward: workgroups at most, each with a [2, D] sum of dw in the workspace
constexpr int BWD_GRID = 512;

struct Tensor {
  const char* x;
  const char* dy;
  char* out;                        // y, or dx
  const float* w;
  unsigned sx[3], so[3], sdy[3];    // b, s, h in 16 bytes
  int H;
  unsigned by_H;                    // see quotient
  float eps;
};

struct Params {
  Tensor t[2];
  const double* pos;
  const double* freq;
  const int32_t* axis;
  int64_t pos_b, pos_a;
  float* part;                      // backward: [grid][2][D]
  int tokens;                       // B * S
  int S;
  unsigned by_S;
  int chunk;                        // tokens a workgroup takes at once
};

// n / d by ceil(2^32 / d) (0 for d = 1): exact while n * d < 2^32 (for a larger
// product the estimate is at most one too large, which the last line takes back)
__device__ __forceinline__ int quotient(int n, int d, unsigned by) {
  if (by == 0u) return n;
  const unsigned q = __umulhi((unsigned)n, by);
  return (int)(q * (unsigned)d > (unsigned)n ? q - 1u : q);
}

// the lane's eight elements of a row: pairs 4t .. 4t + 3, in order
template <int D, bool HALVES>
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

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// the sum over a row's TPR lanes, in each of them: quad_perm {1, 0, 3, 2} and {2, 3,
// 0, 1}, then mirrors of 8 and 16 lanes (whose halves are equal by then), then
// the other 16
template <int TPR>
__device__ __forceinline__ float row_sum(float v) {
  v = dpp_add<0xb1>(v);
  v = dpp_add<0x4e>(v);
  if constexpr (TPR >= 8) v = dpp_add<0x141>(v);
  if constexpr (TPR >= 16) v = dpp_add<0x140>(v);
  if constexpr (TPR >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// a row: its token's place in the workgroup's table, and where it lies
struct Row {
  int token, b, s, h;
};
__device__ __forceinline__ Row row_of(const Params& p, const Tensor& x, int first, int row) {
  Row r;
  r.token = quotient(row, x.H, x.by_H);
  r.h = row - r.token * x.H;
  const int token = first + r.token;
  r.b = quotient(token, p.S, p.by_S);
  r.s = token - r.b * p.S;
  return r;
}
__device__ __forceinline__ int64_t bytes_of(const Row& r, const unsigned (&st)[3]) {
  return (int64_t)(((uint64_t)(unsigned)r.b * st[0] + (uint64_t)(unsigned)r.s * st[1] + (uint64_t)(unsigned)r.h * st[2]) << 4);
}

// cosines and sines of the tokens [first, first + n) into cs [n][D / 2]
template <int D>
__device__ __forceinline__ void turn_table(const Params& p, int first, int n, float2* cs) {
  for (int i = (int)threadIdx.x; i < n * (D / 2); i += THREADS) {
    const int pair = i % (D / 2), token = first + i / (D / 2);
    const int b = quotient(token, p.S, p.by_S), s = token - b * p.S;
    const double turns = p.pos[b * p.pos_b + p.axis[pair] * p.pos_a + s] * p.freq[pair];
    float sn, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &c);
    cs[i] = make_float2(c, sn);
  }
}

// r of a row from its sum of squares: the instruction's result is within an ulp
template <int D>
__device__ __forceinline__ float rsqrt_of(float ss, float eps) {
  return __builtin_amdgcn_rsqf(__builtin_fmaf(ss, 1.0f / D, eps));
}

template <int D, bool HALVES>
__device__ __forceinline__ void load_weight(const float* w, int t, float (&wv)[8]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const float4 v = *reinterpret_cast<const float4*>(w + element_of<D, HALVES>(t, 4 * q));
    wv[4 * q] = v.x, wv[4 * q + 1] = v.y, wv[4 * q + 2] = v.z, wv[4 * q + 3] = v.w;
  }
}

template <int D, bool FP16, bool HALVES, bool NORM>
__global__ void __launch_bounds__(THREADS) axial_rope_kernel(const Params p) {
  constexpr int DT = FP16 ? QIK_DTYPE_FP16 : QIK_DTYPE_BF16;
  constexpr int TPR = D / 8, RPB = THREADS / TPR;
  extern __shared__ float2 cs[];
  const int t = (int)threadIdx.x % TPR;
  const int first = (int)blockIdx.x * p.chunk;
  const int n = min(p.chunk, p.tokens - first);
  turn_table<D>(p, first, n, cs);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const Tensor& x = p.t[k];
    const int rows = n * x.H;
    [[maybe_unused]] float wv[8];
    if constexpr (NORM) {
      if (rows > 0) load_weight<D, HALVES>(x.w, t, wv);
    }
    for (int row0 = (int)threadIdx.x / TPR; row0 < rows; row0 += RPB * UNITS) {
      u32x4 raw[UNITS];
      Row r[UNITS];
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        r[u] = row_of(p, x, first, min(row0 + u * RPB, rows - 1));
        raw[u] = load_pairs<D, HALVES>(x.x + bytes_of(r[u], x.sx), t);
      }
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        float v[8];
        qik_mx::unpack8<DT>(Raw8<DT>{{raw[u]}}, v);
        if constexpr (NORM) {
          float ss = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[e], v[e], ss);
          const float rs = rsqrt_of<D>(row_sum<TPR>(ss), x.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (v[e] * rs) * wv[e];
        }
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 c = cs[r[u].token * (D / 2) + 4 * t + i];
          const float a = v[first_of<HALVES>(i)], b = v[second_of<HALVES>(i)];
          y[first_of<HALVES>(i)] = a * c.x - b * c.y;
          y[second_of<HALVES>(i)] = a * c.y + b * c.x;
        }
        if (row0 + u * RPB < rows) store_pairs<D, HALVES>(x.out + bytes_of(r[u], x.so), t, qik_mx::pack8<DT>(y).w[0]);
      }
    }
  }
}

// The gradient: as above with dy beside x; a workgroup takes every gridDim.x-th
// chunk of tokens and keeps its rows' sums of dw in registers, which become one
// [2, D] sum in the workspace at its end.
template <int D, bool FP16, bool HALVES, bool NORM>
__global__ void __launch_bounds__(THREADS) axial_rope_bwd_kernel(const Params p) {
  constexpr int DT = FP16 ? QIK_DTYPE_FP16 : QIK_DTYPE_BF16;
  constexpr int TPR = D / 8, RPB = THREADS / TPR;
  extern __shared__ float2 cs[];
  const int t = (int)threadIdx.x % TPR;
  float dw[2][8] = {};
  for (int first = (int)blockIdx.x * p.chunk; first < p.tokens; first += (int)gridDim.x * p.chunk) {
    const int n = min(p.chunk, p.tokens - first);
    __syncthreads();  // the last chunk's table has been read
    turn_table<D>(p, first, n, cs);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Tensor& x = p.t[k];
      const int rows = n * x.H;
      [[maybe_unused]] float wv[8];
      if constexpr (NORM) {
        if (rows > 0) load_weight<D, HALVES>(x.w, t, wv);
      }
      for (int row0 = (int)threadIdx.x / TPR; row0 < rows; row0 += RPB * UNITS) {
        u32x4 raw[UNITS], gr[UNITS];
        Row r[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          r[u] = row_of(p, x, first, min(row0 + u * RPB, rows - 1));
          gr[u] = load_pairs<D, HALVES>(x.dy + bytes_of(r[u], x.sdy), t);
          if constexpr (NORM) raw[u] = load_pairs<D, HALVES>(x.x + bytes_of(r[u], x.sx), t);
        }
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const bool live = row0 + u * RPB < rows;
          float g[8], dn[8];
          qik_mx::unpack8<DT>(Raw8<DT>{{gr[u]}}, g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 c = cs[r[u].token * (D / 2) + 4 * t + i];
            const float a = g[first_of<HALVES>(i)], b = g[second_of<HALVES>(i)];
            dn[first_of<HALVES>(i)] = a * c.x + b * c.y;
            dn[second_of<HALVES>(i)] = b * c.x - a * c.y;
          }
          if constexpr (NORM) {
            float v[8];
            qik_mx::unpack8<DT>(Raw8<DT>{{raw[u]}}, v);
            float ss = 0.0f, dot = 0.0f;
            float wd[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              wd[e] = dn[e] * wv[e];
              ss = __builtin_fmaf(v[e], v[e], ss);
              dot = __builtin_fmaf(v[e], wd[e], dot);
            }
            const float rs = rsqrt_of<D>(row_sum<TPR>(ss), x.eps);
            const float pull = row_sum<TPR>(dot) * (1.0f / D) * rs * rs;  // mean(x w dn) r^2
            const float rs_dw = live ? rs : 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              dw[k][e] = __builtin_fmaf(dn[e], v[e] * rs_dw, dw[k][e]);
              dn[e] = rs * __builtin_fmaf(-v[e], pull, wd[e]);
            }
          }
          if (live) store_pairs<D, HALVES>(x.out + bytes_of(r[u], x.so), t, qik_mx::pack8<DT>(dn).w[0]);
        }
      }
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

// dw [2][D] from the workgroups' sums [n][2][D]: a workgroup takes 16 columns,
// each of its 64 lane groups every 64th sum (at most BWD_GRID / 64 loads, all at
// once), added in a fixed order at the end.  With 8 groups and one load after
// the other it took 19 us for 512 sums.
struct SumParams {
  const float* part;
  float* dw[2];
  int n, D;
};
constexpr int SUM_COLUMNS = 16;
constexpr int SUM_THREADS = 1024;
__global__ void __launch_bounds__(SUM_THREADS) rope_dw_kernel(const SumParams p) {
  constexpr int GROUPS = SUM_THREADS / SUM_COLUMNS;
  __shared__ float red[GROUPS][SUM_COLUMNS];
  const int c = (int)threadIdx.x % SUM_COLUMNS, g = (int)threadIdx.x / SUM_COLUMNS;
  const int col = (int)blockIdx.x * SUM_COLUMNS + c;  // of 2 D
  float x[BWD_GRID / GROUPS];
#pragma unroll
  for (int i = 0; i < BWD_GRID / GROUPS; ++i) x[i] = g + i * GROUPS < p.n ? p.part[(int64_t)(g + i * GROUPS) * 2 * p.D + col] : 0.0f;
#pragma unroll
  for (int i = 1; i < BWD_GRID / GROUPS; ++i) x[0] += x[i];
  red[g][c] = x[0];
  __syncthreads();
#pragma unroll
  for (int k = GROUPS / 2; k >= 1; k >>= 1) {
    if (g < k) red[g][c] += red[g + k][c];
    __syncthreads();
  }
  const int w = col >= p.D ? 1 : 0;
  if (g == 0 && p.dw[w] != nullptr) p.dw[w][col - w * p.D] = red[0][c];
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

// (the kernels hold strides in units of 16 bytes and 32 bits)
bool strides_fit(const int64_t st[3]) {
  for (int i = 0; i < 3; ++i)
    if (st[i] < 0 || st[i] / 8 > (int64_t)UINT_MAX) return false;
  return true;
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
  // (a chunk of tokens past the last is still an int)
  if (a->B > lim / a->S || a->B * a->S > (lim - BWD_GRID * 512) / heads) return QIK_ERR_SHAPE;
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
    if (!strides_fit(t.stride_x) || !strides_fit(t.stride_out) || (bwd && !strides_fit(t.stride_dy))) return QIK_ERR_SHAPE;
  }
  if (with && without) return QIK_ERR_NULL_ARG;  // both have a weight, or neither
  *rows = a->B * a->S * heads;
  *norm = with;
  return QIK_OK;
}

unsigned reciprocal(int64_t d) { return d <= 1 ? 0u : (unsigned)((((int64_t)1 << 32) + d - 1) / d); }

// Tokens of a chunk: ROWS_AIM rows of the tensor with more heads, fewer where
// that leaves CUs without a workgroup, as many as the table holds at most.
int chunk_of(const qik_axial_rope_args* a) {
  const int64_t H = std::max<int64_t>(std::max(a->t[0].H, a->t[1].H), 1);
  const int64_t tokens = a->B * a->S;
  const int64_t most = TABLE_BYTES / (a->D / 2 * (int64_t)sizeof(float2));
  int64_t n = std::min((ROWS_AIM + H - 1) / H, most);
  const int64_t spread = tokens / (2 * (int64_t)std::max(qik::device_cus(), 1));
  return (int)std::max<int64_t>(std::min(n, spread), 1);
}

void fill(const qik_axial_rope_args* a, bool bwd, int chunk, Params* p) {
  memset(p, 0, sizeof(*p));
  for (int i = 0; i < 2; ++i) {
    const qik_rope_tensor& t = a->t[i];
    Tensor& d = p->t[i];
    d.x = static_cast<const char*>(t.x);
    d.dy = static_cast<const char*>(t.dy);
    d.out = static_cast<char*>(bwd ? t.dx : t.out);
    d.w = t.weight;
    for (int k = 0; k < 3; ++k) {
      d.sx[k] = (unsigned)(t.stride_x[k] / 8);
      d.so[k] = (unsigned)(t.stride_out[k] / 8);
      d.sdy[k] = (unsigned)(t.stride_dy[k] / 8);
    }
    d.H = (int)t.H;
    d.by_H = reciprocal(t.H);
    d.eps = t.eps;
  }
  p->pos = a->positions;
  p->freq = a->freq;
  p->axis = a->axis;
  p->pos_b = a->stride_pos_b;
  p->pos_a = a->stride_pos_a;
  p->tokens = (int)(a->B * a->S);
  p->S = (int)a->S;
  p->by_S = reciprocal(a->S);
  p->chunk = chunk;
}

size_t table_bytes(int64_t D, int chunk) { return (size_t)chunk * (size_t)(D / 2) * sizeof(float2); }

int bwd_grid(int64_t tokens, int chunk) { return (int)std::min<int64_t>((tokens + chunk - 1) / chunk, BWD_GRID); }

}  // namespace qik_rope

extern "C" {

int qik_axial_rope(const qik_axial_rope_args* a, void* stream) {
  using namespace qik_rope;
  int64_t rows;
  bool norm;
  const int st = validate(a, false, &rows, &norm);
  if (st != QIK_OK || rows == 0) return st;
  Params p;
  const int chunk = chunk_of(a);
  fill(a, false, chunk, &p);
  void* kargs[] = {&p};
  const rope_fn fn = pick<false>(a->D, a->dtype == QIK_DTYPE_FP16, a->halves != 0, norm);
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(fn), dim3((unsigned)((p.tokens - 1) / chunk + 1)), dim3(THREADS),
                                       kargs, table_bytes(a->D, chunk), static_cast<hipStream_t>(stream));
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
  *bytes = (int64_t)bwd_grid(a->B * a->S, chunk_of(a)) * 2 * a->D * 4;
  return QIK_OK;
}

int qik_axial_rope_bwd(const qik_axial_rope_args* a, void* ws, int64_t ws_bytes, void* stream) {
  using namespace qik_rope;
  int64_t rows;
  bool norm;
  int st = validate(a, true, &rows, &norm);
  if (st != QIK_OK || rows == 0) return st;
  Params p;
  const int chunk = chunk_of(a);
  fill(a, true, chunk, &p);
  const int grid = bwd_grid(p.tokens, chunk);
  if (norm && (ws == nullptr || !qik::aligned_to(ws, 16) || ws_bytes < (int64_t)grid * 2 * a->D * 4)) return QIK_ERR_WORKSPACE;
  p.part = static_cast<float*>(ws);
  void* kargs[] = {&p};
  const rope_fn fn = pick<true>(a->D, a->dtype == QIK_DTYPE_FP16, a->halves != 0, norm);
  const size_t lds = std::max(table_bytes(a->D, chunk), (size_t)(THREADS / (a->D / 8) * a->D * 4));
  if (hipLaunchKernel(reinterpret_cast<const void*>(fn), dim3((unsigned)grid), dim3(THREADS), kargs, lds,
                      static_cast<hipStream_t>(stream)) != hipSuccess)
    return QIK_ERR_LAUNCH;
  if (!norm) return QIK_OK;
  SumParams s = {p.part, {a->t[0].H > 0 ? a->t[0].dw : nullptr, a->t[1].H > 0 ? a->t[1].dw : nullptr}, grid, (int)a->D};
  void* sargs[] = {&s};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(rope_dw_kernel), dim3((unsigned)(2 * a->D / SUM_COLUMNS)), dim3(SUM_THREADS),
                                       sargs, 0, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? QIK_OK : QIK_ERR_LAUNCH;
}

}  // extern "C"
