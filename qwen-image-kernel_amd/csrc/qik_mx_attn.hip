// The 4-bit prefix slab and the attention over it: the entry points of
// include/qik_mx_attn.h.  The slab's store and load are byte movers (a thread
// takes eight elements of a row, a quad of lanes a block of 32); the attention
// runs the kernel of qik_mx_rows.h for few query rows and that of
// qik_attn_kernel.h, in its 4-bit instance, for others (4096 rows against 2560 slab
// rows and 4096 fresh keys, 24 heads of 128: 328 to 345 us on different cards, 970
// to 1020 TFLOP/s, 1.04 times a bf16 slab's time; the codes are turned while the
// matrix cores work).

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include <limits.h>
#include <algorithm>
#include <atomic>
#include <cmath>

#include "qik_mx_attn.h"
#include "qik_mx_block.h"
#include "qik_attn_kernel.h"
#include "qik_attn_launch.h"
#include "qik_mx_rows.h"

namespace qik_mx_slabs {

using qik_mx::u32x2;
using qik_mx::u32x4;

constexpr int THREADS = 256;
constexpr int UNITS = 4;  // rows of a thread, their loads issued before any of them is used

// A workgroup takes rows of one (b, h): blockIdx.y, and every gridDim.y-th on;
// blockIdx.z: K or V.  With rows of all heads in one number and a division for
// each, the arithmetic took longer than the bytes (2560 x 24 x 128: 10.2 us
// stored, 11.9 loaded; so 9.0 and 8.3, 4.4 and 4.8 TB/s).
template <int D>
constexpr int rows_of_group() { return THREADS / (D / 8) * UNITS; }

struct StoreParams {
  const char* src[2];            // K, V
  unsigned char* codes[2];
  unsigned char* scales[2];
  int64_t ss[2][3];              // source b, s, h in bytes
  int64_t sc[2][3], se[2][3];    // codes, scales: b, p, h in bytes
  const int32_t* at;
  int32_t* lengths;
  unsigned* arrivals;            // the word that counts workgroups where lengths == at
  int B, S, H;
  int capacity;
};

template <int D, bool FP16>
__global__ void __launch_bounds__(THREADS) slab_store_kernel(const StoreParams p) {
  constexpr int DT = FP16 ? QIK_DTYPE_FP16 : QIK_DTYPE_BF16;
  constexpr int TPR = D / 8;             // threads of a row
  constexpr int RPB = THREADS / TPR;     // rows of a pass
  const int which = blockIdx.z;
  const int t = (int)threadIdx.x % TPR;
  const int s0 = (int)blockIdx.x * rows_of_group<D>() + (int)threadIdx.x / TPR;
  for (int bh = (int)blockIdx.y; bh < p.B * p.H; bh += (int)gridDim.y) {
    const int b = (int)((unsigned)bh / (unsigned)p.H), h = bh - b * p.H;
    const char* const src = p.src[which] + b * p.ss[which][0] + h * p.ss[which][2] + t * 16;
    unsigned char* const codes = p.codes[which] + b * p.sc[which][0] + h * p.sc[which][2] + 4 * t;
    unsigned char* const scales = p.scales[which] + b * p.se[which][0] + h * p.se[which][2] + t / 4;
    const int at0 = p.at == nullptr ? 0 : p.at[b];
    qik_mx::Raw8<DT> raw[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) raw[u] = qik_mx::load8<DT, true>(src + min(s0 + u * RPB, p.S - 1) * p.ss[which][1]);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      float f[8];
      qik_mx::unpack8<DT>(raw[u], f);
      unsigned w0, w1;
      const unsigned byte = qik_mx::block_codes<QIK_MXFP4>(f, w0, w1);
      const int s = s0 + u * RPB;
      const int64_t at = (int64_t)at0 + s;
      if (s >= p.S || at < 0 || at >= p.capacity) continue;
      *reinterpret_cast<unsigned*>(codes + at * p.sc[which][1]) = w0;
      if ((t & 3) == 0) scales[at * p.se[which][1]] = (unsigned char)byte;
    }
  }
  if (p.lengths == nullptr) return;
  // the lengths behind the new rows.  Where they are what `at` was, they change
  // once every workgroup has read it: the last to arrive writes them
  if (p.arrivals != nullptr) {
    __shared__ int last;
    __syncthreads();
    if (threadIdx.x == 0) {
      const unsigned all = gridDim.x * gridDim.y * gridDim.z;
      last = qik::g_fetch_add(p.arrivals, 1u) == all - 1u ? 1 : 0;
      if (last) qik::g_store(p.arrivals, 0u);
    }
    __syncthreads();
    if (last == 0) return;
  } else if (blockIdx.x != 0 || blockIdx.y != 0 || blockIdx.z != 0) {
    return;
  }
  for (int b = (int)threadIdx.x; b < p.B; b += THREADS) {
    const int64_t n = (p.at == nullptr ? 0 : (int64_t)p.at[b]) + p.S;
    p.lengths[b] = (int32_t)min(max(n, (int64_t)0), (int64_t)p.capacity);
  }
}

struct LoadParams {
  const unsigned char* codes[2];
  const unsigned char* scales[2];
  char* out[2];                  // [B, P, H, D]
  int64_t sc[2][3], se[2][3];
  const int32_t* lengths;
  int B, P, H;
};

template <int D, bool FP16>
__global__ void __launch_bounds__(THREADS) slab_load_kernel(const LoadParams p) {
  constexpr int TPR = D / 8;
  constexpr int RPB = THREADS / TPR;
  const int which = blockIdx.z;
  const int t = (int)threadIdx.x % TPR;
  const int s0 = (int)blockIdx.x * rows_of_group<D>() + (int)threadIdx.x / TPR;
  for (int bh = (int)blockIdx.y; bh < p.B * p.H; bh += (int)gridDim.y) {
    const int b = (int)((unsigned)bh / (unsigned)p.H), h = bh - b * p.H;
    const unsigned char* const codes = p.codes[which] + b * p.sc[which][0] + h * p.sc[which][2] + 4 * t;
    const unsigned char* const scales = p.scales[which] + b * p.se[which][0] + h * p.se[which][2] + t / 4;
    char* const out = p.out[which] + ((int64_t)b * p.P * p.H + h) * (D * 2) + t * 16;
    const int n = p.lengths == nullptr ? p.P : min(p.lengths[b], p.P);
    unsigned code[UNITS], e[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int s = s0 + u * RPB;
      code[u] = 0u;
      e[u] = 127u;
      if (s < n) {
        code[u] = *reinterpret_cast<const unsigned*>(codes + s * p.sc[which][1]);
        e[u] = scales[s * p.se[which][1]];
      }
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int s = s0 + u * RPB;
      if (s < p.P)
        *reinterpret_cast<u32x4*>(out + (int64_t)s * p.H * (D * 2)) = qik::dequant_fp4x8<FP16>(code[u], __uint_as_float(e[u] << 23));
    }
  }
}

// the grid of both: rows [B, H, S]
dim3 slab_grid(int64_t B, int64_t S, int64_t H, int64_t D) {
  const int64_t rows = THREADS / (D / 8) * UNITS;
  return dim3((unsigned)((S + rows - 1) / rows), (unsigned)std::min<int64_t>(B * H, 65535), 2);
}

typedef void (*store_fn)(StoreParams);
typedef void (*load_fn)(LoadParams);
template <bool FP16>
store_fn pick_store(int64_t D) {
  switch (D) {
    case 32: return slab_store_kernel<32, FP16>;
    case 64: return slab_store_kernel<64, FP16>;
    case 128: return slab_store_kernel<128, FP16>;
    default: return slab_store_kernel<256, FP16>;
  }
}
template <bool FP16>
load_fn pick_load(int64_t D) {
  switch (D) {
    case 32: return slab_load_kernel<32, FP16>;
    case 64: return slab_load_kernel<64, FP16>;
    case 128: return slab_load_kernel<128, FP16>;
    default: return slab_load_kernel<256, FP16>;
  }
}

// Layout rules of one slab of rows [B, P, H, D].
int slab_status(const qik_mx_slab& s, int64_t B, int64_t P, int64_t H, int64_t D) {
  if (s.codes == nullptr || s.scales == nullptr) return QIK_ERR_NULL_ARG;
  const int64_t eb = D / 32;
  if (!qik::aligned_to(s.codes, 16) || !qik::aligned_to(s.scales, (uintptr_t)eb)) return QIK_ERR_ALIGN;
  if (!qik::stride_ok(s.stride_codes, B, P, H, 16) || !qik::stride_ok(s.stride_scales, B, P, H, eb)) return QIK_ERR_ALIGN;
  if (P > 1 && (s.stride_codes[1] < D / 2 || s.stride_scales[1] < eb)) return QIK_ERR_ALIGN;
  const int64_t lim = ((int64_t)1 << 31) / qik::BN;  // a tile's byte offsets are 31 bits
  if (P > 1 && (s.stride_codes[1] >= lim || s.stride_scales[1] >= lim)) return QIK_ERR_SHAPE;
  return QIK_OK;
}

}  // namespace qik_mx_slabs

namespace qik {

typedef void (*mx_kernel_fn)(MxParams);
typedef void (*rows_kernel_fn)(RowsParams);

template <int D, bool FP16, bool KV>
void pick_mx(Kernels* k) {
  mx_kernel_fn f = attn_fwd_kernel<D, FP16, SlabKV::MX, KV, 1, false>;
  k->one = reinterpret_cast<const void*>(f);
  if constexpr (D <= 128) {
    f = attn_fwd_kernel<D, FP16, SlabKV::MX, KV, 1, true>;
    k->pieces = reinterpret_cast<const void*>(f);
    f = attn_fwd_kernel<D, FP16, SlabKV::MX, KV, 2, false>;
    k->groups = reinterpret_cast<const void*>(f);
  }
}
template <int D>
void pick_mx(bool fp16, bool kv, Kernels* k) {
  if (fp16) kv ? pick_mx<D, true, true>(k) : pick_mx<D, true, false>(k);
  else kv ? pick_mx<D, false, true>(k) : pick_mx<D, false, false>(k);
}
template <int D, int MT, bool SPREAD>
rows_kernel_fn pick_rows(bool fp16, bool kv) {
  if (fp16) return kv ? mx_rows_kernel<D, true, true, MT, SPREAD> : mx_rows_kernel<D, true, false, MT, SPREAD>;
  return kv ? mx_rows_kernel<D, false, true, MT, SPREAD> : mx_rows_kernel<D, false, false, MT, SPREAD>;
}
template <int D>
rows_kernel_fn pick_rows(bool fp16, bool kv, int mt, bool spread) {
  if (spread) return pick_rows<D, 1, true>(fp16, kv);
  return mt == 1 ? pick_rows<D, 1, false>(fp16, kv) : pick_rows<D, 2, false>(fp16, kv);
}

std::atomic<int> g_mx_slots[16][MAX_DEVICES];

Kernels mx_kernels_of(const qik_attn_args* a) {
  const bool fp16 = a->dtype == QIK_DTYPE_FP16;
  const bool kv = (a->flags & QIK_HAS_KEY_VALID) != 0;
  Kernels k = {nullptr, nullptr, nullptr, nullptr};
  int di = 3;
  switch (a->D) {
    case 32: pick_mx<32>(fp16, kv, &k); di = 0; break;
    case 64: pick_mx<64>(fp16, kv, &k); di = 1; break;
    case 128: pick_mx<128>(fp16, kv, &k); di = 2; break;
    default: pick_mx<256>(fp16, kv, &k); break;
  }
  k.slots = g_mx_slots[4 * di + (fp16 ? 2 : 0) + (kv ? 1 : 0)];
  return k;
}

rows_kernel_fn rows_kernel_of(const qik_attn_args* a, int mt, bool spread) {
  const bool fp16 = a->dtype == QIK_DTYPE_FP16;
  const bool kv = (a->flags & QIK_HAS_KEY_VALID) != 0;
  switch (a->D) {
    case 32: return pick_rows<32>(fp16, kv, mt, spread);
    case 64: return pick_rows<64>(fp16, kv, mt, spread);
    case 128: return pick_rows<128>(fp16, kv, mt, spread);
    default: return pick_rows<256>(fp16, kv, mt, spread);
  }
}

// The kernel of few rows (qik_mx_rows.h): 16-row tiles of an item, items for a KV
// head's rows, steps of a piece and pieces of an item at most.
struct RowsPlan {
  bool few;
  int mt, nrt, steps, pieces;
  int row_bits;  // log2 of the rows a piece keeps in the workspace
  int spread;    // pieces that the entries aim at together, 0: `pieces` each
};

// What a call of few rows lasts, in us, fitted to 2500 measured shapes of two
// tiles (17 to 28000 rows of 1 to 24 KV heads, 1 to 4 entries, 16 to 40000 slab
// rows, in up to 12 pieces) and 800 of one tile (1 to 40 entries, 64 to 130000 slab
// rows) on 256 CUs; the errors' root mean square is 7 to 18%.  Rounds of as many
// pieces as the CUs hold, each `piece` and a wave's steps, at `step` at least and
// `fill` for each piece on the CU, one of fresh keys, which are not loaded ahead,
// `fresh` times as long; `once`; and where there are pieces the merge, `join` and
// `merge` for 100 KB of them, which one workgroup reads.  `share`: how many of
// the pieces behind an item's first have keys.
struct RowsCost {
  int held;  // pieces on a CU at once
  double step, fill, fresh, once, piece, join, merge;
};
const RowsCost& rows_cost_of(int64_t D, int mt) {
  static constexpr RowsCost one[4] = {{3, 0.57, 0.57, 1.2, 5.2, 0.75, 2.0, 2.6}, {2, 0.7, 0.7, 2.0, 4.8, 1.5, 1.75, 2.6},
                                      {2, 0.85, 1.1, 2.4, 3.3, 2.7, 1.9, 2.6}, {1, 2.1, 0.75, 2.5, 1.4, 4.1, 2.9, 2.6}};
  static constexpr RowsCost two[4] = {{2, 0.72, 0.635, 1.2, 3.8, 2.6, 2.0, 2.1}, {2, 0.9, 0.82, 2.0, 3.1, 3.0, 2.0, 2.1},
                                      {1, 1.36, 1.36, 2.4, 1.4, 4.7, 3.0, 2.1}, {1, 2.2, 2.2, 2.5, 2.0, 7.2, 6.5, 2.1}};
  return (mt > 1 ? two : one)[D <= 32 ? 0 : D <= 64 ? 1 : D <= 128 ? 2 : 3];
}
// n: all pieces (workgroups with keys), steps: of one, pieces: of the longest item,
// mixed: how long a step lasts beside one of the slab; rows: of an item, in the workspace
double rows_cost(const RowsCost& c, double n, double steps, double mixed, int64_t pieces, int cus, int waves, int64_t rows,
                 int64_t D) {
  const double wave = std::ceil(steps / waves) * mixed, round = (double)c.held * cus;
  const double full = std::floor(n / round), rest = std::ceil((n - full * round) / cus);
  double us = c.once + full * (c.piece + wave * std::max(c.step, c.fill * c.held));
  if (rest > 0.0) us += c.piece + wave * std::max(c.step, c.fill * rest);
  return us + (pieces > 1 ? c.join + (double)(pieces * rows * 4 * D) * c.merge * 1e-5 : 0.0);
}

// The same of the kernel of many rows: `once`, `round` for each two row blocks of
// a CU, its KV tiles at `tile` at least, as a row block's can be split over few
// CUs, and `block` for a CU's first row block and `more` for each further one.
// The choice between the two is 0.3 to 0.8% slower than the best measured one on
// average (by one rule, from D = 128, without the rounds: 1 to 3%, and up to 1.8
// times at D = 256).
struct ManyCost {
  double once, round, tile, block, more;
};
double many_cost(int64_t blocks, int64_t T, int cus, int64_t D) {
  static constexpr ManyCost costs[4] = {
      {1.0, 7.3, 0.28, 0.7, 0.34}, {0.5, 8.4, 0.363, 1.0, 0.45}, {3.1, 7.5, 0.46, 1.34, 1.13}, {0.0, 17.5, 1.83, 4.75, 3.7}};
  const ManyCost& c = costs[D <= 32 ? 0 : D <= 64 ? 1 : D <= 128 ? 2 : 3];
  const double n = (double)blocks / cus;
  return c.once + c.round * (double)cdiv64(blocks, 2 * (int64_t)cus) +
         (double)T * std::max(c.tile, c.block * std::min(n, 1.0) + c.more * std::max(n - 1.0, 0.0));
}

// what a workgroup takes for the lengths of all entries and its place among them, us
constexpr double SPREAD_US = 1.0;

RowsPlan make_rows_plan(int64_t B, int64_t SQ, int64_t SN, int64_t P, int64_t H, int64_t HKV, int64_t D, bool ragged, int cus) {
  RowsPlan r = {false, 0, 0, 0, 0, 0, 0};
  const int64_t G = H / HKV, R = SQ * G;
  r.mt = R <= ROWS_M ? 1 : 2;
  const int64_t nrt = cdiv64(R, r.mt * ROWS_M);
  // limits of the kernel: its grid has the entries in y and the pieces in z, less
  // than 2^32 threads in x, and it divides by multiplication
  if (B > 65535 || HKV * nrt > (1 << 22) || G > INT_MAX / R || HKV * nrt > INT_MAX / HKV) return r;
  r.nrt = (int)nrt;
  cus = std::max(cus, 1);
  const int waves = rows_waves((int)D, r.mt);
  const int64_t slab = cdiv64(P, ROWS_N), T = std::max<int64_t>(slab + cdiv64(SN, ROWS_N), 1);
  const int64_t items = B * HKV * nrt;
  while ((1 << r.row_bits) < std::min<int64_t>(R, r.mt * ROWS_M)) ++r.row_bits;
  // every wave of a piece has a step, two where there are many pieces; an item
  // that is cut has a word of the control words
  const int64_t steps = std::max<int64_t>(T / waves, 1);
  const int64_t most = items > QIK_ATTN_WS_CTL_BYTES / 4 ? 1 : std::min<int64_t>(std::max<int64_t>(steps / 2, std::min<int64_t>(steps, 8)), 65535);
  const RowsCost& c = rows_cost_of(D, r.mt);
  const int64_t rows = (int64_t)1 << r.row_bits;
  const double mixed = ((double)slab + c.fresh * (double)(T - slab)) / (double)T;
  // Pieces that fill the CUs half, once, .. four times.  Against the best measured
  // number this loses 0.4 to 1.6% on average (a workgroup a CU always: 4 to 7);
  // 131072 keys of 8 heads take 31.6 us in 32 pieces, 34.3 in 64, 44.9 in 16.
  // With lengths of several entries P is the longest's only, and a share of the
  // pieces has no keys: a mean over three.  The shares, and the mean length of 0.6 P
  // below, are those of lengths spread evenly from an eighth of the longest to all of
  // it, which were measured; others were not, and only the estimates go by them.
  // (Two tiles, beside the other kernel's estimate: as if all were that long.)
  const bool several = ragged && r.mt == 1 && B > 1;
  auto cost = [&](int64_t n) {
    double us = 0.0;
    const int shares = several && n > 1 ? 3 : 1;
    for (int i = 0; i < shares; ++i) {
      const double share = shares > 1 ? 0.5 + 0.1 * i : 1.0;
      us += rows_cost(c, (double)items * (1.0 + (double)(n - 1) * share), (double)cdiv64(T, n), mixed, n, cus, waves, rows, D);
    }
    return us / shares;
  };
  int64_t pieces = 1;
  double least = cost(1);
  for (int64_t k = 1; k <= 8; ++k) {
    const int64_t n = std::min(std::max<int64_t>((k * cus + items) / (2 * items), 1), most);
    if (n == pieces) continue;
    const double us = cost(n);
    if (us < least) least = us, pieces = n;
  }
  r.few = r.mt == 1 || least < many_cost(B * HKV * cdiv64(R, BM), cdiv64(P, BN) + cdiv64(SN, BN), cus, D);
  r.steps = (int)cdiv64(T, pieces);
  r.pieces = (int)cdiv64(T, r.steps);
  // Or the kernel cuts what it finds into the pieces that the host aims at, which
  // with the last ones of the entries fill the CUs half, once, .. four times (the
  // estimate takes 0.6 P for the mean length, and SPREAD_US for finding them).
  // Ragged calls whose cut this changed: 1.06 to 1.12 times faster on average, 2.4 at
  // best; the worst, of D = 32, take 1.4 times as long.
  if (several && P > 0 && most > 1 && B * T < (1 << 30)) {
    for (int64_t k = 1; k <= 8; ++k) {
      const int64_t z = (k * cus / HKV - B) / 2 - (int64_t)(0.3 * std::sqrt((double)B));
      if (z < 1 || z + B > 65535) continue;
      const double of_piece = std::max(std::ceil(0.6 * (double)(B * T) / (double)z), (double)waves);
      if (of_piece >= (double)T) continue;
      const double n = (double)items * std::max(0.6 * (double)T / of_piece + 0.5, 1.0);
      const double us = SPREAD_US + rows_cost(c, n, of_piece, mixed, (int64_t)std::ceil((double)T / of_piece), cus, waves, rows, D);
      if (us < least) least = us, r.spread = (int)z;
    }
    if (r.spread > 0) {
      r.steps = waves;
      r.pieces = r.spread + (int)B;
    }
  }
  return r;
}

// The plans of the last sizes: the layers of a step ask for the same one, and the
// estimates take 2 us of a call's host time.
RowsPlan rows_plan(int64_t B, int64_t SQ, int64_t SN, int64_t P, int64_t H, int64_t HKV, int64_t D, bool ragged, int cus) {
  struct Entry {
    int64_t key[9];
    RowsPlan plan;
  };
  static thread_local Entry kept[8] = {};  // (D = 0 is no call's)
  const int64_t key[9] = {B, SQ, SN, P, H, HKV, D, ragged ? 1 : 0, cus};
  uint64_t x = 0;
  for (int i = 0; i < 9; ++i) x = (x ^ (uint64_t)key[i]) * 0x9e3779b97f4a7c15ull;
  Entry& e = kept[x >> 61];
  if (memcmp(e.key, key, sizeof(key)) != 0) {
    e.plan = make_rows_plan(B, SQ, SN, P, H, HKV, D, ragged, cus);
    memcpy(e.key, key, sizeof(key));
  }
  return e.plan;
}

int64_t rows_ws_bytes(const RowsPlan& r, int64_t B, int64_t HKV, int64_t D) {
  if (r.pieces <= 1) return 0;
  return QIK_ATTN_WS_CTL_BYTES + (r.spread > 0 ? 1 : B) * HKV * r.nrt * r.pieces * rows_slot((int)D, 1 << r.row_bits);
}

// ceil(2^32 / d) for the kernel's quotient, 0 for 1
unsigned reciprocal(int64_t d) { return d == 1 ? 0u : (unsigned)((((int64_t)1 << 32) + d - 1) / d); }

struct MxLaunch {
  RowsPlan rows;
  Launch many;
  int64_t ws_bytes;
};

bool no_work(const qik_attn_args& a) { return a.B == 0 || a.H == 0 || a.SQ == 0; }

int plan_mx(const qik_mx_attn_args* x, MxLaunch* l) {
  const qik_attn_args& a = x->a;
  l->ws_bytes = 0;
  const int64_t G = a.H / x->HKV;
  // (without slab rows the lengths are not read)
  l->rows = rows_plan(a.B, a.SQ, a.SN, a.P, a.H, x->HKV, a.D, a.P > 0 && x->lengths != nullptr, device_cus());
  if (l->rows.few) {
    l->ws_bytes = rows_ws_bytes(l->rows, a.B, x->HKV, a.D);
    return QIK_OK;
  }
  const int st = plan_launch(a.B * x->HKV, a.SQ * G, a.D, (a.flags & QIK_UNIFORM_L) != 0, mx_kernels_of(&a), true, &l->many);
  l->ws_bytes = l->many.ws_bytes;
  return st;
}

}  // namespace qik

extern "C" {

int qik_mx_slab_store(const qik_mx_slab_store_args* a, void* stream) {
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  if (a->abi_version != QIK_ABI_VERSION) return QIK_ERR_ABI_VERSION;
  if (a->dtype != QIK_DTYPE_BF16 && a->dtype != QIK_DTYPE_FP16) return QIK_ERR_DTYPE;
  if (a->D != 32 && a->D != 64 && a->D != 128 && a->D != 256) return QIK_ERR_HEAD_DIM;
  if (a->B < 0 || a->S < 0 || a->H < 0 || a->capacity < 0 || a->B > INT_MAX || a->S > INT_MAX || a->H > INT_MAX ||
      a->capacity > INT_MAX)
    return QIK_ERR_SHAPE;
  if (a->B == 0 || a->S == 0 || a->H == 0) return QIK_OK;
  if (a->B * a->H > INT_MAX || a->B * a->H > INT_MAX / a->S) return QIK_ERR_SHAPE;
  if (a->k == nullptr || a->v == nullptr) return QIK_ERR_NULL_ARG;
  if (!qik::aligned_to(a->k, 16) || !qik::aligned_to(a->v, 16) || !qik::stride_ok(a->stride_k, a->B, a->S, a->H, 8) ||
      !qik::stride_ok(a->stride_v, a->B, a->S, a->H, 8))
    return QIK_ERR_ALIGN;
  int st = qik_mx_slabs::slab_status(a->k_dst, a->B, a->capacity, a->H, a->D);
  if (st == QIK_OK) st = qik_mx_slabs::slab_status(a->v_dst, a->B, a->capacity, a->H, a->D);
  if (st != QIK_OK) return st;
  const bool grow = a->lengths != nullptr && a->lengths == a->at;
  if (grow && a->arrivals == nullptr) return QIK_ERR_NULL_ARG;

  qik_mx_slabs::StoreParams p;
  memset(&p, 0, sizeof(p));
  const void* src[2] = {a->k, a->v};
  const qik_mx_slab* dst[2] = {&a->k_dst, &a->v_dst};
  const int64_t* st_in[2] = {a->stride_k, a->stride_v};
  for (int w = 0; w < 2; ++w) {
    p.src[w] = static_cast<const char*>(src[w]);
    p.codes[w] = static_cast<unsigned char*>(dst[w]->codes);
    p.scales[w] = static_cast<unsigned char*>(dst[w]->scales);
    for (int i = 0; i < 3; ++i) {
      p.ss[w][i] = st_in[w][i] * 2;
      p.sc[w][i] = dst[w]->stride_codes[i];
      p.se[w][i] = dst[w]->stride_scales[i];
    }
  }
  p.at = a->at;
  p.lengths = a->lengths;
  p.arrivals = grow ? a->arrivals : nullptr;
  p.B = (int)a->B;
  p.S = (int)a->S;
  p.H = (int)a->H;
  p.capacity = (int)a->capacity;
  const auto fn = a->dtype == QIK_DTYPE_FP16 ? qik_mx_slabs::pick_store<true>(a->D) : qik_mx_slabs::pick_store<false>(a->D);
  void* kargs[] = {&p};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(fn), qik_mx_slabs::slab_grid(a->B, a->S, a->H, a->D),
                                       dim3(qik_mx_slabs::THREADS), kargs, 0, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? QIK_OK : QIK_ERR_LAUNCH;
}

int qik_mx_slab_load(const qik_mx_slab_load_args* a, void* stream) {
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  if (a->abi_version != QIK_ABI_VERSION) return QIK_ERR_ABI_VERSION;
  if (a->dtype != QIK_DTYPE_BF16 && a->dtype != QIK_DTYPE_FP16) return QIK_ERR_DTYPE;
  if (a->D != 32 && a->D != 64 && a->D != 128 && a->D != 256) return QIK_ERR_HEAD_DIM;
  if (a->B < 0 || a->P < 0 || a->H < 0 || a->B > INT_MAX || a->P > INT_MAX || a->H > INT_MAX) return QIK_ERR_SHAPE;
  if (a->B == 0 || a->P == 0 || a->H == 0) return QIK_OK;
  if (a->B * a->H > INT_MAX) return QIK_ERR_SHAPE;
  if (a->k == nullptr || a->v == nullptr) return QIK_ERR_NULL_ARG;
  if (!qik::aligned_to(a->k, 16) || !qik::aligned_to(a->v, 16)) return QIK_ERR_ALIGN;
  int st = qik_mx_slabs::slab_status(a->k_src, a->B, a->P, a->H, a->D);
  if (st == QIK_OK) st = qik_mx_slabs::slab_status(a->v_src, a->B, a->P, a->H, a->D);
  if (st != QIK_OK) return st;

  qik_mx_slabs::LoadParams p;
  memset(&p, 0, sizeof(p));
  const qik_mx_slab* src[2] = {&a->k_src, &a->v_src};
  void* out[2] = {a->k, a->v};
  for (int w = 0; w < 2; ++w) {
    p.codes[w] = static_cast<const unsigned char*>(src[w]->codes);
    p.scales[w] = static_cast<const unsigned char*>(src[w]->scales);
    p.out[w] = static_cast<char*>(out[w]);
    for (int i = 0; i < 3; ++i) {
      p.sc[w][i] = src[w]->stride_codes[i];
      p.se[w][i] = src[w]->stride_scales[i];
    }
  }
  p.lengths = a->lengths;
  p.B = (int)a->B;
  p.P = (int)a->P;
  p.H = (int)a->H;
  const auto fn = a->dtype == QIK_DTYPE_FP16 ? qik_mx_slabs::pick_load<true>(a->D) : qik_mx_slabs::pick_load<false>(a->D);
  void* kargs[] = {&p};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(fn), qik_mx_slabs::slab_grid(a->B, a->P, a->H, a->D),
                                       dim3(qik_mx_slabs::THREADS), kargs, 0, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? QIK_OK : QIK_ERR_LAUNCH;
}

int qik_mx_attn_validate(const qik_mx_attn_args* x) {
  if (x == nullptr) return QIK_ERR_NULL_ARG;
  const qik_attn_args& a = x->a;
  if (a.abi_version != QIK_ABI_VERSION || a.reserved0 != 0 || a.reserved1 != 0) return QIK_ERR_ABI_VERSION;
  if (a.dtype != QIK_DTYPE_BF16 && a.dtype != QIK_DTYPE_FP16) return QIK_ERR_DTYPE;
  if (a.D != 32 && a.D != 64 && a.D != 128 && a.D != 256) return QIK_ERR_HEAD_DIM;
  const int64_t lim = (int64_t)INT_MAX;
  if (a.B < 0 || a.SQ < 0 || a.SN < 0 || a.P < 0 || a.H < 0 || x->HKV < 0) return QIK_ERR_SHAPE;
  if (a.SQ > lim || a.SN > lim || a.P > lim || a.H > lim || a.P + a.SN > lim || a.B > lim) return QIK_ERR_SHAPE;
  if ((a.flags & ~(QIK_HAS_CACHE | QIK_HAS_KEY_VALID | QIK_UNIFORM_L)) != 0) return QIK_ERR_SHAPE;
  const bool has_cache = (a.flags & QIK_HAS_CACHE) != 0;
  const bool has_kv = (a.flags & QIK_HAS_KEY_VALID) != 0;
  const bool uniform = (a.flags & QIK_UNIFORM_L) != 0;
  if (has_cache != (a.P > 0) || a.k_cache != nullptr || a.v_cache != nullptr) return QIK_ERR_CACHE;
  if (a.v_scale != nullptr) return QIK_ERR_FP8_SCALE;
  if (has_kv != (a.key_valid != nullptr) || a.debug_tiles != nullptr) return QIK_ERR_NULL_ARG;
  if (qik::no_work(a)) return QIK_OK;
  if (x->HKV < 1 || a.H % x->HKV != 0) return QIK_ERR_SHAPE;
  // row blocks of a KV head's rows, and all of them
  const int64_t G = a.H / x->HKV;
  if (a.SQ > lim / G) return QIK_ERR_SHAPE;
  const int64_t tiles = qik::cdiv64(a.SQ * G, qik::ROWS_M);
  if (a.B > lim / x->HKV || a.B * x->HKV > lim / tiles) return QIK_ERR_SHAPE;

  if (a.q == nullptr || a.out == nullptr) return QIK_ERR_NULL_ARG;
  if (a.SN > 0 && (a.k_new == nullptr || a.v_new == nullptr)) return QIK_ERR_NULL_ARG;
  if (!uniform && a.prefix_lengths == nullptr) return QIK_ERR_NULL_ARG;
  if (!qik::aligned_to(a.q, 16) || !qik::aligned_to(a.out, 16)) return QIK_ERR_ALIGN;
  if (!qik::stride_ok(a.stride_q, a.B, a.SQ, a.H, 8) || !qik::stride_ok(a.stride_out, a.B, a.SQ, a.H, 8)) return QIK_ERR_ALIGN;
  if (a.SN > 0) {
    if (!qik::aligned_to(a.k_new, 16) || !qik::aligned_to(a.v_new, 16)) return QIK_ERR_ALIGN;
    if (!qik::stride_ok(a.stride_k_new, a.B, a.SN, x->HKV, 8) || !qik::stride_ok(a.stride_v_new, a.B, a.SN, x->HKV, 8))
      return QIK_ERR_ALIGN;
    const int64_t tile_lim = ((int64_t)1 << 31) / qik::BN;
    if (a.SN > 1 && (a.stride_k_new[1] < a.D || a.stride_v_new[1] < a.D)) return QIK_ERR_ALIGN;
    if (a.stride_k_new[1] * 2 >= tile_lim || a.stride_v_new[1] * 2 >= tile_lim) return QIK_ERR_SHAPE;
  }
  if (has_cache) {
    int st = qik_mx_slabs::slab_status(x->k_slab, a.B, a.P, x->HKV, a.D);
    if (st == QIK_OK) st = qik_mx_slabs::slab_status(x->v_slab, a.B, a.P, x->HKV, a.D);
    if (st != QIK_OK) return st;
  }
  return QIK_OK;
}

int qik_mx_attn_workspace_size(const qik_mx_attn_args* x, int64_t* bytes) {
  if (bytes == nullptr) return QIK_ERR_NULL_ARG;
  *bytes = 0;
  const int st = qik_mx_attn_validate(x);
  if (st != QIK_OK || qik::no_work(x->a)) return st;
  qik::MxLaunch l;
  const int pst = qik::plan_mx(x, &l);
  if (pst == QIK_OK) *bytes = l.ws_bytes;
  return pst;
}

int qik_mx_attn_fwd(const qik_mx_attn_args* x, void* ws, int64_t ws_bytes, void* stream) {
  const int st = qik_mx_attn_validate(x);
  if (st != QIK_OK || qik::no_work(x->a)) return st;
  const qik_attn_args& a = x->a;
  qik::MxLaunch l;
  const int pst = qik::plan_mx(x, &l);
  if (pst != QIK_OK) return pst;
  if (l.ws_bytes > 0 && (ws == nullptr || !qik::aligned_to(ws, 256) || ws_bytes < l.ws_bytes)) return QIK_ERR_WORKSPACE;
  const int64_t G = a.H / x->HKV;
  const float qk_scale = a.sm_scale * 1.44269504088896340736f;
  const bool cache = a.P > 0;
  const int64_t none[3] = {0, 0, 0};
  const int64_t* kc = cache ? x->k_slab.stride_codes : none;
  const int64_t* vc = cache ? x->v_slab.stride_codes : none;
  const int64_t* ks = cache ? x->k_slab.stride_scales : none;
  const int64_t* vs = cache ? x->v_slab.stride_scales : none;
  const void* fn;
  void* kargs[1];
  dim3 grid;
  unsigned threads;
  qik::RowsParams r;
  qik::MxParams p;
  if (l.rows.few) {
    memset(&r, 0, sizeof(r));
    r.q = static_cast<const char*>(a.q);
    r.k_new = static_cast<const char*>(a.k_new);
    r.v_new = static_cast<const char*>(a.v_new);
    if (cache) {
      r.k_codes = static_cast<const char*>(x->k_slab.codes);
      r.v_codes = static_cast<const char*>(x->v_slab.codes);
      r.k_scales = static_cast<const char*>(x->k_slab.scales);
      r.v_scales = static_cast<const char*>(x->v_slab.scales);
      r.lengths = x->lengths;
    }
    r.L = a.prefix_lengths;
    r.key_valid = a.key_valid;
    r.out = static_cast<char*>(a.out);
    if (l.ws_bytes > 0) {
      r.ctl = static_cast<unsigned*>(ws);
      r.part = reinterpret_cast<float*>(static_cast<char*>(ws) + QIK_ATTN_WS_CTL_BYTES);
    }
    for (int i = 0; i < 3; ++i) {
      r.sq[i] = a.stride_q[i];
      r.skn[i] = a.stride_k_new[i];
      r.svn[i] = a.stride_v_new[i];
      r.so[i] = a.stride_out[i];
      r.skc[i] = kc[i];
      r.svc[i] = vc[i];
      r.sks[i] = ks[i];
      r.svs[i] = vs[i];
    }
    r.svalid_b = a.stride_valid_b;
    r.sL_b = x->stride_lengths_b;
    r.R = (int)(a.SQ * G);
    r.SN = (int)a.SN;
    r.P = (int)a.P;
    r.HKV = (int)x->HKV;
    r.G = (int)G;
    r.KV = (int)(a.P + a.SN);
    r.uniform = (a.flags & QIK_UNIFORM_L) ? 1 : 0;
    r.steps = l.rows.steps;
    r.B = (int)a.B;
    r.spread = l.rows.spread;
    r.by_G = qik::reciprocal(G);
    r.by_HKV = qik::reciprocal(x->HKV);
    r.row_bits = l.rows.row_bits;
    r.qk_scale = qk_scale;
    fn = reinterpret_cast<const void*>(qik::rows_kernel_of(&a, l.rows.mt, l.rows.spread > 0));
    grid = dim3((unsigned)(x->HKV * l.rows.nrt), l.rows.spread > 0 ? 1u : (unsigned)a.B, (unsigned)l.rows.pieces);
    threads = 64u * (unsigned)qik::rows_waves((int)a.D, l.rows.mt);
    kargs[0] = &r;
  } else {
    if (l.many.grid == 0) return QIK_OK;
    memset(&p, 0, sizeof(p));
    p.q = static_cast<const char*>(a.q);
    p.k_new = static_cast<const char*>(a.k_new);
    p.v_new = static_cast<const char*>(a.v_new);
    if (cache) {
      p.k_cache = static_cast<const char*>(x->k_slab.codes);
      p.v_cache = static_cast<const char*>(x->v_slab.codes);
      p.k_scales = static_cast<const uint8_t*>(x->k_slab.scales);
      p.v_scales = static_cast<const uint8_t*>(x->v_slab.scales);
      p.lengths = x->lengths;
    }
    p.L = a.prefix_lengths;
    p.key_valid = a.key_valid;
    p.out = static_cast<char*>(a.out);
    if (l.ws_bytes > 0) {
      p.ctl = static_cast<unsigned*>(ws);
      p.ws_slots = static_cast<char*>(ws) + l.many.ctl_bytes;
    }
    for (int i = 0; i < 3; ++i) {
      p.sq[i] = a.stride_q[i];
      p.skn[i] = a.stride_k_new[i];
      p.svn[i] = a.stride_v_new[i];
      p.so[i] = a.stride_out[i];
      p.skc[i] = kc[i];
      p.svc[i] = vc[i];
      p.sks[i] = ks[i];
      p.svs[i] = vs[i];
    }
    p.svalid_b = a.stride_valid_b;
    p.sL_b = x->stride_lengths_b;
    p.SQ = (int)(a.SQ * G);
    p.SN = (int)a.SN;
    p.P = (int)a.P;
    p.H = (int)x->HKV;
    p.KV = (int)(a.P + a.SN);
    p.has_cache = cache ? 1 : 0;
    p.has_key_valid = (a.flags & QIK_HAS_KEY_VALID) ? 1 : 0;
    p.uniform = (a.flags & QIK_UNIFORM_L) ? 1 : 0;
    p.qk_scale = qk_scale;
    p.plan = l.many.plan;
    p.G = (int)G;
    fn = l.many.fn;
    grid = dim3((unsigned)l.many.grid);
    threads = (unsigned)l.many.threads;
    kargs[0] = &p;
  }
  const hipError_t e = hipLaunchKernel(fn, grid, dim3(threads), kargs, 0, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? QIK_OK : QIK_ERR_LAUNCH;
}

int qik_mx_attn_plan(int64_t B, int64_t SQ, int64_t SN, int64_t P, int64_t H, int64_t HKV, int64_t D,
                     int32_t ragged, int32_t cus, int32_t* few, int32_t* row_tiles, int32_t* pieces) {
  if (few == nullptr || row_tiles == nullptr || pieces == nullptr) return QIK_ERR_NULL_ARG;
  if (B < 1 || SQ < 1 || SN < 0 || P < 0 || HKV < 1 || H < HKV || H % HKV != 0 || cus < 1) return QIK_ERR_SHAPE;
  if (D != 32 && D != 64 && D != 128 && D != 256) return QIK_ERR_HEAD_DIM;
  const qik::RowsPlan r = qik::rows_plan(B, SQ, SN, P, H, HKV, D, ragged != 0, cus);
  *few = r.few ? 1 : 0;
  *row_tiles = r.mt * r.nrt;
  *pieces = r.spread > 0 ? r.spread : r.pieces;
  return QIK_OK;
}

}  // extern "C"
