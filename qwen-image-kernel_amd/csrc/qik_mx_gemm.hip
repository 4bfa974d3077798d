// Product of microscaled operands on MI355X (gfx950): A in MXFP4 or MXFP8, W in
// MXFP4, on the scaled matrix instructions v_mfma_scale_f32_*_f8f6f4, which
// multiply each block of 32 by its two power-of-two scales as they sum it.
//
// Many rows (`tile_kernel`): a workgroup computes a BM x BN tile of out^T = W .
// A^T (first operand weight rows n, second activation rows m, so that a lane
// ends with 4 consecutive n of one row m per register quad).  Codes and scales
// reach LDS directly, two to four stages in flight, and the fragments of the
// next k-step are read while the matrix cores run on the current ones.
//
// Few rows (`rows_kernel`): every wave takes 16 or 32 weight rows and a share
// of K, loads the codes straight into registers and meets the others of its
// workgroup in LDS.  It is bound by the weight's bytes.  Of a token or a few, the
// workgroup quantises the elements itself: one launch.

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include <limits.h>
#include <algorithm>
#include <type_traits>
#include <utility>

#include "qik_mx.h"
#include "qik_mx_block.h"
#include "qik_tile.h"

namespace qik_mx {

using qik_tile::cdiv;
using qik_tile::choose_group_m;
using qik_tile::choose_plan;
using qik_tile::device_cus;
using qik_tile::dma16_at;
using qik_tile::dma4_at;
using qik_tile::GemmPlan;
using qik_tile::lds_ptr_t;
using qik_tile::rsrc_words;
using qik_tile::tile_origin;
using qik_tile::TileRun;
using qik_tile::TileShape;
using qik_tile::TileTable;
using qik_tile::wait_vmcnt;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int FMT_E4M3 = 0, FMT_E2M1 = 4;  // the instruction's operand formats

// A range of output columns computed with one tile shape.
struct MxRegion : TileRun {
  const unsigned char* w;   // weight row of the region's first column
  const unsigned char* ws;  // its group of scales
  const char* bias;         // its first bias element, or null
  char* out;                // its first output column
  int N;                    // columns in the region
  int wgs;                  // workgroups: tiles rounded up to a multiple of 8
};

struct MxGemmParams {
  const unsigned char* a;
  const unsigned char* as;
  int M, K, C;      // C = ceil(K / 256)
  int64_t lda, ldw;  // bytes
  int64_t ldc;       // elements
  bool fp16;         // type of bias and out
  bool vec;          // out's rows are at multiples of 16 bytes
  MxRegion r[2];     // columns [0, n1) with the larger tile, then [n1, N)
  int small_first;   // 1: region 1's workgroups come first in blockIdx order
  int ksplit;        // split launches: k-slices per tile (region 0 only)
  float* partial;    // split launches: [ksplit][M][ldp] fp32 sums of each slice
  int64_t ldp;       // N rounded up to 4
  unsigned row_magic;  // rows of elements: 2^32 / (K / 8), rounded up
};

// round to nearest even into bf16 or fp16
__device__ __forceinline__ unsigned short round16(float f, bool fp16) {
  asm volatile("" : "+v"(f));  // an fp32 value: no mixed-precision fma rounds it
  return fp16 ? __builtin_bit_cast(unsigned short, (_Float16)f) : __builtin_bit_cast(unsigned short, (__bf16)f);
}
__device__ __forceinline__ float widen16(unsigned short h, bool fp16) {
  return fp16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((unsigned)h << 16);
}
__device__ __forceinline__ float bias_at(const MxGemmParams& p, const MxRegion& rg, int n) {
  return rg.bias != nullptr && n < rg.N ? widen16(reinterpret_cast<const unsigned short*>(rg.bias)[n], p.fp16) : 0.0f;
}

__device__ __forceinline__ i32x8 operand(u32x4 lo, u32x4 hi) {
  return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// ---------------------------------------------------------------------------
// Tiles
// ---------------------------------------------------------------------------

template <int I>
using num = std::integral_constant<int, I>;

// f(num<0>) .. f(num<N - 1>)
template <class F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
  (f(num<I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
  each_of(f, std::make_integer_sequence<int, N>{});
}

// f(num<(kt - kb) % U>, kt) for kt of [kb, nk), nk > kb
template <class F, int... I>
__device__ __forceinline__ void stages_of(int kt, const int nk, F&& f, std::integer_sequence<int, I...>) {
  while (((f(num<I>{}, kt), ++kt < nk) && ...)) {
  }
}
template <int U, class F>
__device__ __forceinline__ void stages(const int kb, const int nk, F&& f) {
  stages_of(kb, nk, f, std::make_integer_sequence<int, U>{});
}

// Tile shape BM x BN, WGM x WGN waves, NS stages.  A stage holds 128 bytes of
// every A row (256 k of MXFP4, 128 of MXFP8), the W codes of the same k (128 or
// 64 bytes a row), and of every 32 rows the 256 bytes of scales of the 256 k
// around them.
template <int BM_, int BN_, int WGM_, int WGN_, int NS_, bool A8_, bool WS_>
struct Tile {
  static constexpr bool WS = WS_;  // fragments are read a whole stage at a time (gemm_tile)
  static constexpr bool A8 = A8_;
  static constexpr int BM = BM_, BN = BN_, NS = NS_;
  static constexpr int WGM = WGM_, WGN = WGN_;        // waves along m and n
  static constexpr int NW = WGM * WGN, NT = 64 * NW;
  static constexpr int WM = BM / WGM, WN = BN / WGN;  // wave tile
  static constexpr int MI = WM / 32, NJ = WN / 32;
  static constexpr int KV = A8 ? 128 : 256;           // k of a stage
  static constexpr int KS = KV / 64;                  // MFMA k-steps of a stage
  static constexpr int RA = 128, RW = A8 ? 64 : 128;  // bytes of a stage's row
  static constexpr int W_AT = BM * RA;                // stage: A codes, W codes, A scales, W scales
  static constexpr int S_AT = W_AT + BN * RW;
  static constexpr int SBLK = (BM + BN) / 32;
  static constexpr int STAGE = S_AT + SBLK * 256;
  static constexpr int AI = BM * RA / (1024 * NW);    // 1 KiB copies per wave and stage
  static constexpr int WI = BN * RW / (1024 * NW);
  static constexpr int SI = (SBLK + NW - 1) / NW;     // 256-byte copies
  static constexpr int COPIES = AI + WI + SI;
  static constexpr int BIAS_AT = NS * STAGE;          // behind the stages: the columns' bias, 16 bits each
  static constexpr int BIAS_COPIES = (BN * 2 + 255) / 256;
  static constexpr int LDS = BIAS_AT + 256 * BIAS_COPIES;
  static_assert(NW == 4 || NW == 8, "one or two waves per SIMD");
  static_assert(NS >= 2 && (NS - 1) * COPIES < 64, "the prologue's copies fit the vmcnt field");
  static_assert(LDS <= 160 * 1024, "the stages and the bias fit LDS");
  static_assert(BIAS_COPIES <= NW, "one copy of bias per wave");
  static_assert(AI * 1024 * NW == BM * RA && WI * 1024 * NW == BN * RW, "whole copies per wave");
  static_assert(MI * 32 == WM && NJ * 32 == WN, "whole MFMA blocks per wave");
  static_assert((BN & (BN - 1)) == 0, "the output staging's swizzle needs a power of two");
  static_assert(BM * BN * 2 <= NS * STAGE, "the output tile fits the stages");
};

// The tile's outputs, staged through LDS (the stages, once every copy has
// landed and every wave is done with them) so that a store writes whole rows:
// staged row ml keeps its 16-byte chunk c at c ^ (ml % CPR), which spreads a
// fragment's 32 rows over the banks.  Rows of out at other than multiples of 16
// bytes, and the last columns of an N that is no multiple of 8, are stored an
// element at a time.
template <class T>
__device__ __forceinline__ void store_tile(const MxGemmParams& p, const MxRegion& rg, const int m0, const int n0,
                                           const f32x16 (&acc)[T::NJ][T::MI], unsigned char* lds, const int wave,
                                           const int lane) {
  const int wm = wave % T::WGM, wn = wave / T::WGM;
  constexpr int RB = T::BN * 2;  // bytes of a staged row
  constexpr int CPR = RB / 16;   // 16-byte chunks per row
  constexpr int RPI = 64 / CPR;  // rows per store instruction
  // the bias was copied in whole dwords: an odd last element is read here
  const bool odd_end = (rg.N & 1) != 0 && n0 + T::BN >= rg.N;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < T::NJ; ++j) {
#pragma unroll
    for (int qd = 0; qd < 4; ++qd) {
      const int nl = wn * T::WN + j * 32 + qd * 8 + (lane >> 5) * 4;
      const u32x2 braw = *reinterpret_cast<const u32x2*>(lds + T::BIAS_AT + nl * 2);
      float bv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) bv[e] = widen16((unsigned short)(braw[e / 2] >> (16 * (e % 2))), p.fp16);
      if (odd_end && n0 + nl <= rg.N - 1 && n0 + nl + 4 > rg.N - 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n0 + nl + e == rg.N - 1) bv[e] = bias_at(p, rg, rg.N - 1);
      }
#pragma unroll
      for (int i = 0; i < T::MI; ++i) {
        const int ml = wm * T::WM + i * 32 + (lane & 31);
        unsigned short y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = round16(acc[j][i][qd * 4 + e] + bv[e], p.fp16);
        const u32x2 o = {(unsigned)y[0] | (unsigned)y[1] << 16, (unsigned)y[2] | (unsigned)y[3] << 16};
        *reinterpret_cast<u32x2*>(lds + ml * RB + ((nl >> 3) ^ (ml & (CPR - 1))) * 16 + (lane >> 5) * 8) = o;
      }
    }
  }
  __syncthreads();
  const int c = lane % CPR;
  const int n = n0 + c * 8;
#pragma unroll 4
  for (int r0 = wave * RPI; r0 < T::BM; r0 += T::NW * RPI) {
    const int ml = r0 + lane / CPR;
    const u32x4 v = *reinterpret_cast<const u32x4*>(lds + ml * RB + ((c ^ (ml & (CPR - 1))) * 16));
    const int m = m0 + ml;
    if (m >= p.M) continue;
    char* o = rg.out + (m * p.ldc + n) * 2;
    if (p.vec && n + 8 <= rg.N) {
      *reinterpret_cast<u32x4*>(o) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < rg.N) reinterpret_cast<unsigned short*>(o)[e] = (unsigned short)(v[e / 2] >> (16 * (e % 2)));
    }
  }
}

// The fp32 sums of one k-slice of a tile into p.partial, 4 columns of one row
// per lane and register quad.
template <class T>
__device__ __forceinline__ void store_partial(const MxGemmParams& p, const MxRegion& rg, const int m0, const int n0,
                                              const f32x16 (&acc)[T::NJ][T::MI], const int slice, const int wave,
                                              const int lane) {
  const int wm = wave % T::WGM, wn = wave / T::WGM;
  float* dst = p.partial + (int64_t)slice * p.M * p.ldp;
#pragma unroll
  for (int j = 0; j < T::NJ; ++j) {
#pragma unroll
    for (int qd = 0; qd < 4; ++qd) {
      const int n = n0 + wn * T::WN + j * 32 + qd * 8 + (lane >> 5) * 4;
#pragma unroll
      for (int i = 0; i < T::MI; ++i) {
        const int m = m0 + wm * T::WM + i * 32 + (lane & 31);
        if (m < p.M && n < rg.N)
          *reinterpret_cast<f32x4*>(dst + m * p.ldp + n) =
              f32x4{acc[j][i][qd * 4], acc[j][i][qd * 4 + 1], acc[j][i][qd * 4 + 2], acc[j][i][qd * 4 + 3]};
      }
    }
  }
}

// One BM x BN tile of region rg; bx counts the region's workgroups.  SPLIT: the
// sums of slice `slice` of the stages, into p.partial.  In LDS the 16-byte chunk c of a 128-byte row r sits at
// chunk c ^ (r / 2) % 8, of a 64-byte row at c ^ (r / 4) % 4: a fragment read
// (16 lanes on 16 consecutive rows, one chunk each) then touches all 64 banks
// once, and a 1 KiB copy writes one contiguous KiB.
//
// The matrix instruction is 32x32x64: lane l of a wave holds row l % 32.  Which
// k of memory a lane's k of an instruction stand for is free as long as both
// operands and the scales agree.  MXFP4: lane half h = l / 32 takes block 4 h +
// s of the stage's 8 at k-step s, so its four scales are four consecutive bytes
// and the instruction picks byte s.  With MXFP8 activations an E4M3 lane holds
// two runs of 16 k, h and 2 + h of the step's four, its scale that of block h;
// half h takes W's block 2 s + h and shifts its scale bytes down by h.
template <class T, bool SPLIT>
__device__ __forceinline__ void gemm_tile(const MxGemmParams& p, const MxRegion& rg, const int bx, unsigned char* lds,
                                          const int slice) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // uniform: copy targets go to SGPRs
  const int wm = wave % T::WGM, wn = wave / T::WGM;
  int m0, n0;
  if (!tile_origin(rg, T::BM, T::BN, bx, m0, n0)) return;
  const int mrows = min(T::BM, p.M - m0), nrows = min(T::BN, rg.N - n0);

  // copies: one of A fills 8 rows (lane l: row l / 8, chunk l % 8), one of W 8
  // rows of 128 bytes or 16 of 64, one of scales the 256 bytes of 32 rows.  The
  // rows of a wave's copies are a multiple of 16 apart, so one chunk serves all.
  const int arow = wave * 8 + (lane >> 3);
  const int achunk = ((lane & 7) ^ ((arow >> 1) & 7)) * 16;
  const int wrow = T::A8 ? wave * 16 + (lane >> 2) : arow;
  const int wchunk = T::A8 ? ((lane & 3) ^ ((wrow >> 2) & 3)) * 16 : achunk;
  constexpr int WROWS = 1024 / T::RW;  // rows of a copy of W
  uint32_t aoff[T::AI], woff[T::WI];
#pragma unroll
  for (int i = 0; i < T::AI; ++i) aoff[i] = (uint32_t)((arow + 8 * T::NW * i) * (int)p.lda);
#pragma unroll
  for (int i = 0; i < T::WI; ++i) woff[i] = (uint32_t)((wrow + WROWS * T::NW * i) * (int)p.ldw);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
  const unsigned char* abase = p.a + (int64_t)m0 * p.lda;
  const unsigned char* wbase = rg.w + (int64_t)n0 * p.ldw;
  const int group = p.C * 256;  // bytes of a row group's scales
  const unsigned char* asbase = p.as + (int64_t)(m0 / 32) * group;
  const unsigned char* wsbase = rg.ws + (int64_t)(n0 / 32) * group;
  const int agroups = (mrows + 31) / 32, wgroups = (nrows + 31) / 32;
  const int nkall = (p.K + T::KV - 1) / T::KV;
  const int kb = SPLIT ? (int)((int64_t)nkall * slice / p.ksplit) : 0;
  const int nk = SPLIT ? (int)((int64_t)nkall * (slice + 1) / p.ksplit) : nkall;  // end of the stages

  // The copies of one step.  Resources hold for all of them (rows past the
  // tile's last are out of range: zeros) and only lanes' offsets move on: with
  // one wave per SIMD the instructions of a stage are what a small tile waits
  // for, and resources made anew each step were a third of them.  Past the end of
  // K, or of the slice, a lane's chunk would read the next row, so its offset
  // gets the top bit (out of range); every step issues the same copies, so the
  // waits stay uniform.  Scales past the end are of other blocks and meet no code.
  const int rowa = T::A8 ? p.K : p.K / 2, roww = p.K / 2;
  const u32x4 ra = rsrc_words(abase, (uint32_t)((mrows - 1) * (int)p.lda + rowa));
  const u32x4 rw = rsrc_words(wbase, (uint32_t)((nrows - 1) * (int)p.ldw + roww));
  const uint32_t aend = (uint32_t)min(rowa, nk * T::RA), wend = (uint32_t)min(roww, nk * T::RW);
  u32x4 rs[T::SI];
  uint32_t soff[T::SI], sdst[T::SI];
  const uint32_t cdst = lds0 + (uint32_t)wave * 1024;
#pragma unroll
  for (int i = 0; i < T::SI; ++i) {
    // the surplus waves of the last round copy the last group again
    const int b = min(wave + T::NW * i, T::SBLK - 1);
    const bool of_a = b < T::BM / 32;
    rs[i] = rsrc_words(of_a ? asbase : wsbase, (uint32_t)((of_a ? agroups : wgroups) * group));
    soff[i] = (uint32_t)((of_a ? b : b - T::BM / 32) * group + lane * 4);
    sdst[i] = lds0 + (uint32_t)(T::S_AT + b * 256);
  }
  struct Step {
    uint32_t ka, kw;    // offset of the lane's chunk in its row, or out of range
    uint32_t ks;        // of the stage's scales in a row group's
  };
  auto prepare = [&](const int kt) __attribute__((always_inline)) {
    Step sc;
    sc.ka = (uint32_t)(kt * T::RA + achunk);
    sc.ka = sc.ka < aend ? sc.ka : 0x80000000u;
    sc.kw = sc.ka;
    if constexpr (T::A8) {
      sc.kw = (uint32_t)(kt * T::RW + wchunk);
      sc.kw = sc.kw < wend ? sc.kw : 0x80000000u;
    }
    sc.ks = (uint32_t)((T::A8 ? kt >> 1 : kt) * 256);
    return sc;
  };
  // copies [C0, C1) of the step into stage ST
  auto issue = [&](auto st_tag, const Step& sc, auto c0_tag, auto c1_tag) __attribute__((always_inline)) {
    constexpr int ST = decltype(st_tag)::value * T::STAGE, C0 = decltype(c0_tag)::value, C1 = decltype(c1_tag)::value;
    auto copy = [&](auto i_tag) __attribute__((always_inline)) {
      constexpr int i = C0 + decltype(i_tag)::value;
      if constexpr (i < T::AI) {
        dma16_at<ST + T::NW * i * 1024>(ra, cdst, aoff[i] + sc.ka);
      } else if constexpr (i < T::AI + T::WI) {
        constexpr int k = i - T::AI;
        dma16_at<ST + T::W_AT + T::NW * k * 1024>(rw, cdst, woff[k] + sc.kw);
      } else {
        constexpr int k = i - T::AI - T::WI;
        dma4_at<ST>(rs[k], sdst[k], soff[k] + sc.ks);
      }
    };
    each<C1 - C0>(copy);
  };

  // fragment reads: lane l reads row l % 32 of a 32-row block; the offsets hold
  // the wave's place, so that a stage and a block are an instruction's constant
  const int frow = lane & 31, half = lane >> 5;
  constexpr int ACH = T::A8 ? 2 : 1;  // chunks of an A fragment
  uint32_t fa_off[T::KS][ACH], fw_off[T::KS];
#pragma unroll
  for (int s = 0; s < T::KS; ++s) {
    const int c0 = T::A8 ? 4 * s + half : 4 * half + s;
    const uint32_t r0 = (uint32_t)((wm * T::WM + frow) * 128);
    fa_off[s][0] = r0 + (uint32_t)((c0 ^ ((frow >> 1) & 7)) * 16);
    if constexpr (T::A8) fa_off[s][ACH - 1] = r0 + (uint32_t)(((c0 + 2) ^ ((frow >> 1) & 7)) * 16);
    fw_off[s] = (uint32_t)((wn * T::WN + frow) * T::RW) +
                (uint32_t)(T::A8 ? ((2 * s + half) ^ ((frow >> 2) & 3)) * 16 : (c0 ^ ((frow >> 1) & 7)) * 16);
  }
  const uint32_t sc_off = (uint32_t)(frow * 8 + (T::A8 ? 0 : half * 4));
  const uint32_t sa_off = sc_off + (uint32_t)(wm * T::MI * 256), sw_off = sc_off + (uint32_t)(wn * T::NJ * 256);

  // fragments in two buffers, of a k-step each, or of a whole stage (T::WS)
  constexpr int SLOTS = T::WS ? T::KS : 1;
  u32x4 fa[2][SLOTS][T::MI][ACH], fw[2][SLOTS][T::NJ];
  int sa[T::MI], sw[T::NJ], nsa[T::MI], nsw[T::NJ];
  constexpr int NRD = T::MI * ACH + T::NJ;  // reads of a k-step's fragments
  constexpr int NSR = T::MI + T::NJ;        // reads of a stage's scales
  auto read_frag = [&](const int stage, const int s, const int r, const int buf) __attribute__((always_inline)) {
    const unsigned char* st = lds + stage * T::STAGE;
    const int slot = T::WS ? s : 0;
    if (r < T::MI * ACH) {
      const int f = r / ACH;
      fa[buf][slot][f][r % ACH] = *reinterpret_cast<const u32x4*>(st + f * 32 * T::RA + fa_off[s][r % ACH]);
    } else {
      const int f = r - T::MI * ACH;
      fw[buf][slot][f] = *reinterpret_cast<const u32x4*>(st + T::W_AT + f * 32 * T::RW + fw_off[s]);
    }
  };
  auto read_scale = [&](const int stage, const int odd, const int r) __attribute__((always_inline)) {
    const int b = r < T::MI ? r : T::BM / 32 + r - T::MI;
    const unsigned char* at = lds + stage * T::STAGE + T::S_AT + b * 256;
    const int v = *reinterpret_cast<const int*>(at + (r < T::MI ? sa_off : sw_off) + (T::A8 ? odd * 4 : 0));
    if (r < T::MI) nsa[r] = v;
    else nsw[r - T::MI] = v;
  };
  auto take_scales = [&]() __attribute__((always_inline)) {
    const int sh = T::A8 ? 8 * half : 0;
#pragma unroll
    for (int i = 0; i < T::MI; ++i) sa[i] = T::A8 ? (int)((unsigned)nsa[i] >> sh) : nsa[i];
#pragma unroll
    for (int j = 0; j < T::NJ; ++j) sw[j] = T::A8 ? (int)((unsigned)nsw[j] >> sh) : nsw[j];
  };

  f32x16 acc[T::NJ][T::MI];
#pragma unroll
  for (int j = 0; j < T::NJ; ++j)
#pragma unroll
    for (int i = 0; i < T::MI; ++i) acc[j][i] = f32x16{};

  // prologue: the bias (zeros without one), then every stage in flight, stage 0
  // published, its first fragments read
  if constexpr (!SPLIT) {
    const int b = wave % T::BIAS_COPIES;
    const u32x4 rb = rsrc_words(reinterpret_cast<const unsigned char*>(rg.bias) + n0 * 2,
                                rg.bias != nullptr ? (uint32_t)(nrows / 2 * 4) : 0u);
    dma4_at<T::BIAS_AT>(rb, lds0 + (uint32_t)(b * 256), (uint32_t)(b * 256 + lane * 4));
  }
  each<T::NS>([&](auto s_tag) __attribute__((always_inline)) {
    issue(s_tag, prepare(kb + decltype(s_tag)::value), num<0>{}, num<T::COPIES>{});
  });
  wait_vmcnt<(T::NS - 1) * T::COPIES>();
  __syncthreads();
#pragma unroll
  for (int r = 0; r < SLOTS * NRD; ++r) read_frag(0, r / NRD, r % NRD, 0);
#pragma unroll
  for (int r = 0; r < NSR; ++r) read_scale(0, kb & 1, r);

  constexpr int NMF = T::NJ * T::MI;  // MFMAs of a k-step
  const u32x4 zero = {0u, 0u, 0u, 0u};
  auto mfma = [&](auto s_tag, const int idx, const int buf) __attribute__((always_inline)) {
    constexpr int S = decltype(s_tag)::value;
    constexpr int OP = T::A8 ? 2 * S : S;  // the scale's byte
    const int j = idx / T::MI, i = idx % T::MI, slot = T::WS ? S : 0;
    acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
        operand(fw[buf][slot][j], zero), operand(fa[buf][slot][i][0], T::A8 ? fa[buf][slot][i][ACH - 1] : zero), acc[j][i],
        FMT_E2M1, T::A8 ? FMT_E4M3 : FMT_E2M1, OP, sw[j], OP, sa[i]);
  };

  // The loops are unrolled over the stages: a stage's LDS addresses are constants.
  if constexpr (!T::WS) {
    // k-step S of a stage on fragments S % 2, with the reads of the next k-step
    // into the others between its MFMAs.  The last one (COPY) issues its first
    // PRE MFMAs before the wait for the next stage's copies and the barrier,
    // which publishes that stage and releases this one (every wave has read all
    // of it; the barrier's LDS fence waits for those reads), then the reads of
    // the next stage and the copies of the stage after next into this one's
    // memory.
    constexpr int PRE = 2 < NMF ? 2 : 1;
    auto kstep = [&](auto s_tag, auto st_tag, const int next_odd, const Step& sc) __attribute__((always_inline)) {
      constexpr int S = decltype(s_tag)::value;
      constexpr int stage = decltype(st_tag)::value, next = (stage + 1) % T::NS;
      constexpr bool COPY = S == T::KS - 1;
      // reads (and copies) after MFMAs [R0, R0 + H)
      constexpr int R0 = COPY ? (NMF > PRE ? PRE : PRE - 1) : 0;
      constexpr int H = COPY ? NMF - R0 : (NMF >= 2 ? NMF / 2 : 1);
      constexpr int RD = NRD + (COPY ? NSR : 0);
      each<NMF>([&](auto idx_tag) __attribute__((always_inline)) {
        constexpr int idx = decltype(idx_tag)::value;
        mfma(s_tag, idx, S % 2);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (COPY) {
          if (idx == PRE - 1) {
            wait_vmcnt<(T::NS - 2) * T::COPIES>();  // the next stage's copies have landed
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        if (idx >= R0 && idx < R0 + H) {
#pragma unroll
          for (int r = (idx - R0) * RD / H; r < (idx - R0 + 1) * RD / H; ++r) {
            if (r < NRD) read_frag(COPY ? next : stage, COPY ? 0 : S + 1, r, (S + 1) % 2);
            else read_scale(next, next_odd, r - NRD);
          }
          if constexpr (COPY && idx >= R0 && idx < R0 + H)
            issue(st_tag, sc, num<(idx - R0) * T::COPIES / H>{}, num<(idx - R0 + 1) * T::COPIES / H>{});
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    stages<T::NS>(kb, nk, [&](auto st_tag, const int kt) __attribute__((always_inline)) {
      const Step none = {};
      take_scales();
      kstep(num<0>{}, st_tag, 0, none);
      if constexpr (T::KS == 4) {
        kstep(num<1>{}, st_tag, 0, none);
        kstep(num<2>{}, st_tag, 0, none);
      }
      __builtin_amdgcn_sched_barrier(0);
      const Step sc = prepare(kt + T::NS);
      kstep(num<T::KS - 1>{}, st_tag, (kt + 1) & 1, sc);
    });
  } else {
    // A tile of few MFMAs per k-step is bound by the latency of its fragment
    // reads (about 130 cycles a k-step at one MFMA of 32), so a whole stage of
    // fragments is read at a time, one stage ahead: all MFMAs of a stage run on
    // registers, and the stage's memory is free for the copies of the stage NS
    // later as soon as the barrier says that every wave has its fragments.
    auto stage_step = [&](auto u_tag, const int kt) __attribute__((always_inline)) {
      constexpr int BUF = decltype(u_tag)::value % 2, st = decltype(u_tag)::value % T::NS, nst = (st + 1) % T::NS;
      constexpr int TOTAL = T::KS * NMF;
      constexpr int PRE = TOTAL / 4 < 2 ? 1 : 2;
      constexpr int H = TOTAL - PRE;  // MFMAs with reads and copies beside them
      constexpr int RD = T::KS * NRD + NSR;
      take_scales();
      const Step sc = prepare(kt + T::NS);
      auto run = [&](auto s_tag) __attribute__((always_inline)) {
        constexpr int S = decltype(s_tag)::value;
        each<NMF>([&](auto i_tag) __attribute__((always_inline)) {
          constexpr int i = decltype(i_tag)::value, idx = S * NMF + i;
          mfma(s_tag, i, BUF);
          __builtin_amdgcn_sched_barrier(0);
          if (idx == PRE - 1) {
            wait_vmcnt<(T::NS - 2) * T::COPIES>();  // the next stage's copies have landed
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
          }
          if constexpr (idx >= PRE - 1 && idx < PRE - 1 + H) {
            constexpr int q = idx - (PRE - 1);
#pragma unroll
            for (int r = q * RD / H; r < (q + 1) * RD / H; ++r) {
              if (r < T::KS * NRD) read_frag(nst, r / NRD, r % NRD, BUF ^ 1);
              else read_scale(nst, (kt + 1) & 1, r - T::KS * NRD);
            }
            issue(num<st>{}, sc, num<q * T::COPIES / H>{}, num<(q + 1) * T::COPIES / H>{});
          }
          __builtin_amdgcn_sched_barrier(0);
        });
      };
      each<T::KS>(run);
    };
    stages<T::NS % 2 == 0 ? T::NS : 2 * T::NS>(kb, nk, stage_step);  // both buffers' turns too
  }
  wait_vmcnt<0>();  // the copies of the steps past the end still land in their stages
  if constexpr (SPLIT) store_partial<T>(p, rg, m0, n0, acc, slice, wave, lane);
  else store_tile<T>(p, rg, m0, n0, acc, lds, wave, lane);
}

// Region 0 (T1 tiles) and region 1 (T2 tiles), one after the other in blockIdx
// order; the smaller tiles fill the CUs that the big ones' last round leaves
// free (small_first: the other way round, when it is estimated no slower).
template <class T1, class T2>
__global__ void __launch_bounds__(T1::NT) __attribute__((amdgpu_waves_per_eu(T1::NW / 4, T1::NW / 4)))
tile_kernel(const MxGemmParams p) {
  static_assert(T1::NT == T2::NT, "one workgroup size per launch");
  constexpr int L1 = T1::LDS, L2 = T2::LDS;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[L1 > L2 ? L1 : L2];
  const int bx = blockIdx.x;
  const int off0 = p.small_first ? p.r[1].wgs : 0;  // first workgroup of each region
  const int off1 = p.small_first ? 0 : p.r[0].wgs;
  if (bx >= off0 && bx < off0 + p.r[0].wgs) gemm_tile<T1, false>(p, p.r[0], bx - off0, lds, 0);
  else gemm_tile<T2, false>(p, p.r[1], bx - off1, lds, 0);
}

// Split launch: workgroup b sums slice b / wgs of tile b % wgs (wgs is a
// multiple of 8, so a tile's slices run on one XCD).
template <class T>
__global__ void __launch_bounds__(T::NT) __attribute__((amdgpu_waves_per_eu(T::NW / 4, T::NW / 4)))
split_kernel(const MxGemmParams p) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[T::LDS];
  const int wgs = p.r[0].wgs;
  gemm_tile<T, true>(p, p.r[0], blockIdx.x % wgs, lds, blockIdx.x / wgs);
}

// out = round(the slices' sums in slice order + bias), 4 outputs per thread.
__global__ void __launch_bounds__(256) join_kernel(const MxGemmParams p) {
  const MxRegion& rg = p.r[0];
  const int per_row = (int)(p.ldp / 4);
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (g >= (int64_t)p.M * per_row) return;
  const int m = (int)(g / per_row);
  const int n = (int)(g - (int64_t)m * per_row) * 4;
  const int64_t slice = (int64_t)p.M * p.ldp;
  const float* src = p.partial + m * p.ldp + n;
  f32x4 y = *reinterpret_cast<const f32x4*>(src);
  for (int k = 1; k < p.ksplit; ++k) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(src + k * slice);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += v[e];
  }
  unsigned short o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = round16(y[e] + bias_at(p, rg, n + e), p.fp16);
  unsigned short* to = reinterpret_cast<unsigned short*>(rg.out) + m * p.ldc + n;
  if (p.vec && n + 4 <= rg.N) {
    *reinterpret_cast<u32x2*>(to) = u32x2{(unsigned)o[0] | (unsigned)o[1] << 16, (unsigned)o[2] | (unsigned)o[3] << 16};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < rg.N) to[e] = o[e];
  }
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

// Where the rows of A come from: codes, or elements of a type that the
// workgroup quantises into LDS first.
enum { SRC_CODES = -1 };  // else QIK_DTYPE_BF16, _FP16 or _FP32

// Most elements of A that a workgroup quantises for itself (takes_raw).
constexpr int RAW_ELEMS = 32768;

// KW waves of a workgroup share K by chunks of 256; BC chunks of W are in
// flight ahead of the ones that are multiplied.
template <int SRC, bool A8, int MB, int NB, int KW>
__global__ void __launch_bounds__(64 * KW) rows_kernel(const MxGemmParams p) {
  constexpr bool RAW = SRC != SRC_CODES;
  constexpr int BC = NB == 1 ? 4 : 2;
  constexpr int CODE_BYTES = RAW ? RAW_ELEMS / (A8 ? 1 : 2) : 16, SCALE_BYTES = RAW ? RAW_ELEMS / 32 : 16;
  __shared__ f32x4 red[KW][NB * MB][64];
  __shared__ __attribute__((aligned(16))) unsigned char lcodes[CODE_BYTES];
  __shared__ unsigned char lscales[SCALE_BYTES];
  const MxRegion& rg = p.r[0];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * NB), m0 = blockIdx.y * (16 * MB);
  const u32x4 zero = {0u, 0u, 0u, 0u};

  // rows past the end repeat the last one; their sums are not stored
  const unsigned char* wr[NB];
  const unsigned char* wsr[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int n = min(n0 + j * 16 + r, rg.N - 1);
    wr[j] = rg.w + n * p.ldw;
    wsr[j] = rg.ws + (int64_t)(n >> 5) * p.C * 256 + (n & 31) * 8;
  }
  const unsigned char* ar[MB];   // a row's codes
  const unsigned char* asr[MB];  // its scales
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int m = min(m0 + i * 16 + r, p.M - 1);
    ar[i] = RAW ? lcodes + m * (A8 ? p.K : p.K / 2) : p.a + m * p.lda;
    asr[i] = RAW ? lscales + m * (p.K / 32) : p.as + (int64_t)(m >> 5) * p.C * 256 + (m & 31) * 8;
  }

  f32x4 acc[NB][MB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int c0 = p.C * wave / KW, c1 = p.C * (wave + 1) / KW;
  u32x4 wf[2][BC][2][NB];
  u32x2 wsc[2][BC][NB];
  // a lane's blocks past K are zeros (loaded from the row's start, then cleared)
  auto load_w = [&](const int buf, const int c) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < BC; ++b) {
      if (c + b >= c1) break;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = (c + b) * 256 + s * 128 + g * 32;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(wr[j] + (k < p.K ? k / 2 : 0));
          wf[buf][b][s][j] = k < p.K ? v : zero;
        }
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) wsc[buf][b][j] = *reinterpret_cast<const u32x2*>(wsr[j] + (c + b) * 256);
    }
  };
  // what a lane holds of 16 rows of A for step s of chunk c, and its scale
  struct AFrag {
    u32x4 lo, hi;
    int scale;
  };
  auto load_a = [&](const int i, const int c, const int s, const u32x2 asc) __attribute__((always_inline)) {
    AFrag f;
    const int kb = c * 256 + s * 128 + g * 32;  // the block of the lane's scale
    if constexpr (A8) {
      const int k = c * 256 + s * 128 + g * 16;
      const u32x4 lo = *reinterpret_cast<const u32x4*>(ar[i] + (k < p.K ? k : 0));
      const u32x4 hi = *reinterpret_cast<const u32x4*>(ar[i] + (k + 64 < p.K ? k + 64 : 0));
      f.lo = k < p.K ? lo : zero;
      f.hi = k + 64 < p.K ? hi : zero;
    } else {
      const u32x4 lo = *reinterpret_cast<const u32x4*>(ar[i] + (kb < p.K ? kb / 2 : 0));
      f.lo = kb < p.K ? lo : zero;
      f.hi = zero;
    }
    if constexpr (RAW) f.scale = kb < p.K ? asr[i][kb / 32] : 0;
    else f.scale = (int)(asc[s] >> (8 * g));
    return f;
  };
  auto multiply = [&](const int buf, const int c) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < BC; ++b) {
      if (c + b >= c1) break;
      AFrag a[2][MB];
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        u32x2 asc = {0u, 0u};
        if constexpr (!RAW) asc = *reinterpret_cast<const u32x2*>(asr[i] + (c + b) * 256);
#pragma unroll
        for (int s = 0; s < 2; ++s) a[s][i] = load_a(i, c + b, s, asc);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < MB; ++i)
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                operand(wf[buf][b][s][j], zero), operand(a[s][i].lo, a[s][i].hi), acc[j][i], FMT_E2M1,
                A8 ? FMT_E4M3 : FMT_E2M1, 0, (int)(wsc[buf][b][j][s] >> (8 * g)), 0, a[s][i].scale);
    }
  };
  load_w(0, c0);
  if constexpr (RAW) {  // while the first weights are on their way
    constexpr int FMT = A8 ? QIK_MXFP8 : QIK_MXFP4;
    constexpr int IT = 4;  // vectors of a thread in flight
    const int per_row = p.K / 8, total = p.M * per_row;  // vectors of 8; a multiple of 4 a row: whole quads
    for (int v0 = threadIdx.x; v0 < total; v0 += IT * 64 * KW) {
      Raw8<SRC> x[IT];
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int v = v0 + i * 64 * KW, m = (int)__umulhi((unsigned)v, p.row_magic);
        x[i] = Raw8<SRC>{};
        if (v < total)
          x[i] = load8<SRC, false>(reinterpret_cast<const char*>(p.a) +
                                   (m * p.lda + (v - m * per_row) * 8) * elem_bytes<SRC>());
      }
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int v = v0 + i * 64 * KW;
        if (v >= total) continue;
        float f[8];
        unpack8<SRC>(x[i], f);
        unsigned w0, w1;
        const unsigned byte = block_codes<FMT>(f, w0, w1);
        store_codes<FMT>(lcodes, v, w0, w1);  // rows lie one behind the other
        if ((v & 3) == 0) lscales[v / 4] = (unsigned char)byte;
      }
    }
    __syncthreads();
  }
  for (int c = c0; c < c1; c += 2 * BC) {
    load_w(1, c + BC);
    multiply(0, c);
    load_w(0, c + 2 * BC);
    multiply(1, c + BC);
  }

#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) red[wave][j * MB + i][lane] = acc[j][i];
  __syncthreads();
  for (int e = threadIdx.x; e < NB * MB * 256; e += 64 * KW) {
    const int nl = e % (16 * NB), ml = e / (16 * NB);
    const int n = n0 + nl, m = m0 + ml;
    if (n >= rg.N || m >= p.M) continue;
    const int tile = (nl / 16) * MB + ml / 16, ln = (nl % 16) / 4 * 16 + ml % 16;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < KW; ++k) y += red[k][tile][ln][nl % 4];  // the shares in order
    reinterpret_cast<unsigned short*>(rg.out)[m * p.ldc + n] = round16(y + bias_at(p, rg, n), p.fp16);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

inline bool aligned_to(const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) % a) == 0; }

inline bool known_sizes(int64_t M, int64_t N, int64_t K) {
  return M >= 0 && M <= ((int64_t)1 << 30) && N >= 1 && N < ((int64_t)1 << 28) && K >= 32 && K <= 262144 && K % 32 == 0;
}

// with_a: a, a_scales and lda are checked too
int validate_gemm(const qik_mx_gemm_args* a, bool with_a) {
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  if (a->abi_version != QIK_ABI_VERSION || a->reserved0 != 0) return QIK_ERR_ABI_VERSION;
  if (a->out_dtype != QIK_DTYPE_BF16 && a->out_dtype != QIK_DTYPE_FP16) return QIK_ERR_DTYPE;
  if (a->a_format != QIK_MXFP4 && a->a_format != QIK_MXFP8) return QIK_ERR_DTYPE;
  if (!known_sizes(a->M, a->N, a->K)) return QIK_ERR_SHAPE;
  const int64_t row_a = a->a_format == QIK_MXFP4 ? a->K / 2 : a->K;
  // a tile's rows must be addressable by a 31-bit buffer offset
  if (a->ldw < a->K / 2 || a->ldw > INT_MAX / 256 || a->ldc < a->N || a->ldc > ((int64_t)1 << 40)) return QIK_ERR_SHAPE;
  if (with_a && (a->lda < row_a || a->lda > INT_MAX / 256)) return QIK_ERR_SHAPE;
  if (a->M == 0) return QIK_OK;
  if (a->w == nullptr || a->w_scales == nullptr || a->out == nullptr) return QIK_ERR_NULL_ARG;
  if (!aligned_to(a->w, 16) || !aligned_to(a->w_scales, 16) || a->ldw % 16 != 0) return QIK_ERR_ALIGN;
  if (!aligned_to(a->out, 2) || !aligned_to(a->bias, 4)) return QIK_ERR_ALIGN;
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
  p.M = (int)a->M;
  p.K = (int)a->K;
  p.C = (int)cdiv(a->K, 256);
  p.lda = a->lda;
  p.ldw = a->ldw;
  p.ldc = a->ldc;
  p.fp16 = a->out_dtype == QIK_DTYPE_FP16;
  p.vec = aligned_to(a->out, 16) && a->ldc % 8 == 0;
  return p;
}

// Region of columns [c0, c1) with tiles of bm x bn (of `abytes` and `wbytes` a stage).
int set_region(MxRegion& rg, const qik_mx_gemm_args* a, int64_t c0, int64_t c1, int bm, int bn, int abytes, int wbytes) {
  rg.w = static_cast<const unsigned char*>(a->w) + c0 * a->ldw;
  rg.ws = static_cast<const unsigned char*>(a->w_scales) + c0 / 32 * cdiv(a->K, 256) * 256;  // c0: whole tiles
  rg.bias = a->bias != nullptr ? static_cast<const char*>(a->bias) + c0 * 2 : nullptr;
  rg.out = static_cast<char*>(a->out) + c0 * 2;
  rg.N = (int)(c1 - c0);
  rg.ntm = (int)cdiv(a->M, bm);
  rg.ntn = (int)cdiv(c1 - c0, bn);
  rg.group_m = choose_group_m(rg.ntm, rg.ntn, abytes, wbytes);
  const int64_t wgs = cdiv((int64_t)rg.ntm * rg.ntn, 8) * 8;
  if (wgs > (int64_t)INT_MAX / 16) return QIK_ERR_SHAPE;
  rg.wgs = (int)wgs;
  return QIK_OK;
}
template <class T>
int set_region(MxRegion& rg, const qik_mx_gemm_args* a, int64_t c0, int64_t c1) {
  return set_region(rg, a, c0, c1, T::BM, T::BN, T::BM * T::RA, T::BN * T::RW);
}

int launch(const void* fn, dim3 grid, int threads, MxGemmParams& p, hipStream_t s) {
  if ((uint64_t)grid.x * (unsigned)threads >> 32 != 0) return QIK_ERR_SHAPE;  // more than a launch holds
  void* args[] = {&p};
  return hipLaunchKernel(fn, grid, dim3((unsigned)threads), args, 0, s) == hipSuccess ? QIK_OK : QIK_ERR_LAUNCH;
}

template <class T1, class T2>
int launch_tiles(MxGemmParams& p, const qik_mx_gemm_args* a, int64_t n1, hipStream_t s) {
  int st = set_region<T1>(p.r[0], a, 0, n1);
  if (st == QIK_OK) st = set_region<T2>(p.r[1], a, n1, a->N);
  if (st != QIK_OK) return st;
  return launch((const void*)tile_kernel<T1, T2>, dim3((unsigned)p.r[0].wgs + (unsigned)p.r[1].wgs), T1::NT, p, s);
}

template <class T>
int launch_split(MxGemmParams& p, const qik_mx_gemm_args* a, hipStream_t s) {
  int st = set_region<T>(p.r[0], a, 0, a->N);
  if (st != QIK_OK) return st;
  st = launch((const void*)split_kernel<T>, dim3((unsigned)p.r[0].wgs * (unsigned)p.ksplit), T::NT, p, s);
  if (st != QIK_OK) return st;
  return launch((const void*)join_kernel, dim3((unsigned)cdiv(a->M * (p.ldp / 4), 256)), 256, p, s);
}

template <int SRC, bool A8, int MB, int NB, int KW>
int launch_rows_shape(MxGemmParams& p, const qik_mx_gemm_args* a, hipStream_t s) {
  const int st = set_region(p.r[0], a, 0, a->N, 16 * MB, 16 * NB, 0, 0);
  if (st != QIK_OK) return st;
  return launch((const void*)rows_kernel<SRC, A8, MB, NB, KW>, dim3((unsigned)p.r[0].ntn, (unsigned)p.r[0].ntm), 64 * KW, p,
                s);
}

// Weight rows (in 16s) and waves of a workgroup.  Past 8192 columns there is a
// workgroup of 16 rows for every second wave slot: four waves each (1 x 12288 x
// 4096 7.8 us, 9.3 with eight), and past 16384, or where they are to be quantised,
// 32 rows that share the codes of A (9 x 24576 x 1024 6.7 us with 16 rows, 5.7 with
// 32; 16 x 12288 x 1024 3.8 and 4.2).  Below, eight waves share a long K (1 x 4096 x 12288 8.6 us, 11.2 with
// four; 1 x 4096 x 1536 3.0 and 3.1, x 1024 2.8 and 2.7), or the quantising of
// elements, which goes by threads.
struct RowsPlan {
  int nb, kw;
};
RowsPlan choose_rows(int64_t M, int64_t N, int64_t K, bool raw) {
  return {M > 8 && N > (raw ? 8192 : 16384) ? 2 : 1, N > 8192 || (!raw && K <= 4 * 256) ? 4 : 8};
}

template <int SRC, bool A8, int MB>
int launch_rows(MxGemmParams& p, const qik_mx_gemm_args* a, hipStream_t s) {
  const RowsPlan plan = choose_rows(a->M, a->N, a->K, SRC != SRC_CODES);
  // more than 16 rows of codes come here with up to 4096 columns (takes_rows), so
  // never in pairs of 16; of elements past 8192 columns always in pairs
  if constexpr (MB == 1 || SRC != SRC_CODES) {
    if (plan.nb == 2) return launch_rows_shape<SRC, A8, MB, 2, 4>(p, a, s);
  }
  if constexpr (MB == 1 || SRC == SRC_CODES) {
    if (plan.kw == 4) return launch_rows_shape<SRC, A8, MB, 1, 4>(p, a, s);
  }
  return launch_rows_shape<SRC, A8, MB, 1, 8>(p, a, s);
}

// Time of a tile of each shape (qik_tile.h), for A in MXFP4 and in MXFP8: fitted
// to launches of one round on MI355X, each shape forced, 64 to 8704 rows, N x K
// from 1024 x 1024 to 12288 x 4096 and 4096 x 12288, operands from memory.  A
// launch that keeps all its CUs busy takes a quarter longer than its tile times
// (the card's power limit lowers the clock: 1.7 GHz at 8192 x 8192 x 8192);
// tiles of 64 rows, which wait more than they multiply, do not.
enum { T256x256, T256x128, T128x256, T128x128, T192x256, T192x128, T64x128, T64x64, NSHAPES };
static const TileShape kShapes[2][NSHAPES] = {
    {{256, 256, 8.75, 1.16}, {256, 128, 6.25, 0.58, 1.4}, {128, 256, 6.35, 0.55, 1.4}, {128, 128, 4.35, 0.37, 0.7},
     {192, 256, 7.5, 0.965}, {192, 128, 5.45, 0.495, 0.9}, {64, 128, 4.15, 0.29, 0.0}, {64, 64, 3.75, 0.18, 0.0}},
    {{256, 256, 9.15, 0.93}, {256, 128, 5.9, 0.525, 1.2}, {128, 256, 5.95, 0.505, 1.2}, {128, 128, 4.05, 0.335, 0.6},
     {192, 256, 7.8, 0.705}, {192, 128, 5.1, 0.445, 0.8}, {64, 128, 3.65, 0.27, 0.0}, {64, 64, 3.45, 0.165, 0.0}}};
constexpr int NPAIRS = 5;
static const int kPairs[NPAIRS][2] = {{T256x256, T256x128}, {T256x256, T128x128}, {T128x256, T128x128},
                                      {T192x256, T192x128}, {T64x128, T64x64}};
static const TileTable kTables[2] = {{kShapes[0], kPairs, NPAIRS, 0, 0.5, 0.5},
                                     {kShapes[1], kPairs, NPAIRS, 0, 0.5, 0.5}};

enum { SPLIT64, SPLIT128 };
// How a product of more than a few rows is launched: slices > 1 splits K.
struct MxPlan {
  int pair;
  int64_t n1;
  bool small_first;
  int slices, split;
};

// A K split pays for a launch with few tiles and a long K: S slices of 64 x 64 or
// 128 x 128 tiles, as many as the CUs run in one round (all slices of a tile on
// one XCD), and a second launch that joins them: 3 us, and the fp32 sums written
// and read at about 4 TB/s (64 x 4096 x 12288 13.0 us unsplit, 12.2 in 4 slices,
// 14.8 in 8, with MXFP8 rows 19.8, 12.6 and 15.7; 200 x 1024 x 8192 with MXFP8 rows
// 13.9 and 10.8 in 4; 203 x 4096 x 12288 14.0 and 22.0 in 4 of 128 x 128).
MxPlan choose(int64_t M, int64_t N, int64_t K, bool a8, int cus) {
  const int64_t steps = cdiv(K, a8 ? 128 : 256), P = std::max(1, (cus > 0 ? cus : 256) / 8);
  const GemmPlan g = choose_plan(kTables[a8], M, N, steps, cus);
  MxPlan plan = {g.pair, g.n1, g.small_first, 1, SPLIT64};
  double best = 0.95 * g.t;
  for (int which = SPLIT64; which <= SPLIT128; ++which) {
    const TileShape& t = kShapes[a8][which == SPLIT64 ? T64x64 : T128x128];
    const int64_t per_xcd = cdiv(cdiv(M, t.bm) * cdiv(N, t.bn), 8);
    const int64_t most = std::min<int64_t>({P / per_xcd, 8, steps / 4});
    for (int64_t S = 2; S <= most; ++S) {
      const double us = t.time(cdiv(steps, S)) + 3.0 + (double)(S * M * N) * 8.0 / 4e6;
      if (us < best) {
        best = us;
        plan.slices = (int)S;
        plan.split = which;
      }
    }
  }
  return plan;
}

template <bool A8>
int launch_plan(MxGemmParams& p, const qik_mx_gemm_args* a, const MxPlan& plan, float* partial, hipStream_t s) {
  typedef Tile<256, 256, 2, 4, A8 ? 3 : 2, A8, false> C256x256;
  typedef Tile<256, 128, 2, 4, 3, A8, true> C256x128;
  typedef Tile<128, 256, 2, 4, 3, A8, true> C128x256;
  typedef Tile<128, 128, 2, 4, 3, A8, true> C128x128;
  typedef Tile<192, 256, 2, 4, A8 ? 3 : 2, A8, A8> C192x256;
  typedef Tile<192, 128, 2, 4, 3, A8, true> C192x128;
  typedef Tile<64, 128, 1, 4, 3, A8, true> C64x128;
  typedef Tile<64, 64, 2, 2, 4, A8, true> C64x64;
  if (plan.slices > 1) {
    p.ksplit = plan.slices;
    p.partial = partial;
    p.ldp = cdiv(a->N, 4) * 4;
    return plan.split == SPLIT64 ? launch_split<C64x64>(p, a, s) : launch_split<C128x128>(p, a, s);
  }
  p.small_first = plan.small_first ? 1 : 0;
  switch (plan.pair) {
    case 0: return launch_tiles<C256x256, C256x128>(p, a, plan.n1, s);
    case 1: return launch_tiles<C256x256, C128x128>(p, a, plan.n1, s);
    case 2: return launch_tiles<C128x256, C128x128>(p, a, plan.n1, s);
    case 3: return launch_tiles<C192x256, C192x128>(p, a, plan.n1, s);
    default: return launch_tiles<C64x128, C64x64>(p, a, plan.n1, s);
  }
}

// Few rows: the tiles of 64 would multiply mostly padding.  They do better all
// the same where N has tiles for most CUs and K is long, or where K is so long
// that splitting it over workgroups pays (us, rows then tiles: 1 x 4096 x 12288
// 8.6 / 10.1, 8 x 512 x 16384 8.6 / 7.6, 8 x 12288 x 2048 5.7 / 6.0 and x 4096 8.4 /
// 7.9; 16 x 4096 x 8192 7.4 / 9.7 and with MXFP8 rows x 12288 11.9 / 11.3, 16 x
// 12288 x 1024 4.1 / 4.5 and x 2048 6.5 / 6.1; 32 x 4096 x 6144 7.6 / 7.9 and x 8192
// 9.4 / 9.0, with MXFP8 rows x 4096 7.3 / 8.0 and x 6144 10.3 / 9.8, 32 x 5120 x
// 2048 5.3 / 4.8).
bool takes_rows(int64_t M, int64_t N, int64_t K, bool a8) {
  const bool narrow = N <= 4096;
  if (M <= 8) return narrow ? K <= 12288 : N * K <= (1 << 25);
  if (M <= 16) return narrow ? K <= 8192 : N * K <= (1 << 24);
  return M <= 32 && narrow && K <= (a8 ? 4096 : 6144);
}

// A linear whose workgroups each quantise all of x for themselves saves a
// launch: up to 2 us in a graph, 4 us of host time in a loop of calls.  It costs
// what a CU's workgroups quantise, about 2.5 us for 32768 elements.  One launch and
// two, called in a loop: 1 x 4096 x 4096 7.6 / 11.4 us, 32 x 4096 x 1024 7.5 / 12.0,
// 4 x 12288 x 4096 9.7 / 11.8, 17 x 5001 x 1504 7.5 / 12.1, with MXFP8 8.3 / 12.1; in
// a graph 4.3 / 5.9, 5.4 / 5.7, 10.4 / 9.9, 6.2 / 7.2 and 8.7 / 7.8.  The limits go
// by the loop; a graph of the third and the last would do 5 and 12% better with
// two.
bool takes_raw(const qik_mx_gemm_args* a) {
  if (a->M * a->K > RAW_ELEMS || (a->M > 16 && (a->M > 32 || a->N * a->K > (1 << 24)))) return false;
  const int64_t wgs = cdiv(a->N, 16 * choose_rows(a->M, a->N, a->K, true).nb);
  return cdiv(wgs, 256) * a->M * a->K <= 2 * RAW_ELEMS;
}

// How a call is launched, and the bytes of its slices' sums.
struct Launch {
  bool rows;  // the few-rows kernel, else by plan
  MxPlan plan;
  int64_t partial_bytes;
};
Launch plan_launch(int64_t M, int64_t N, int64_t K, int32_t a_format, int cus) {
  const bool a8 = a_format == QIK_MXFP8;
  Launch l = {takes_rows(M, N, K, a8), {0, 0, false, 1, SPLIT64}, 0};
  if (l.rows) return l;
  l.plan = choose(M, N, K, a8, cus);
  if (l.plan.slices > 1) l.partial_bytes = (int64_t)l.plan.slices * M * cdiv(N, 4) * 4 * (int64_t)sizeof(float);
  return l;
}
Launch plan_launch(const qik_mx_gemm_args* a) { return plan_launch(a->M, a->N, a->K, a->a_format, device_cus()); }

template <bool A8>
int launch_gemm(const qik_mx_gemm_args* a, const Launch& l, float* partial, hipStream_t s) {
  MxGemmParams p = gemm_params(a);
  if (l.rows) return a->M <= 16 ? launch_rows<SRC_CODES, A8, 1>(p, a, s) : launch_rows<SRC_CODES, A8, 2>(p, a, s);
  return launch_plan<A8>(p, a, l.plan, partial, s);
}
int launch_gemm(const qik_mx_gemm_args* a, const Launch& l, float* partial, hipStream_t s) {
  return a->a_format == QIK_MXFP8 ? launch_gemm<true>(a, l, partial, s) : launch_gemm<false>(a, l, partial, s);
}

template <int SRC>
int launch_raw(const qik_mx_linear_args* l, hipStream_t s) {
  MxGemmParams p = gemm_params(&l->g);
  p.a = static_cast<const unsigned char*>(l->x);
  p.lda = l->ldx;  // elements
  // v / (K / 8) = umulhi(v, magic) for v < RAW_ELEMS / 8 and K / 8 from 4 to 4096:
  // the product is off by less than v (K / 8) / 2^32 < 1 / (K / 8)
  p.row_magic = (unsigned)((((uint64_t)1 << 32) + p.K / 8 - 1) / (p.K / 8));
  if (l->g.a_format == QIK_MXFP8)
    return p.M <= 16 ? launch_rows<SRC, true, 1>(p, &l->g, s) : launch_rows<SRC, true, 2>(p, &l->g, s);
  return p.M <= 16 ? launch_rows<SRC, false, 1>(p, &l->g, s) : launch_rows<SRC, false, 2>(p, &l->g, s);
}

inline int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// bytes of x's codes and scales in a linear's workspace
int64_t code_bytes(const qik_mx_gemm_args* g) { return round256(g->M * (g->a_format == QIK_MXFP4 ? g->K / 2 : g->K)); }
int64_t scale_bytes(const qik_mx_gemm_args* g) { return cdiv(g->M, 32) * cdiv(g->K, 256) * 256; }

}  // namespace qik_mx

extern "C" {

int qik_mx_gemm_workspace_size(const qik_mx_gemm_args* a, int64_t* bytes) {
  using namespace qik_mx;
  if (bytes == nullptr) return QIK_ERR_NULL_ARG;
  *bytes = 0;
  const int st = validate_gemm(a, true);
  if (st != QIK_OK || a->M == 0) return st;
  *bytes = plan_launch(a).partial_bytes;
  return QIK_OK;
}

int qik_mx_gemm(const qik_mx_gemm_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace qik_mx;
  const int st = validate_gemm(a, true);
  if (st != QIK_OK || a->M == 0) return st;
  const Launch l = plan_launch(a);
  if (l.partial_bytes > 0 &&
      (workspace == nullptr || workspace_bytes < l.partial_bytes || !aligned_to(workspace, 256)))
    return QIK_ERR_WORKSPACE;
  return launch_gemm(a, l, static_cast<float*>(workspace), static_cast<hipStream_t>(stream));
}

int qik_mx_gemm_plan(int64_t M, int64_t N, int64_t K, int32_t a_format, int32_t cus, int32_t* plan, int64_t* n1) {
  using namespace qik_mx;
  if (plan == nullptr || n1 == nullptr) return QIK_ERR_NULL_ARG;
  if (a_format != QIK_MXFP4 && a_format != QIK_MXFP8) return QIK_ERR_DTYPE;
  if (!known_sizes(M, N, K) || M < 1) return QIK_ERR_SHAPE;
  const Launch l = plan_launch(M, N, K, a_format, cus > 0 ? cus : 256);
  const TileShape* shapes = kShapes[a_format == QIK_MXFP8];
  *n1 = N;
  if (l.rows) {
    const RowsPlan r = choose_rows(M, N, K, false);
    const int32_t v[6] = {M <= 16 ? 16 : 32, 16 * r.nb, r.kw, 0, 0, 0};
    memcpy(plan, v, sizeof(v));
  } else if (l.plan.slices > 1) {
    const TileShape& t = shapes[l.plan.split == SPLIT64 ? T64x64 : T128x128];
    const int32_t v[6] = {t.bm, t.bn, t.bm, t.bn, 0, l.plan.slices};
    memcpy(plan, v, sizeof(v));
  } else {
    const TileShape &t1 = shapes[kPairs[l.plan.pair][0]], &t2 = shapes[kPairs[l.plan.pair][1]];
    const int32_t v[6] = {t1.bm, t1.bn, t2.bm, t2.bn, l.plan.small_first ? 1 : 0, 1};
    memcpy(plan, v, sizeof(v));
    *n1 = l.plan.n1;
  }
  return QIK_OK;
}

// workspace of a linear: the split's sums, x's codes, x's scales
int qik_mx_linear_workspace_size(const qik_mx_linear_args* a, int64_t* bytes) {
  using namespace qik_mx;
  if (bytes == nullptr) return QIK_ERR_NULL_ARG;
  *bytes = 0;
  const int st = validate_linear(a);
  if (st != QIK_OK || a->g.M == 0) return st;
  if (!takes_raw(&a->g)) *bytes = round256(plan_launch(&a->g).partial_bytes) + code_bytes(&a->g) + scale_bytes(&a->g);
  return QIK_OK;
}

int qik_mx_linear(const qik_mx_linear_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace qik_mx;
  const int st = validate_linear(a);
  if (st != QIK_OK || a->g.M == 0) return st;
  if (takes_raw(&a->g)) {
    const hipStream_t s = static_cast<hipStream_t>(stream);
    switch (a->x_dtype) {
      case QIK_DTYPE_BF16: return launch_raw<QIK_DTYPE_BF16>(a, s);
      case QIK_DTYPE_FP16: return launch_raw<QIK_DTYPE_FP16>(a, s);
      default: return launch_raw<QIK_DTYPE_FP32>(a, s);
    }
  }
  const Launch l = plan_launch(&a->g);
  const int64_t sums = round256(l.partial_bytes), codes = code_bytes(&a->g);
  const int64_t need = sums + codes + scale_bytes(&a->g);
  if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 256)) return QIK_ERR_WORKSPACE;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  qik_mx_gemm_args g = a->g;
  g.a = ws + sums;
  g.a_scales = ws + sums + codes;
  g.lda = g.a_format == QIK_MXFP4 ? g.K / 2 : g.K;
  qik_mx_quant_args q;
  memset(&q, 0, sizeof(q));
  q.abi_version = QIK_ABI_VERSION;
  q.dtype = a->x_dtype;
  q.format = g.a_format;
  q.x = a->x;
  q.codes = ws + sums;
  q.scales = ws + sums + codes;
  q.M = g.M;
  q.K = g.K;
  q.ldx = a->ldx;
  const int qs = qik_mx_quantize(&q, stream);
  if (qs != QIK_OK) return qs;
  return launch_gemm(&g, l, reinterpret_cast<float*>(ws), static_cast<hipStream_t>(stream));
}

}  // extern "C"
