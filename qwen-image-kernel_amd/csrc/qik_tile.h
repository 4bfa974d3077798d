// What the tiled products share: copies from global memory straight into LDS,
// the buffer resources that bound them and the wait for them; the order of the
// tiles; and the host's choice of tile shapes for a launch.
#ifndef QIK_TILE_H
#define QIK_TILE_H

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

namespace qik_tile {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) void* lds_ptr_t;

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 64 lanes x 16 B global -> LDS (buffer_load_dwordx4 ... lds): lane l's 16
// bytes land at LDS byte lds_addr + 16*l.  Asm, so the compiler neither moves
// the fragment reads around it nor waits for it; the main loop waits for the
// copies itself (vmcnt) before the barrier that publishes a stage.
__device__ __forceinline__ void dma16(u32x4 rsrc, uint32_t lds_addr, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rsrc) : "m0");
}
// The same to LDS byte lds_addr + AT, and with 4 bytes a lane: 256 contiguous
// bytes of LDS.
template <uint32_t AT>
__device__ __forceinline__ void dma16_at(u32x4 rsrc, uint32_t lds_addr, uint32_t voff) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rsrc), "i"(AT) : "m0", "scc");
}
template <uint32_t AT>
__device__ __forceinline__ void dma4_at(u32x4 rsrc, uint32_t lds_addr, uint32_t voff) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rsrc), "i"(AT) : "m0", "scc");
}
#pragma clang diagnostic pop

// Wave-uniform buffer resource over [base, base + bytes): loads at or past
// `bytes` return zeros.
__device__ __forceinline__ u32x4 rsrc_words(const unsigned char* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)base;
  return u32x4{(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, bytes, 0x00020000u};
}

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt field");
  // vmcnt in bits 3:0 and 15:14, expcnt (7) and lgkmcnt (63) left alone
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (0x7 << 4) | (0x3f << 8));
}

// The tiles of one region of the output and their order.
struct TileRun {
  int ntm, ntn;  // tiles along m and n
  int group_m;   // tile rows per group of the tile order
};

// Origin of the tile of workgroup bx of region rg (bx % 8 is the XCD: every
// region starts at a multiple of 8): XCD x takes a contiguous run of the tile
// order, which walks group_m tile rows at a time.  False for a padding
// workgroup.
__device__ __forceinline__ bool tile_origin(const TileRun& rg, const int bm, const int bn, const int bx, int& m0,
                                            int& n0) {
  const int T = rg.ntm * rg.ntn;
  const int x = bx & 7, s = bx >> 3;
  const int q = T >> 3, r = T & 7;
  if (s >= q + (x < r ? 1 : 0)) return false;
  const int t = x * q + min(x, r) + s;
  const int gsz_full = rg.group_m * rg.ntn;
  const int g = t / gsz_full;
  const int first = g * rg.group_m;
  const int gm = min(rg.group_m, rg.ntm - first);
  const int tr = t - g * gsz_full;
  m0 = (first + tr % gm) * bm;
  n0 = (tr / gm) * bn;
  return true;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// CUs of the current device (0 if the runtime cannot say), cached per device
inline int device_cus() {
  static int cache[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  if (dev >= 0 && dev < 64) {
    const int c = __atomic_load_n(&cache[dev], __ATOMIC_RELAXED);
    if (c > 0) return c;
  }
  int cus = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
  if (dev >= 0 && dev < 64) __atomic_store_n(&cache[dev], cus, __ATOMIC_RELAXED);
  return cus;
}

// A tile shape and the time of a tile, in us: t0 (prologue, output, the
// launch's share) + t1 per stage of K.
struct TileShape {
  int bm, bn;
  double t0, t1;
  double load = 1.0;  // its share of the table's load_slope
  double time(int64_t steps) const { return t0 + t1 * (double)steps; }
};

// The shapes of a product, the (big, small) pairs a launch can take (indices
// into shapes; both of a pair have the same number of waves), and the clock
// under load: from long_steps steps on, a launch that keeps a share u of its CUs
// busy takes 1 + load_slope * max(0, u - load_from) times its tile times.
struct TileTable {
  const TileShape* shapes;
  const int (*pairs)[2];
  int npairs;
  int64_t long_steps;
  double load_slope, load_from;
};

// Finish time of one XCD whose P CUs run t1 tiles of time d1 and then t2
// tiles of time d2, one workgroup per CU (a workgroup of these tiles holds
// a CU's four SIMDs), each started on the CU that frees first.
inline double xcd_makespan(int64_t t1, double d1, int64_t t2, double d2, int64_t P) {
  const int64_t full = t1 / P, rem = t1 % P;
  const double a = (double)full * d1, b = a + d1;  // CUs free after t1: P - rem at a, rem at b
  const int64_t na = P - rem, nb = rem;
  const double end1 = nb > 0 ? b : a;
  if (t2 == 0) return end1;
  // the j-th tile of t2 starts at the j-th smallest of {a + k d2} (na times
  // each) and {b + k d2} (nb times each)
  int64_t ka = 0, kb = 0, placed = 0;
  double last = a;
  while (placed < t2) {
    const double ta = a + (double)ka * d2, tb = nb > 0 ? b + (double)kb * d2 : 1e300;
    if (ta <= tb) {
      last = ta;
      placed += na;
      ++ka;
    } else {
      last = tb;
      placed += nb;
      ++kb;
    }
  }
  return std::max(end1, last + d2);
}

// Columns [0, n1) with the pair's first tile shape, [n1, N) with its second.
struct GemmPlan {
  int pair;  // index into the table's pairs
  int64_t n1;
  double t;  // makespan from the tile times, us
  bool small_first;  // launch the small tiles' region first
};

// Estimated time of a launch of (mostly) tiles of shape s whose busiest XCD of P
// CUs has `work` of tile time and ends after `t`.
inline double launch_time(const TileTable& tb, const TileShape& s, double t, double work, int64_t P, int64_t steps) {
  if (steps < tb.long_steps) return t;
  return t * (1.0 + tb.load_slope * s.load * std::max(0.0, work / (t * (double)P) - tb.load_from));
}

// The split with the shortest estimated time on `cus` CUs.  Workgroups go
// to the XCDs in turn, so the XCD that finishes last holds ceil(tiles / 8) of
// each region.  The split points are whole big-tile columns; n1 = N is one
// region of the big shape, n1 = 0 one of the small shape.  A later candidate
// replaces an earlier one only if it is estimated faster by what the estimate
// is good to (1%; 3% below long_steps); the first candidate is the first pair's
// big tiles alone.
inline GemmPlan choose_plan(const TileTable& tb, int64_t M, int64_t N, int64_t steps, int cus) {
  const int64_t P = std::max(1, (cus > 0 ? cus : 256) / 8);
  GemmPlan best = {0, N, 0.0, false};
  double best_t = 1e300;
  const double ahead = steps < tb.long_steps ? 0.97 : 0.99;
  for (int pr = 0; pr < tb.npairs; ++pr) {
    const TileShape& s1 = tb.shapes[tb.pairs[pr][0]];
    const TileShape& s2 = tb.shapes[tb.pairs[pr][1]];
    const double d1 = s1.time(steps), d2 = s2.time(steps);
    const int64_t rows1 = cdiv(M, s1.bm), rows2 = cdiv(M, s2.bm);
    // of more than 512 columns of tiles, as many split points (512 x 151936 x
    // 4096: 36 us of host time a call with every one, 15 with these)
    const int64_t cols = cdiv(N, s1.bn), skip = 1 + cols / 512;
    for (int64_t k = cols; k >= 0; k = k > 0 ? std::max<int64_t>(k - skip, 0) : -1) {
      // no launch with a big tile ends before that tile: on to the small ones
      // alone (a few rows into 9216 columns: 4.4 us of host time a call -> 0.2)
      if (d1 >= best_t * ahead) k = 0;
      const int64_t n1 = std::min(k * s1.bn, N);
      const int64_t t1 = rows1 * k;
      const int64_t t2 = rows2 * ((uint32_t)(N - n1 + s2.bn - 1) / (uint32_t)s2.bn);
      // no order of the tiles ends before their total time shared by the CUs
      const TileShape& lead = k > 0 ? s1 : s2;
      const double work = (double)cdiv(t1, 8) * d1 + (double)cdiv(t2, 8) * d2;
      if (launch_time(tb, lead, work / (double)P, work, P, steps) >= best_t * ahead) continue;
      const double t = xcd_makespan(cdiv(t1, 8), d1, cdiv(t2, 8), d2, P);
      const double est = launch_time(tb, lead, t, work, P, steps);
      if (est < best_t * ahead) {
        best_t = est;
        best = {pr, n1, t, false};
      }
    }
  }
  // the small tiles first when that is estimated no slower (measured on the fp8
  // product: 1-2% faster where the makespans are equal either way, as at 4352 rows
  // into 9216 and 12288 columns; 12% slower at 1543 x 9232 x 1104, whose are not)
  const TileShape& s1 = tb.shapes[tb.pairs[best.pair][0]];
  const TileShape& s2 = tb.shapes[tb.pairs[best.pair][1]];
  const int64_t t1 = cdiv(M, s1.bm) * cdiv(best.n1, s1.bn);
  const int64_t t2 = cdiv(M, s2.bm) * cdiv(N - best.n1, s2.bn);
  if (t1 > 0 && t2 > 0)
    best.small_first = xcd_makespan(cdiv(t2, 8), s2.time(steps), cdiv(t1, 8), s1.time(steps), P) <= best.t * 1.0001;
  return best;
}

// tile rows per group of the tile order: the group size that minimises the
// bytes one XCD's run of tiles reads (its distinct A row blocks + W row blocks)
inline int choose_group_m(int ntm, int ntn, int abytes, int wbytes) {
  const int64_t T = (int64_t)ntm * ntn;
  const int64_t per_xcd = std::max<int64_t>(1, (T + 7) / 8);
  int best = 1;
  double best_bytes = 1e300;
  for (int gm = 1; gm <= std::min(ntm, 16); ++gm) {
    const int64_t rows = std::min<int64_t>(gm, per_xcd);
    const int64_t cols = std::min<int64_t>(ntn, (per_xcd + gm - 1) / gm);
    const double bytes = (double)rows * abytes + (double)cols * wbytes;
    if (bytes < best_bytes) {
      best_bytes = bytes;
      best = gm;
    }
  }
  return best;
}

}  // namespace qik_tile

#endif  // QIK_TILE_H
