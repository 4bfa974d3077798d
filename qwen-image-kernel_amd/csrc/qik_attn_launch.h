// Launch geometry of the attention kernel (qik_attn_kernel.h), shared by the
// entry points that launch it: which form runs, the work plan, the workspace.
#ifndef QIK_ATTN_LAUNCH_H
#define QIK_ATTN_LAUNCH_H

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include <limits.h>
#include <algorithm>
#include <atomic>

#include "qik_attn.h"
#include "qik_attn_kernel.h"
#include "qik_plan.h"

namespace qik {

// How a launch runs its row blocks: one unit per workgroup or a queue of units
// (ONE), the queue with items of more than two pieces (PIECES), or a two-group
// workgroup per row block (GROUPS).  At D = 256 ONE only: two groups' LDS
// stages are more than a CU holds, and its registers leave no room to merge
// many pieces.
enum class Form { ONE, PIECES, GROUPS };

inline bool two_group_dim(int64_t D) { return D <= 128; }
inline int max_pieces_dim(int64_t D) { return D <= 128 ? MAX_PIECES : 2; }

inline int slot_bytes_d(int64_t D) {
  switch (D) {
    case 32: return slot_bytes<32>();
    case 64: return slot_bytes<64>();
    case 128: return slot_bytes<128>();
    default: return slot_bytes<256>();
  }
}

inline bool aligned_to(const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) % a) == 0; }

// A stride only matters along a dim of size > 1.
inline bool stride_ok(const int64_t st[3], int64_t nb, int64_t ns, int64_t nh, int64_t mult) {
  if (nb > 1 && st[0] % mult != 0) return false;
  if (ns > 1 && st[1] % mult != 0) return false;
  if (nh > 1 && st[2] % mult != 0) return false;
  return true;
}

inline int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int MAX_DEVICES = 64;
inline std::atomic<int> g_xcds[MAX_DEVICES];
inline std::atomic<int> g_cus[MAX_DEVICES];

// Compute units of the current device, cached per device (0 if unknown).
inline int device_cus() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  if (dev >= 0 && dev < MAX_DEVICES) {
    const int c = g_cus[dev].load(std::memory_order_relaxed);
    if (c > 0) return c;
  }
  int cus = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 0;
  if (dev >= 0 && dev < MAX_DEVICES) g_cus[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// XCDs of the current device (hipDeviceAttributeNumberOfXccs; NXCD if the
// runtime cannot say), clamped to [1, NXCD_MAX], cached per device.
inline int device_xcds() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return NXCD;
  if (dev >= 0 && dev < MAX_DEVICES) {
    const int c = g_xcds[dev].load(std::memory_order_relaxed);
    if (c > 0) return c;
  }
  int nx = 0;
  if (hipDeviceGetAttribute(&nx, hipDeviceAttributeNumberOfXccs, dev) != hipSuccess || nx <= 0) nx = NXCD;
  nx = std::min(std::max(nx, 1), NXCD_MAX);
  if (dev >= 0 && dev < MAX_DEVICES) g_xcds[dev].store(nx, std::memory_order_relaxed);
  return nx;
}

// The three forms of one call's kernel (pieces and groups NULL at D = 256), and
// where the workgroups an XCD holds at once of `one` are kept per device (0:
// not known yet).
struct Kernels {
  const void* one;
  const void* pieces;
  const void* groups;
  std::atomic<int>* slots;  // [MAX_DEVICES]
};

// Workgroups one XCD of the current device holds at once for kernel k.one:
// occupancy per CU x CUs / XCDs, cached per device.
inline int slots_per_xcd(const Kernels& k, int* out) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return QIK_ERR_DEVICE;
  if (dev >= 0 && dev < MAX_DEVICES) {
    const int c = k.slots[dev].load(std::memory_order_relaxed);
    if (c > 0) {
      *out = c;
      return QIK_OK;
    }
  }
  int cus = 0, occ = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    return QIK_ERR_DEVICE;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&occ, k.one, NTHREADS, 0) != hipSuccess || occ <= 0)
    return QIK_ERR_DEVICE;
  const int sx = std::max(1, occ * cus / device_xcds());
  if (dev >= 0 && dev < MAX_DEVICES) k.slots[dev].store(sx, std::memory_order_relaxed);
  *out = sx;
  return QIK_OK;
}

// Launch geometry of one call.  Without `split`: one workgroup per unit, no
// workspace.  With it: the last partial round's row blocks split into pieces
// (qik_plan.h), sx workgroups per XCD pulling units from the XCD's queue, and
// a workspace of control words (zero between launches) and partial-state
// slots.
struct Launch {
  const void* fn;
  WorkPlan plan;
  int64_t grid;
  int threads;         // per workgroup: NTHREADS, or 2 * NTHREADS for the two-group kernel
  int64_t ws_bytes;    // 0: no workspace
  int64_t ctl_bytes;   // control words at the start of the workspace
  int slot;
};

// heads: B * H of the keys' heads; rows: query rows of each; heads * cdiv(rows,
// BM) <= INT_MAX (the callers validate it)
inline int plan_launch(int64_t heads, int64_t rows, int64_t D, bool uniform, const Kernels& k, bool split, Launch* L) {
  const int64_t nmb = cdiv64(rows, BM);
  const int64_t n = heads * nmb;
  L->fn = k.one;
  L->slot = slot_bytes_d(D);
  L->ws_bytes = 0;
  L->ctl_bytes = 0;
  L->grid = 0;
  L->threads = NTHREADS;
  memset(&L->plan, 0, sizeof(L->plan));
  if (n == 0) return QIK_OK;
  const int nx = device_xcds();
  int sx = 1;
  const int cus = device_cus();
  if (split && two_group_dim(D) && n <= cus) {
    // row blocks fit the CUs once: one two-group workgroup per row block, its
    // KV tiles split between the groups and merged in LDS (no workspace) ...
    L->fn = k.groups;
    L->threads = 2 * NTHREADS;
    if (2 * n <= cus && cus >= nx) {
      // ... or, with at most half the CUs' worth of row blocks (one GPU's share
      // of the heads), each row block split into two equal pieces on two CUs,
      // every piece split between the groups, the pieces merged through the
      // workspace as the split launch below merges them
      L->plan = make_plan((int)n, (int)nmb, cus / nx, 1, uniform ? 0 : 1, nx, 2);
      if (L->plan.ns == 2 && L->plan.wpx <= cus / nx && 2 * NXCD_MAX + L->plan.ngroups <= QIK_ATTN_WS_CTL_BYTES / 4) {
        L->grid = (int64_t)nx * L->plan.wpx;
        L->ctl_bytes = QIK_ATTN_WS_CTL_BYTES;
        L->ws_bytes = L->ctl_bytes + (int64_t)L->plan.ngroups * L->plan.ns * L->slot;
        return QIK_OK;
      }
    }
    L->plan = make_plan((int)n, (int)nmb, 1, 0, 1, nx);
    L->grid = (int64_t)nx * L->plan.wpx;
    return QIK_OK;
  }
  if (split) {
    const int st = slots_per_xcd(k, &sx);
    if (st != QIK_OK) return st;
    L->plan = make_plan((int)n, (int)nmb, sx, 1, uniform ? 0 : 1, nx, max_pieces_dim(D));
    // queue positions are mapped through loc * nx + x, which must fit an
    // int, and the arrival words must fit the fixed control region (the same
    // for every shape, so that no launch leaves slot data where another
    // launch keeps its control words)
    if ((int64_t)nx * L->plan.wpx <= INT_MAX && 2 * NXCD_MAX + L->plan.ngroups <= QIK_ATTN_WS_CTL_BYTES / 4) {
      if (L->plan.ns > 2) L->fn = k.pieces;
      L->grid = (int64_t)nx * std::min(sx, L->plan.wpx);
      L->ctl_bytes = QIK_ATTN_WS_CTL_BYTES;
      L->ws_bytes = L->ctl_bytes + (int64_t)L->plan.ngroups * L->plan.ns * L->slot;
      return QIK_OK;
    }
  }
  L->plan = make_plan((int)n, (int)nmb, sx, 0, 1, nx);
  L->grid = (int64_t)nx * L->plan.wpx;
  return QIK_OK;
}

}  // namespace qik

#endif  // QIK_ATTN_LAUNCH_H
