// The block-causal attention entry points of include/qik_attn.h: the launches of
// the kernel of qik_attn_kernel.h, the causal-length builder and the host mirrors
// of the work assignment.

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include <limits.h>
#include <algorithm>
#include <atomic>

#include "qik_attn.h"
#include "qik_attn_kernel.h"
#include "qik_attn_launch.h"

namespace qik {

// ---------------------------------------------------------------------------
// Causal-length builder (processors.py:22-36), one thread per row.
constexpr int MAX_SEG_PER_LAUNCH = 64;
struct SegList {
  int n;
  int start[MAX_SEG_PER_LAUNCH];
  int end[MAX_SEG_PER_LAUNCH];
};

__global__ void build_lengths_kernel(const SegList segs, int init, int apply_prefix, int prefix_end,
                                     int seq_len, int32_t* L) {
  const int q = blockIdx.x * blockDim.x + threadIdx.x;
  if (q >= seq_len) return;
  int v = init ? q : L[q];
  for (int i = 0; i < segs.n; ++i)
    if (q >= segs.start[i] && q < segs.end[i]) v = segs.end[i] - 1;
  if (apply_prefix && q >= prefix_end) v = seq_len - 1;
  L[q] = v;
}

// ---------------------------------------------------------------------------
// The workspace of qik_attn_fwd_noalloc: one array per device, never
// allocated by the library.  Host code uses its device address from
// hipGetSymbolAddress (scratch_ptr below), never the name.
static __device__ __align__(256) unsigned char scratch[QIK_ATTN_SCRATCH_BYTES];

// Zero `n16` 16-byte words (the scratch's control words) with vector stores;
// a fill kernel rather than hipMemsetAsync, so that a captured graph replays it.
__global__ void zero16_kernel(u32x4* p, int n16) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n16) p[i] = u32x4{0u, 0u, 0u, 0u};
}

// ---------------------------------------------------------------------------
// host side

typedef void (*kernel_fn)(Params);

template <int D, bool KV, int KS, bool MANY>
kernel_fn pick_kernel(bool fp16, bool vfp8) {
  if (fp16) return attn_fwd_kernel<D, true, SlabKV::ELEM, KV, KS, MANY>;
  if (vfp8) return attn_fwd_kernel<D, false, SlabKV::V_FP8, KV, KS, MANY>;
  return attn_fwd_kernel<D, false, SlabKV::ELEM, KV, KS, MANY>;
}

// key_valid is a template parameter: without a mask the kernel carries none
// of its code (the tile loop is then the same as with no mask support at all)
template <int D, bool KV>
void pick_kernels(bool fp16, bool vfp8, Kernels* k) {
  k->one = reinterpret_cast<const void*>(pick_kernel<D, KV, 1, false>(fp16, vfp8));
  if constexpr (D <= 128) {
    k->pieces = reinterpret_cast<const void*>(pick_kernel<D, KV, 1, true>(fp16, vfp8));
    k->groups = reinterpret_cast<const void*>(pick_kernel<D, KV, 2, false>(fp16, vfp8));
  }
}

template <int D>
void pick_kernels(bool fp16, bool vfp8, bool kv, Kernels* k) {
  if (kv) pick_kernels<D, true>(fp16, vfp8, k);
  else pick_kernels<D, false>(fp16, vfp8, k);
}

std::atomic<int> g_slots[24][MAX_DEVICES];

Kernels kernels_of(const qik_attn_args* a) {
  const bool fp16 = a->dtype == QIK_DTYPE_FP16;
  const bool vfp8 = (a->flags & QIK_V_CACHE_FP8) != 0;
  const bool kv = (a->flags & QIK_HAS_KEY_VALID) != 0;
  Kernels k = {nullptr, nullptr, nullptr, nullptr};
  switch (a->D) {
    case 32: pick_kernels<32>(fp16, vfp8, kv, &k); break;
    case 64: pick_kernels<64>(fp16, vfp8, kv, &k); break;
    case 128: pick_kernels<128>(fp16, vfp8, kv, &k); break;
    default: pick_kernels<256>(fp16, vfp8, kv, &k); break;
  }
  const int di = a->D == 32 ? 0 : a->D == 64 ? 1 : a->D == 128 ? 2 : 3;
  k.slots = g_slots[2 * (3 * di + (fp16 ? 1 : (vfp8 ? 2 : 0))) + (kv ? 1 : 0)];
  return k;
}

int schedule_one(int64_t Lmax, int64_t P, int64_t SN, bool has_cache) {
  int64_t run0 = 0, run1 = 0;
  const int64_t s1 = has_cache ? P : 0;
  if (has_cache && Lmax >= 0) run0 = std::min(cdiv64(P, BN), Lmax / BN + 1);
  if (Lmax >= s1) run1 = std::min(cdiv64(SN, BN), (Lmax - s1) / BN + 1);
  return (int)(run0 + run1);
}

int plan_launch(const qik_attn_args* a, bool split, Launch* L) {
  return plan_launch(a->B * a->H, a->SQ, a->D, (a->flags & QIK_UNIFORM_L) != 0, kernels_of(a), split, L);
}

// Device address of `scratch` on the current device, resolved once per device.
std::atomic<void*> g_scratch[MAX_DEVICES];

int scratch_ptr(void** out) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEVICES) return QIK_ERR_DEVICE;
  void* p = g_scratch[dev].load(std::memory_order_acquire);
  if (p == nullptr) {
    if (hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)) != hipSuccess || p == nullptr) return QIK_ERR_DEVICE;
    g_scratch[dev].store(p, std::memory_order_release);
  }
  *out = p;
  return QIK_OK;
}

int launch(const qik_attn_args* a, bool split, void* ws, int64_t ws_bytes, void* stream) {
  const int st = qik_attn_validate(a);
  if (st != QIK_OK) return st;
  Launch L;
  const int pst = plan_launch(a, split, &L);
  if (pst != QIK_OK) return pst;
  if (L.grid == 0) return QIK_OK;
  if (L.ws_bytes > 0 && (ws == nullptr || !aligned_to(ws, 256) || ws_bytes < L.ws_bytes)) return QIK_ERR_WORKSPACE;

  Params p;
  memset(&p, 0, sizeof(p));
  p.q = static_cast<const char*>(a->q);
  p.k_new = static_cast<const char*>(a->k_new);
  p.v_new = static_cast<const char*>(a->v_new);
  p.k_cache = static_cast<const char*>(a->k_cache);
  p.v_cache = static_cast<const char*>(a->v_cache);
  p.v_scale = a->v_scale;
  p.L = a->prefix_lengths;
  p.key_valid = a->key_valid;
  p.out = static_cast<char*>(a->out);
  p.debug_tiles = a->debug_tiles;
  if (L.ws_bytes > 0) {
    p.ctl = static_cast<unsigned*>(ws);
    p.ws_slots = static_cast<char*>(ws) + L.ctl_bytes;
  }
  for (int i = 0; i < 3; ++i) {
    p.sq[i] = a->stride_q[i];
    p.skn[i] = a->stride_k_new[i];
    p.svn[i] = a->stride_v_new[i];
    p.skc[i] = a->stride_k_cache[i];
    p.svc[i] = a->stride_v_cache[i];
    p.so[i] = a->stride_out[i];
  }
  p.svalid_b = a->stride_valid_b;
  p.SQ = (int)a->SQ;
  p.SN = (int)a->SN;
  p.P = (int)a->P;
  p.H = (int)a->H;
  p.KV = (int)(a->P + a->SN);
  p.has_cache = (a->flags & QIK_HAS_CACHE) ? 1 : 0;
  p.has_key_valid = (a->flags & QIK_HAS_KEY_VALID) ? 1 : 0;
  p.uniform = (a->flags & QIK_UNIFORM_L) ? 1 : 0;
  // qk_scale = sm_scale * log2(e), both fp32, as triton_attention.py:93 computes it
  p.qk_scale = a->sm_scale * 1.44269504088896340736f;
  p.plan = L.plan;

  void* kargs[] = {&p};
  const hipError_t e = hipLaunchKernel(L.fn, dim3((unsigned)L.grid),
                                       dim3((unsigned)L.threads), kargs, 0, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? QIK_OK : QIK_ERR_LAUNCH;
}

}  // namespace qik

extern "C" {

int qik_abi_version(void) { return QIK_ABI_VERSION; }

const char* qik_strerror(int status) {
  switch (status) {
    case QIK_OK: return "ok";
    case QIK_ERR_NULL_ARG: return "a required pointer is NULL";
    case QIK_ERR_ABI_VERSION: return "qik_attn_args.abi_version does not match the library";
    case QIK_ERR_DTYPE: return "fp16/bf16 only";
    case QIK_ERR_HEAD_DIM: return "head_dim must be 32, 64, 128 or 256";
    case QIK_ERR_SHAPE: return "negative or oversized B/SQ/SN/P/H";
    case QIK_ERR_CACHE: return "cache flag, P and cache pointers are inconsistent";
    case QIK_ERR_FP8_SCALE: return "fp8 cache V needs the cache, a v_scale pointer and bf16 q/k/v";
    case QIK_ERR_ALIGN: return "pointers and b/s/h strides must be multiples of 8 elements, and K/V row strides at least D";
    case QIK_ERR_LAUNCH: return "HIP kernel launch failed";
    case QIK_ERR_SEGMENTS: return "segments need 0 <= start <= end, and 0 <= prefix_end <= seq_len";
    case QIK_ERR_DEVICE: return "HIP device query failed";
    case QIK_ERR_WORKSPACE: return "workspace NULL, not 256-byte aligned, or smaller than qik_attn_workspace_size";
    case QIK_ERR_SCRATCH: return "the call needs more workspace than QIK_ATTN_SCRATCH_BYTES";
    default: return "unknown qik status";
  }
}

int qik_attn_block_shape(int32_t* block_m, int32_t* block_n) {
  if (block_m == nullptr || block_n == nullptr) return QIK_ERR_NULL_ARG;
  *block_m = qik::BM;
  *block_n = qik::BN;
  return QIK_OK;
}

int qik_attn_validate(const qik_attn_args* a) {
  if (a == nullptr) return QIK_ERR_NULL_ARG;
  if (a->abi_version != QIK_ABI_VERSION || a->reserved0 != 0 || a->reserved1 != 0) return QIK_ERR_ABI_VERSION;
  if (a->dtype != QIK_DTYPE_BF16 && a->dtype != QIK_DTYPE_FP16) return QIK_ERR_DTYPE;
  if (a->D != 32 && a->D != 64 && a->D != 128 && a->D != 256) return QIK_ERR_HEAD_DIM;
  const int64_t lim = (int64_t)INT_MAX;
  if (a->B < 0 || a->SQ < 0 || a->SN < 0 || a->P < 0 || a->H < 0) return QIK_ERR_SHAPE;
  if (a->SQ > lim || a->SN > lim || a->P > lim || a->H > lim || a->P + a->SN > lim) return QIK_ERR_SHAPE;
  const int64_t nmb = qik::cdiv64(a->SQ, qik::BM);
  if (a->B > 0 && a->H > 0 && nmb > 0 && a->B * a->H > lim / nmb) return QIK_ERR_SHAPE;
  if ((a->flags & ~(QIK_HAS_CACHE | QIK_HAS_KEY_VALID | QIK_UNIFORM_L | QIK_V_CACHE_FP8)) != 0)
    return QIK_ERR_SHAPE;

  const bool has_cache = (a->flags & QIK_HAS_CACHE) != 0;
  const bool vfp8 = (a->flags & QIK_V_CACHE_FP8) != 0;
  const bool has_kv = (a->flags & QIK_HAS_KEY_VALID) != 0;
  const bool uniform = (a->flags & QIK_UNIFORM_L) != 0;
  if (has_cache != (a->P > 0)) return QIK_ERR_CACHE;
  if (has_cache && (a->k_cache == nullptr || a->v_cache == nullptr)) return QIK_ERR_CACHE;
  if (vfp8 && (!has_cache || a->v_scale == nullptr || a->dtype != QIK_DTYPE_BF16)) return QIK_ERR_FP8_SCALE;
  if (!vfp8 && a->v_scale != nullptr) return QIK_ERR_FP8_SCALE;
  if (has_kv != (a->key_valid != nullptr)) return QIK_ERR_NULL_ARG;

  const bool work = a->B > 0 && a->H > 0 && a->SQ > 0;
  if (!work) return QIK_OK;
  if (a->q == nullptr || a->out == nullptr) return QIK_ERR_NULL_ARG;
  if (a->SN > 0 && (a->k_new == nullptr || a->v_new == nullptr)) return QIK_ERR_NULL_ARG;
  if (!uniform && a->prefix_lengths == nullptr) return QIK_ERR_NULL_ARG;

  // 16-byte chunks of 8 elements: bases 16-B aligned, strides multiples of 8 elements
  if (!qik::aligned_to(a->q, 16) || !qik::aligned_to(a->out, 16)) return QIK_ERR_ALIGN;
  if (!qik::stride_ok(a->stride_q, a->B, a->SQ, a->H, 8)) return QIK_ERR_ALIGN;
  if (!qik::stride_ok(a->stride_out, a->B, a->SQ, a->H, 8)) return QIK_ERR_ALIGN;
  if (a->SN > 0) {
    if (!qik::aligned_to(a->k_new, 16) || !qik::aligned_to(a->v_new, 16)) return QIK_ERR_ALIGN;
    if (!qik::stride_ok(a->stride_k_new, a->B, a->SN, a->H, 8)) return QIK_ERR_ALIGN;
    if (!qik::stride_ok(a->stride_v_new, a->B, a->SN, a->H, 8)) return QIK_ERR_ALIGN;
  }
  // a KV tile's byte offsets must fit in 31 bits (the tile copies use 32-bit
  // buffer offsets): BN * row stride < 2^31
  const int64_t tile_lim = ((int64_t)1 << 31) / qik::BN;
  if (a->stride_k_new[1] * 2 >= tile_lim || a->stride_v_new[1] * 2 >= tile_lim) return QIK_ERR_SHAPE;
  if (has_cache && (a->stride_k_cache[1] * 2 >= tile_lim || a->stride_v_cache[1] * 2 >= tile_lim)) return QIK_ERR_SHAPE;
  // K/V rows must not overlap (the tile copies zero-fill a segment tail through
  // buffer bounds that assume row_stride >= D)
  if (a->SN > 1 && (a->stride_k_new[1] < a->D || a->stride_v_new[1] < a->D)) return QIK_ERR_ALIGN;
  if (has_cache && a->P > 1 && (a->stride_k_cache[1] < a->D || a->stride_v_cache[1] < a->D)) return QIK_ERR_ALIGN;
  if (has_cache) {
    if (!qik::aligned_to(a->k_cache, 16)) return QIK_ERR_ALIGN;
    if (!qik::aligned_to(a->v_cache, vfp8 ? 8 : 16)) return QIK_ERR_ALIGN;
    if (!qik::stride_ok(a->stride_k_cache, a->B, a->P, a->H, 8)) return QIK_ERR_ALIGN;
    if (!qik::stride_ok(a->stride_v_cache, a->B, a->P, a->H, 8)) return QIK_ERR_ALIGN;
  }
  return QIK_OK;
}

int qik_attn_fwd(const qik_attn_args* a, void* stream) { return qik::launch(a, false, nullptr, 0, stream); }

int qik_attn_workspace_size(const qik_attn_args* a, int64_t* bytes) {
  if (bytes == nullptr) return QIK_ERR_NULL_ARG;
  *bytes = 0;
  const int st = qik_attn_validate(a);
  if (st != QIK_OK) return st;
  qik::Launch L;
  const int pst = qik::plan_launch(a, true, &L);
  if (pst != QIK_OK) return pst;
  *bytes = L.ws_bytes;
  return QIK_OK;
}

int qik_attn_fwd_ws(const qik_attn_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  return qik::launch(a, true, workspace, workspace_bytes, stream);
}

int qik_attn_fwd_noalloc(const qik_attn_args* a, void* stream) {
  const int st = qik_attn_validate(a);
  if (st != QIK_OK) return st;
  qik::Launch L;
  const int pst = qik::plan_launch(a, true, &L);
  if (pst != QIK_OK) return pst;
  if (L.grid == 0) return QIK_OK;
  if (L.ws_bytes > (int64_t)QIK_ATTN_SCRATCH_BYTES) return QIK_ERR_SCRATCH;
  void* ws = nullptr;
  if (L.ws_bytes > 0) {
    const int sst = qik::scratch_ptr(&ws);
    if (sst != QIK_OK) return sst;
    // the control words must be zero when the attention launch starts
    const int n16 = (int)(L.ctl_bytes / 16);
    void* kargs[] = {&ws, (void*)&n16};
    if (hipLaunchKernel(reinterpret_cast<const void*>(qik::zero16_kernel), dim3((unsigned)((n16 + 255) / 256)),
                        dim3(256), kargs, 0, static_cast<hipStream_t>(stream)) != hipSuccess)
      return QIK_ERR_LAUNCH;
  }
  return qik::launch(a, true, ws, (int64_t)QIK_ATTN_SCRATCH_BYTES, stream);
}

int qik_attn_work_map(int64_t n_items, int32_t n_row_blocks, int32_t slots_per_xcd, int32_t split,
                      int32_t* item, int32_t* piece, int32_t* group, int64_t cap, int64_t* grid,
                      int64_t* ngroups, int32_t* pieces) {
  return qik_attn_work_map_xcds(n_items, n_row_blocks, slots_per_xcd, split, qik::NXCD, item, piece, group, cap,
                                grid, ngroups, pieces);
}

int qik_attn_work_map_xcds(int64_t n_items, int32_t n_row_blocks, int32_t slots_per_xcd, int32_t split,
                           int32_t n_xcds, int32_t* item, int32_t* piece, int32_t* group, int64_t cap,
                           int64_t* grid, int64_t* ngroups, int32_t* pieces) {
  if (grid == nullptr || ngroups == nullptr) return QIK_ERR_NULL_ARG;
  if (n_items < 0 || n_items > INT_MAX || n_row_blocks < 1 || slots_per_xcd < 1) return QIK_ERR_SHAPE;
  if (n_xcds < 1 || n_xcds > qik::NXCD_MAX) return QIK_ERR_SHAPE;
  const qik::WorkPlan pl = qik::make_plan((int)n_items, n_row_blocks, slots_per_xcd, split ? 1 : 0, 1, n_xcds);
  if ((int64_t)pl.nx * pl.wpx > INT_MAX) return QIK_ERR_SHAPE;
  *grid = (int64_t)pl.nx * pl.wpx;
  *ngroups = pl.ngroups;
  if (pieces != nullptr) *pieces = pl.ns;
  if (item == nullptr && piece == nullptr && group == nullptr) return QIK_OK;
  if (item == nullptr || piece == nullptr || group == nullptr) return QIK_ERR_NULL_ARG;
  if (cap < *grid) return QIK_ERR_SHAPE;
  for (int64_t b = 0; b < *grid; ++b) {
    const qik::Work w = qik::plan_work(pl, (int)b);
    item[b] = w.item;
    piece[b] = w.piece;
    group[b] = w.group;
  }
  return QIK_OK;
}

int qik_attn_tile_schedule(int64_t SQ, int64_t P, int64_t SN, int32_t flags, const int32_t* L, int32_t* out) {
  if (out == nullptr) return QIK_ERR_NULL_ARG;
  if (SQ < 0 || P < 0 || SN < 0) return QIK_ERR_SHAPE;
  const bool has_cache = (flags & QIK_HAS_CACHE) != 0;
  const bool uniform = (flags & QIK_UNIFORM_L) != 0;
  if (has_cache != (P > 0)) return QIK_ERR_CACHE;
  if (!uniform && SQ > 0 && L == nullptr) return QIK_ERR_NULL_ARG;
  const int64_t nmb = qik::cdiv64(SQ, qik::BM);
  for (int64_t mb = 0; mb < nmb; ++mb) {
    int64_t Lmax;
    if (uniform) {
      Lmax = P + SN - 1;
    } else {
      Lmax = -1;
      const int64_t r1 = std::min(SQ, (mb + 1) * qik::BM);
      for (int64_t r = mb * qik::BM; r < r1; ++r) Lmax = std::max<int64_t>(Lmax, L[r]);
    }
    out[mb] = qik::schedule_one(Lmax, P, SN, has_cache);
  }
  return QIK_OK;
}

int qik_build_prefix_lengths(const int32_t* segments, int32_t nseg, int64_t prefix_end, int64_t seq_len,
                             int32_t* L, void* stream) {
  if (nseg < 0 || seq_len < 0 || seq_len > INT_MAX) return QIK_ERR_SEGMENTS;
  if (prefix_end < 0 || prefix_end > seq_len) return QIK_ERR_SEGMENTS;
  if (nseg > 0 && segments == nullptr) return QIK_ERR_NULL_ARG;
  for (int i = 0; i < nseg; ++i) {
    const int32_t s = segments[3 * i], e = segments[3 * i + 1];
    if (s < 0 || e < s) return QIK_ERR_SEGMENTS;
  }
  if (seq_len == 0) return QIK_OK;
  if (L == nullptr) return QIK_ERR_NULL_ARG;
  const int threads = 256;
  const unsigned blocks = (unsigned)((seq_len + threads - 1) / threads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  // non-text segments in order, MAX_SEG_PER_LAUNCH per launch; later launches see earlier writes
  int i = 0;
  bool first = true;
  do {
    qik::SegList segs;
    memset(&segs, 0, sizeof(segs));
    while (i < nseg && segs.n < qik::MAX_SEG_PER_LAUNCH) {
      if (segments[3 * i + 2] == 0) {
        segs.start[segs.n] = segments[3 * i];
        segs.end[segs.n] = segments[3 * i + 1];
        ++segs.n;
      }
      ++i;
    }
    int last = (i >= nseg) ? 1 : 0;
    int init = first ? 1 : 0, pe = (int)prefix_end, sl = (int)seq_len;
    void* kargs[] = {&segs, &init, &last, &pe, &sl, &L};
    if (hipLaunchKernel(reinterpret_cast<const void*>(qik::build_lengths_kernel), dim3(blocks), dim3(threads),
                        kargs, 0, s) != hipSuccess)
      return QIK_ERR_LAUNCH;
    first = false;
  } while (i < nseg);
  return QIK_OK;
}

}  // extern "C"
