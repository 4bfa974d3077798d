/*
 * qik_mx_attn.h -- C ABI of the prefix slab in 4 bits and of the attention that
 * reads it:
 *
 *   qik_mx_slab_store     K and V rows -> codes and scale bytes in the slab, at
 *                         each batch entry's own place
 *   qik_mx_slab_load      the values that slab rows stand for
 *   qik_mx_attn_fwd       block-causal attention over [slab, fresh keys], query
 *                         heads in groups that share a KV head
 *
 * Same conventions as qik_attn.h: plain C, no allocation, device pointers of
 * the current HIP device, `stream` a hipStream_t as void*, asynchronous and
 * stream-ordered launches, return QIK_OK or a negative qik_status.
 *
 * A slab row is one token's K (or V) of one head: D elements in blocks of 32,
 * each block one scale byte e (E8M0: 2^(e - 127), 255 NaN) and 32 E2M1 elements,
 * two to a byte, the first in the low half, as qik_mx.h defines MXFP4.  Codes
 * and scales are apart: D / 2 and D / 32 bytes a row, with byte strides over
 * the batch, the rows and the heads.
 */
#ifndef QIK_MX_ATTN_H
#define QIK_MX_ATTN_H

#include <stdint.h>

#include "qik_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One slab of rows [B, P, H, D].  codes: 16-byte aligned, strides multiples of
 * 16; scales: address and strides multiples of D / 32; rows of codes and of
 * scales do not overlap, and 64 rows are less than 2^31 bytes apart.  Strides count where their dimension is larger than 1. */
typedef struct qik_mx_slab {
  void* codes;
  void* scales;
  int64_t stride_codes[3];    /* b, p, h in bytes                                    */
  int64_t stride_scales[3];   /* b, p, h in bytes                                    */
} qik_mx_slab;

/* Row s of batch entry b goes to slab row at[b] + s (s where `at` is NULL); rows
 * that would lie before 0 or at `capacity` and beyond are not written.  With
 * `lengths`, lengths[b] becomes min(max(at[b] + S, 0), capacity) (min(S,
 * capacity)); `lengths` may be `at` itself (the entries grow by S) and then
 * `arrivals` points to a word that is zero before the launch and after it, of
 * which concurrent launches must not share one; else the two do not overlap. */
typedef struct qik_mx_slab_store_args {
  int32_t abi_version;        /* QIK_ABI_VERSION                                     */
  int32_t dtype;              /* enum qik_dtype of k and v                           */
  const void* k;              /* [B, S, H, D], unit D stride, 16-byte aligned rows   */
  const void* v;
  qik_mx_slab k_dst, v_dst;
  const int32_t* at;          /* [B] or NULL                                         */
  int32_t* lengths;           /* [B] or NULL                                         */
  uint32_t* arrivals;         /* one word, where lengths == at != NULL               */
  int64_t B, S, H, D;         /* D in {32, 64, 128, 256}; B * S * H < 2^31           */
  int64_t capacity;           /* rows of the slab                                    */
  int64_t stride_k[3];        /* b, s, h in elements, multiples of 8                 */
  int64_t stride_v[3];
} qik_mx_slab_store_args;

int qik_mx_slab_store(const qik_mx_slab_store_args* args, void* stream);

/* k, v [B, P, H, D] contiguous, in `dtype`: the values of the slabs' first P
 * rows, zeros from lengths[b] on where `lengths` is given.  Exact in bf16; fp16
 * rounds below 2^-14 and is infinite past 65504. */
typedef struct qik_mx_slab_load_args {
  int32_t abi_version;        /* QIK_ABI_VERSION                                     */
  int32_t dtype;              /* enum qik_dtype of k and v                           */
  qik_mx_slab k_src, v_src;
  const int32_t* lengths;     /* [B] or NULL                                         */
  void* k;
  void* v;
  int64_t B, P, H, D;
} qik_mx_slab_load_args;

int qik_mx_slab_load(const qik_mx_slab_load_args* args, void* stream);

/* The attention of qik_attn_fwd_ws with a slab in 4 bits.  a: as there, except
 *   - H counts the query heads and HKV (dividing H) the heads of the keys,
 *     fresh and in the slab: query head h reads KV head h / (H / HKV);
 *   - k_cache, v_cache, their strides and v_scale are NULL / 0: `k_slab` and
 *     `v_slab` take their place, and QIK_HAS_CACHE says P > 0 as there;
 *     QIK_V_CACHE_FP8 is not set, debug_tiles is NULL;
 *   - prefix_lengths is [B, SQ] with batch stride stride_lengths_b (0: one for
 *     all entries, as there).
 * lengths (optional): batch entry b has min(max(lengths[b], 0), P) keys in the
 * slab; the rows behind them are never read.  The fresh keys keep their index
 * P + n.  A key that key_valid hides may hold anything, in the slab and among
 * the fresh ones; a value row that prefix_lengths alone hides from a row has to
 * be finite (it is multiplied by zero).  The values of slab rows are used as
 * they are: exact in bf16, rounded to fp16 as in qik_mx_slab_load.
 *
 * Few query rows (a token's, or some tokens') run a kernel of their own, which
 * cuts the keys into pieces of one length, one a workgroup; others the kernel of qik_attn_fwd_ws, with
 * the slab's tiles turned into the element type on their way into LDS.  The
 * workspace is qik_attn_fwd_ws's kind: at least qik_mx_attn_workspace_size
 * bytes, 256-byte aligned, its first QIK_ATTN_WS_CTL_BYTES zero before its first
 * use and left zero by every launch; one serves both entry points in turn on a
 * stream. */
typedef struct qik_mx_attn_args {
  qik_attn_args a;
  qik_mx_slab k_slab, v_slab;
  const int32_t* lengths;     /* [B] or NULL                                         */
  int64_t HKV;
  int64_t stride_lengths_b;
} qik_mx_attn_args;

int qik_mx_attn_validate(const qik_mx_attn_args* args);
int qik_mx_attn_workspace_size(const qik_mx_attn_args* args, int64_t* bytes);
int qik_mx_attn_fwd(const qik_mx_attn_args* args, void* workspace, int64_t workspace_bytes, void* stream);

/* Host only: which kernel a call of this shape takes on a device of `cus`
 * compute units, with lengths (`ragged`) or without.  few: 1 for the kernel of few
 * rows; row_tiles: 16-row tiles of each (b, KV head)'s rows there; pieces:
 * workgroups that share its keys, or with lengths of several entries and one tile
 * the workgroups that a KV head's entries together aim at. */
int qik_mx_attn_plan(int64_t B, int64_t SQ, int64_t SN, int64_t P, int64_t H, int64_t HKV, int64_t D,
                     int32_t ragged, int32_t cus, int32_t* few, int32_t* row_tiles, int32_t* pieces);

#ifdef __cplusplus
}
#endif

#endif /* QIK_MX_ATTN_H */
