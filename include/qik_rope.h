/*
 * qik_rope.h -- C ABI of the per-head RMSNorm and rotation by positions on
 * several axes (time, height and width of an image or a video; text tokens at
 * the same place on each), of a layer's Q and K in one launch, and its gradient.
 *
 * Same conventions as qik_attn.h: plain C, no allocation, device pointers of
 * the current HIP device, `stream` a hipStream_t as void*, asynchronous and
 * stream-ordered launches, return QIK_OK or a negative qik_status.
 *
 * Per row x of D elements (one head of one token), in fp32:
 *   r = 1 / sqrt(mean(x^2) + eps),  n = (x * r) * w,
 *   pair i:  (y0, y1) = (n0 cos - n1 sin, n0 sin + n1 cos),
 *   angle 2 pi positions[axis[i], s] * freq[i],
 * y rounded once to the element type.  The product position * frequency and its
 * fraction are taken in fp64, so an angle is as exact far from zero as near it.
 * Without a weight n is x: the rotation alone.
 * Pair i is (x[2 i], x[2 i + 1]), or with `halves` (x[i], x[i + D / 2]).
 * The gradients, for dy of y:  dn = the rotation backwards of dy,
 *   dx = r (w dn) - x r^3 mean(x w dn),   dw = sum over the rows of dn x r,
 * dx rounded once, dw in fp32, its rows added in an order that depends on the
 * sizes alone.
 */
#ifndef QIK_ROPE_H
#define QIK_ROPE_H

#include <stdint.h>

#include "qik_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One tensor [B, S, H, D]; b, s, h strides in elements, multiples of 8, the D
 * stride 1, addresses 16-byte aligned. */
typedef struct qik_rope_tensor {
  const void* x;
  void* out;                  /* forward: y                                          */
  const float* weight;        /* [D] fp32, 16-byte aligned, or NULL: no norm         */
  const void* dy;             /* backward                                            */
  void* dx;                   /* backward                                            */
  float* dw;                  /* backward: [D] fp32, with a weight                   */
  int64_t H;                  /* 0: no such tensor, nothing of it is read            */
  int64_t stride_x[3];
  int64_t stride_out[3];      /* of out or dx                                        */
  int64_t stride_dy[3];
  float eps;
  int32_t reserved0;          /* must be 0                                           */
} qik_rope_tensor;

typedef struct qik_axial_rope_args {
  int32_t abi_version;        /* QIK_ABI_VERSION                                     */
  int32_t dtype;              /* enum qik_dtype of x, out, dy and dx                 */
  int32_t halves;             /* 0: a pair is two neighbours, 1: i and i + D / 2     */
  int32_t naxes;              /* at least 1                                          */
  const double* positions;    /* position of token s of entry b on axis a at
                                 b * stride_pos_b + a * stride_pos_a + s             */
  const double* freq;         /* [D / 2] turns per unit of position                  */
  const int32_t* axis;        /* [D / 2], 0 .. naxes - 1                             */
  int64_t stride_pos_b;       /* in elements; 0: one for all entries                 */
  int64_t stride_pos_a;
  int64_t B, S, D;            /* D in {32, 64, 128, 256}; B * S * (H of both) < 2^31 */
  qik_rope_tensor t[2];       /* Q and K, or one tensor and H = 0                    */
} qik_axial_rope_args;

int qik_axial_rope(const qik_axial_rope_args* args, void* stream);

/* The gradients.  The workspace holds the workgroups' sums of dw: at least
 * qik_axial_rope_bwd_workspace_size bytes, 16-byte aligned, contents irrelevant
 * (0 bytes where no tensor has a weight). */
int qik_axial_rope_bwd_workspace_size(const qik_axial_rope_args* args, int64_t* bytes);
int qik_axial_rope_bwd(const qik_axial_rope_args* args, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QIK_ROPE_H */
