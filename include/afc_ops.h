/*
 * afc_ops.h -- C ABI of libafc_ops.so: operators of sequence models for the learner that sits next to the environment
 * (a policy with memory and its training step), as hand-written kernels for gfx950.
 *
 *   afc_conv*   short causal convolution along the sequence, one filter per channel
 *   afc_scan*   selective state space scan
 *   afc_clip*   global 2-norm of many gradient tensors, and clipping by it
 *
 * Conventions: plain C, no torch types, DEVICE pointers everywhere except in the arrays of pointers of afc_clip_args.
 * Every call returns 0 or a negative AFC_E* (afc_env.h); afc_ops_last_error() has the calling thread's last message.
 * Work is queued on `hip_stream` of `device` (NULL: that device's default stream) and the call returns at once; it
 * allocates nothing, waits for nothing and keeps nothing, so it may be captured into a graph and called from several
 * threads.  The device that is current for the thread is the same after the call.  Outputs must not overlap inputs unless
 * a field says so.
 *
 * A sequence tensor has the element (b, l, w) at data[b*stride_batch + l*stride_length + w], one with groups has
 * (b, l, g, n) at data[b*stride_batch + l*stride_length + g*stride_group + n]: the last axis is contiguous, the others
 * are free (strides in elements, not negative).  data == NULL stands for "not given".
 * `lengths` (int32 per row, or NULL: all of `length`) are the rows' own lengths in a padded batch; a value outside
 * 0..length counts as the nearer end.  Behind a row's length nothing is read, outputs and gradients are zero, and the
 * final state is the one at the row's length.  batch == 0 and length == 0 are valid.
 * Refused (AFC_EINVAL), before anything is queued: an axis of 2^30 or more, more than 2^48 elements, work of 2^31 blocks or more.
 * A term whose operand is not given is left out.  Infinite values reach what the formulas let them reach; where they enter a sum
 * (over states, channels or positions) it is infinite or NaN.
 */
#ifndef AFC_OPS_H
#define AFC_OPS_H

#include <stdint.h>

#include "afc_env.h" /* AFC_OK, AFC_EINVAL, AFC_ENODEV, AFC_EHIP */

#ifdef __cplusplus
extern "C" {
#endif

/* element types of sequence tensors (parameters and scan states are always float) */
#define AFC_F32 0
#define AFC_BF16 1
#define AFC_F16 2

typedef struct afc_seq {
  void *data;
  int64_t stride_batch, stride_length, stride_group;
} afc_seq;

const char *afc_ops_last_error(void);

/* y[b,l,w] = f(bias[w] + sum_k weight[w,k] x[b, l - taps + 1 + k, w]),  f = silu or identity; the positions in front of
 * the row come from initial_state [batch, taps-1, width] (oldest first; NULL: zeros), final_state (the last taps-1 inputs)
 * has the same layout.  Sums in float, one rounding at the end. */
typedef struct afc_conv_args {
  int32_t device, dtype; /* dtype of x, y, the states and their gradients */
  int32_t taps;          /* 2, 3 or 4 */
  int32_t silu;
  int64_t batch, length, width;
  afc_seq x, y;
  const float *weight; /* [width, taps] */
  const float *bias;   /* [width] or NULL */
  const void *initial_state;
  void *final_state; /* NULL: not wanted.  afc_conv_step: the same memory as initial_state, updated in place */
  const int32_t *lengths;
  /* afc_conv_grad only */
  afc_seq dy;
  const void *dfinal_state; /* [batch, taps-1, width] or NULL */
  afc_seq dx;
  float *dweight, *dbias; /* NULL: not wanted */
  void *dinitial_state;   /* NULL: not wanted */
  void *workspace;        /* afc_conv_workspace() bytes, any contents, 256-byte aligned */
  uint64_t workspace_bytes;
} afc_conv_args;

int afc_conv(const afc_conv_args *args, void *hip_stream);
/* gradients of the x, weight, bias and initial_state of afc_conv with the same arguments (y, final_state are not read) */
int afc_conv_grad(const afc_conv_args *args, void *hip_stream);
int afc_conv_workspace(const afc_conv_args *args, uint64_t *bytes);
/* one token per row (length == 1, no lengths, no gradients): y from initial_state and x, the state moves on by x */
int afc_conv_step(const afc_conv_args *args, void *hip_stream);

/* delta = dt + dt_bias, or softplus of it;  h[b,l,w,:] = exp(delta a[w,:]) h[b,l-1,w,:] + delta x b[b,l,g(w),:];
 * y = <c[b,l,g(w),:], h> + d[w] x, times silu(z) where z is given;  g(w) = w / (width / groups).
 * The state is held in float.  a = -inf (taken as -3.4e38) forgets everything at every delta of
 * 1e-36 and more, and nothing at zero. */
typedef struct afc_scan_args {
  int32_t device, dtype; /* dtype of x, dt, b, c, z, y and their gradients */
  int32_t softplus;
  int32_t state; /* 1..64: size of the last axis of a, b, c and the states */
  int64_t batch, length, width, groups;
  afc_seq x, dt, b, c, z, y;
  const float *a;       /* [width, state] */
  const float *d;       /* [width] or NULL */
  const float *dt_bias; /* [width] or NULL */
  const float *initial_state; /* [batch, width, state] or NULL: zeros */
  float *final_state;   /* NULL: not wanted.  afc_scan_step: the same memory as initial_state, updated in place */
  const int32_t *lengths;
  float *checkpoints;   /* afc_scan: written for afc_scan_grad with the same arguments (afc_scan_workspace() bytes), or NULL */
  /* afc_scan_grad only; a NULL output is not wanted (dx, ddt, db and dc always are) */
  afc_seq dy;
  const float *dfinal_state;
  afc_seq dx, ddt, db, dc, dz;
  float *da, *dd, *ddt_bias, *dinitial_state;
  void *workspace; /* 256-byte aligned, any contents */
  uint64_t workspace_bytes;
} afc_scan_args;

int afc_scan(const afc_scan_args *args, void *hip_stream);
int afc_scan_grad(const afc_scan_args *args, void *hip_stream);
/* bytes of `checkpoints`, and of `workspace` for afc_scan and for afc_scan_grad (0: none needed) */
int afc_scan_workspace(const afc_scan_args *args, uint64_t *checkpoint_bytes, uint64_t *scan_bytes, uint64_t *grad_bytes);
/* one token per row (length == 1, no lengths, no gradients) */
int afc_scan_step(const afc_scan_args *args, void *hip_stream);

/* *norm = 2-norm over the elements of all `count` tensors; where max_norm >= 0 every out[i] = in[i] * min(1, max_norm /
 * (norm + 1e-6)).  out[i] may be in[i] (of the same type); otherwise no two tensors overlap.  Elements are taken in storage
 * order.  The sum of squares is accumulated in double in a fixed order: it neither overflows nor depends on timing.  A norm
 * that is not finite acts on the gradients as the formula says.  The arrays are host memory and free after the call. */
typedef struct afc_clip_args {
  int32_t device, count;
  void *const *in;
  void *const *out; /* NULL: only the norm */
  const int64_t *numel;
  const int32_t *in_dtype, *out_dtype;
  float max_norm;
  float *norm; /* device */
  void *workspace;
  uint64_t workspace_bytes;
} afc_clip_args;

int afc_clip(const afc_clip_args *args, void *hip_stream);
int afc_clip_workspace(const afc_clip_args *args, uint64_t *bytes);

#ifdef __cplusplus
}
#endif
#endif /* AFC_OPS_H */
