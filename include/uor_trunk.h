/*
 * uor_trunk.h - C ABI of a float trunk's operators on MI355X (gfx950).
 *
 * Beside the served integer step of uor_fbs.h: parts of the layers of recurrent trunks that are trained,
 * and answer, in floating point. They are neighbours of the served layers and not their float form (the
 * served recurrence turns quaternions, its gate is a product of them, it has no norm after a block, and
 * its windows may be longer), and nothing here exports to the served container:
 *
 *   scan    the selective state space scan, one decay a head and position:
 *             D_t = softplus(dt_t + dt_bias),  h_t = exp(D_t A) h_(t-1) + D_t x_t (x) B_t,
 *             y_t = h_t C_t + D x_t
 *           with x_t of `dim` values a head, h of dim x state values a head, and B, C of `state`
 *           values shared by the heads / groups heads of a group;
 *   conv    the short causal convolution of each channel over its last `taps` rows;
 *   norms   the norms before and after a block fused with its gate and residual scale:
 *             v = out silu(gate),  r' = residual + scale v rsqrt(mean v^2 + eps) post,
 *             n = r' rsqrt(mean r'^2 + eps) pre.
 *
 * Rows are packed: sequence s owns rows offsets[s] .. offsets[s + 1] - 1 (int32 on the device,
 * ascending; values outside 0 .. tokens are taken as the nearest inside). Of offsets that do not ascend
 * the results are not defined, but no call reads or writes past its arrays. A sequence may have no
 * rows. Rows before offsets[0] and from offsets[seqs] on are no sequence's: y, dx, ddt, dB and dC are
 * zeros there, and no other output depends on them. Rows of x, dt, B, C and y lie `*_stride` values
 * apart (of one row the stride is not looked at) and are dense inside.
 *
 * Types: activations (x, dt, B, C, y, out, gate, residual and their gradients, the convolution's
 * state) are all bf16 or all f32; parameters (A, D, dt_bias, weight, bias, post, scale, pre), the
 * scan's states and the parameters' gradients are f32.
 *
 * What is infinite or no number reaches the results that depend on it by these formulas and their
 * gradients, as an infinity or NaN, and no others.
 *
 * Every call takes device pointers, runs on `stream` (a hipStream_t) of `device` and allocates
 * nothing: where a call needs scratch memory, the caller passes at least *_workspace_bytes of it,
 * aligned to 16 bytes. Results do not depend on the order in which blocks run. The calls can be
 * captured into a graph.
 *
 * Return codes: 0 success, -1 invalid argument, -2 device error (uor_trunk_last_error()).
 */
#ifndef UOR_TRUNK_H
#define UOR_TRUNK_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define UOR_TRUNK_ABI_VERSION 1u
#define UOR_TRUNK_MAX_DIM 128u
#define UOR_TRUNK_MAX_STATE 128u
#define UOR_TRUNK_MAX_TAPS 4u
#define UOR_TRUNK_MAX_WIDTH 8192u

#define UOR_TRUNK_BF16 0u
#define UOR_TRUNK_F32 1u

uint32_t uor_trunk_abi_version(void);
const char *uor_trunk_last_error(void);
uint64_t uor_trunk_sizeof_scan(void);
uint64_t uor_trunk_sizeof_conv(void);
uint64_t uor_trunk_sizeof_norms(void);

typedef struct {
  int32_t device;
  uint32_t dtype;
  uint32_t tokens, seqs;                /* rows and sequences; a step has one row a sequence */
  uint32_t heads, groups, dim, state;   /* heads a multiple of groups */
  uint32_t slots;                       /* a step's: how many states there are */
  uint32_t reserved;
  int64_t x_stride, dt_stride, b_stride, c_stride, y_stride; /* values between rows; y_stride is dy's in a gradient */
  const void *x, *dt, *B, *C;           /* [tokens][heads][dim], [tokens][heads], [tokens][groups][state] x 2 */
  const float *A, *D, *dt_bias;         /* [heads]; D and dt_bias may be NULL */
  const int32_t *offsets;               /* [seqs + 1]; NULL: one sequence of all rows */
  const float *initial;                 /* [seqs][heads][dim][state] or NULL for zeros */
  void *y;                              /* [tokens][heads][dim] */
  float *final;                         /* [seqs][heads][dim][state] or NULL */
  const int32_t *index;                 /* a step's: each row's state (outside 0 .. slots - 1: the row is
                                           skipped and its y is 0); NULL: row i's is i. No two rows alike. */
  float *states;                        /* a step's: [slots][heads][dim][state], updated in place */
  /* a gradient's: */
  const void *dy;                       /* [tokens][heads][dim] */
  const float *dfinal;                  /* like final, or NULL for zeros */
  void *dx, *ddt, *dB, *dC;             /* dense rows */
  float *dA, *dD, *ddt_bias, *dinitial; /* dD, ddt_bias and dinitial may be NULL */
} uor_trunk_scan_args;

uint64_t uor_trunk_scan_workspace_bytes(const uor_trunk_scan_args *args);
int uor_trunk_scan_async(const uor_trunk_scan_args *args, void *workspace, uint64_t bytes, void *stream);
uint64_t uor_trunk_scan_backward_workspace_bytes(const uor_trunk_scan_args *args);
int uor_trunk_scan_backward_async(const uor_trunk_scan_args *args, void *workspace, uint64_t bytes, void *stream);
int uor_trunk_scan_step_async(const uor_trunk_scan_args *args, void *stream);

typedef struct {
  int32_t device;
  uint32_t dtype;
  uint32_t tokens, seqs, channels, taps;
  uint32_t slots, silu;                 /* silu: 1 for y = silu(..), 0 for y = .. */
  int64_t x_stride, y_stride;           /* y_stride is dy's in a gradient */
  const void *x;                        /* [tokens][channels] */
  const float *weight, *bias;           /* [channels][taps] (the last tap is the row's own); [channels] or NULL */
  const int32_t *offsets;
  const void *initial;                  /* [seqs][taps - 1][channels]: the rows before, or NULL for zeros */
  void *y, *final;                      /* final: like initial, the last rows, or NULL */
  const int32_t *index;                 /* a step's, as the scan's */
  void *states;                         /* a step's: [slots][taps - 1][channels], updated in place */
  /* a gradient's: */
  const void *dy, *dfinal;              /* dfinal like final, or NULL for zeros */
  void *dx, *dinitial;                  /* dinitial may be NULL */
  float *dweight, *dbias;               /* dbias may be NULL */
} uor_trunk_conv_args;

int uor_trunk_conv_async(const uor_trunk_conv_args *args, void *stream);
uint64_t uor_trunk_conv_backward_workspace_bytes(const uor_trunk_conv_args *args);
int uor_trunk_conv_backward_async(const uor_trunk_conv_args *args, void *workspace, uint64_t bytes, void *stream);
int uor_trunk_conv_step_async(const uor_trunk_conv_args *args, void *stream);

/* `out` NULL: no block, r' = residual. `residual` NULL: r' = scale v rsqrt(..) post. `pre` NULL: no
 * norm before the next block. gate, post and scale may be NULL (1). n is of the unrounded r'. In a
 * gradient `residual` and `residual_out` are the call's own: with a block r' is computed again. */
typedef struct {
  int32_t device;
  uint32_t dtype;
  uint32_t rows, width;
  float eps;
  uint32_t reserved;
  int64_t residual_stride, out_stride, gate_stride;
  const void *residual, *out, *gate;    /* [rows][width] */
  const float *post, *scale, *pre;      /* [width] */
  void *residual_out, *normed;          /* [rows][width], dense; residual_out needs `out` */
  /* a gradient's: */
  const void *dresidual_out, *dnormed;  /* dense; either may be NULL for zeros */
  void *dresidual, *dout, *dgate;       /* dense; dresidual may be NULL */
  float *dpost, *dscale, *dpre;         /* [width], each there where its parameter is */
} uor_trunk_norms_args;

int uor_trunk_norms_async(const uor_trunk_norms_args *args, void *stream);
uint64_t uor_trunk_norms_backward_workspace_bytes(const uor_trunk_norms_args *args);
int uor_trunk_norms_backward_async(const uor_trunk_norms_args *args, void *workspace, uint64_t bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* UOR_TRUNK_H */
