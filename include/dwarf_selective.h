/*
 * Entry points for a selective mixer beside the DSQG blocks (libdwarf_dsqg.so,
 * gfx950): RMS norm with the residual's addition (and with rows in 8 bits), a
 * short causal convolution of each channel, and the selective scan, for
 * training and prompts and (convolution, scan) single tokens.  Conventions
 * (status codes, strides in elements, dwarf_stream_t) are those of
 * dwarf_dsqg.h, element types those of dwarf_mixer.h.  Results share no memory
 * with the inputs or with each other; but a step's new_state may be its state,
 * and the pool that it writes shares none with the rest.
 */
#ifndef DWARF_SELECTIVE_H
#define DWARF_SELECTIVE_H

#include "dwarf_mixer.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * s = x + residual, rounded to residual_dtype (x itself where residual is NULL); y = s / sqrt(mean(s^2) + eps) *
 * weight[g] over the last D elements of each row, in fp32.  x [rows][groups][D] in dtype: row stride, group stride,
 * unit element stride; residual and sum the same shape in residual_dtype (dtype or DWARF_F32).  weight
 * [groups][D] fp32, contiguous, may be NULL (1).  y in dtype, rounded once; where scale is given, y holds e4m3
 * bytes instead: y / scale, scale [rows][groups] fp32 = max|y| / 448 of the row, at least the smallest normal fp32.
 */
typedef struct {
  int64_t rows;
  int32_t groups, D;
  int32_t dtype, residual_dtype;
  float eps;
  const void* x; int64_t x_stride[2];
  const void* residual; int64_t residual_stride[2];
  const float* weight;
  void* sum; int64_t sum_stride[2];
  void* y; int64_t y_stride[2];
  float* scale;
} dwarf_rms_norm_fwd_args;

int dwarf_rms_norm_fwd(const dwarf_rms_norm_fwd_args* args, dwarf_stream_t stream);

/*
 * The gradients, from the rows that were normalised: stream [rows][groups][D] in stream_dtype (x, or with a residual
 * the sum).  ds = the gradient through y, plus dsum (stream_dtype; NULL: zero); dx = ds in dtype, dresidual = ds in
 * stream_dtype (each may be NULL), dweight [groups][D] fp32 summed over the rows in a fixed order (may be NULL).
 */
typedef struct {
  int64_t rows;
  int32_t groups, D;
  int32_t dtype, stream_dtype;
  float eps;
  const void* stream; int64_t stream_stride[2];
  const float* weight;
  const void* dy; int64_t dy_stride[2];
  const void* dsum; int64_t dsum_stride[2];
  void* dx; int64_t dx_stride[2];
  void* dresidual; int64_t dresidual_stride[2];
  float* dweight;
  void* workspace; size_t workspace_bytes;   /* 16-byte aligned */
} dwarf_rms_norm_bwd_args;

size_t dwarf_rms_norm_bwd_workspace_bytes(const dwarf_rms_norm_bwd_args* args);
int dwarf_rms_norm_bwd(const dwarf_rms_norm_bwd_args* args, dwarf_stream_t stream);

/*
 * y_t = f(bias + sum_j weight[:, j] x_{t-W+1+j}) for each channel, f = silu where that is set; x and y [B][N][D]
 * (batch stride, token stride, unit channel stride), weight [D][W] and bias [D] fp32 (bias may be NULL),
 * 1 <= W <= 8.  In front of the first token lie the W - 1 rows of initial [B][W-1][D] (in dtype, contiguous; NULL:
 * zero).  Of each sequence the first lengths[b] tokens count (all where NULL; clamped to [0, N]): y is zero behind
 * them, and final [B][W-1][D] (may be NULL) holds the last W - 1 inputs in front of their end.
 */
typedef struct {
  int32_t B, N, D, W;
  int32_t dtype, silu;
  const void* x; int64_t x_stride[2];
  const float* weight;
  const float* bias;
  const int32_t* lengths;
  const void* initial;
  void* y; int64_t y_stride[2];
  void* final;
} dwarf_causal_conv_fwd_args;

int dwarf_causal_conv_fwd(const dwarf_causal_conv_fwd_args* args, dwarf_stream_t stream);

/*
 * The gradients for dy (and dfinal, NULL: zero): dx in dtype, dinitial in dtype (may be NULL), dweight [D][W] and
 * dbias [D] fp32 (each may be NULL), summed in a fixed order.  fwd.y and fwd.final are not used.
 */
typedef struct {
  dwarf_causal_conv_fwd_args fwd;
  const void* dy; int64_t dy_stride[2];
  const void* dfinal;
  void* dx; int64_t dx_stride[2];
  float* dweight;
  float* dbias;
  void* dinitial;
  void* workspace; size_t workspace_bytes;   /* 16-byte aligned */
} dwarf_causal_conv_bwd_args;

size_t dwarf_causal_conv_bwd_workspace_bytes(const dwarf_causal_conv_bwd_args* args);
int dwarf_causal_conv_bwd(const dwarf_causal_conv_bwd_args* args, dwarf_stream_t stream);

/*
 * One token of each of R rows against a pool [pool][W-1][D] of the rows in front of it (dtype; slot stride in
 * elements, each slot contiguous): row r takes slot slots[r] (r itself where slots is NULL).  The rows moved on by
 * one go to new_state (the pool itself, or another one of the same slot stride).  A slot outside [0, pool) marks a
 * row that pads the batch: no state is touched and its output is zero.  Rows of one slot are consecutive tokens of
 * its sequence, in row order.  x, out [R][D] by row stride.
 */
typedef struct {
  int32_t R, D, W, pool;
  int32_t dtype, silu;
  const void* x; int64_t x_stride;
  const float* weight;
  const float* bias;
  const int32_t* slots;
  const void* state;
  void* new_state;
  int64_t slot_stride;
  void* out; int64_t out_stride;
} dwarf_causal_conv_step_args;

int dwarf_causal_conv_step(const dwarf_causal_conv_step_args* args, dwarf_stream_t stream);

/*
 * The selective scan.  For each channel, with S states (1 <= S <= 64) and the group g of D / G channels it is in,
 *   step = delta + delta_bias, through softplus where that is set;  a = exp(step A)
 *   h_t = a h_{t-1} + step x_t B_t[g],   y_t = (C_t[g] . h_t + skip x_t) silu(gate_t)
 * over the first lengths[b] tokens (all N where NULL; clamped to [0, N]), y zero behind them and nothing used there.
 * x, delta, gate (may be NULL: factor 1) and y [B][N][D] (batch stride, token stride, unit channel stride); Bm, Cm
 * [B][N][G][S] (batch, token, group stride, unit state stride), all in dtype; token strides, the backward's too, lie in
 * [0, 2^22) elements, D below 2^22.  A [D][S], skip and delta_bias [D]
 * (each may be NULL: 0) fp32.  h_{-1} = initial [B][D][S] fp32 (NULL: zero), final [B][D][S] = the state behind the
 * last live token (may be NULL).  checkpoints: dwarf_selective_scan_checkpoint_bytes() bytes that the backward reads,
 * NULL where there will be none; with them the limit of the gradients, B G N + 4.2 D below 2^24, holds forward too.
 * A step of 0 passes the state on, also where A is minus infinity, and has no part in the gradients of A; under the
 * softplus, where a step of 0 has no slope, neither in those of delta and delta_bias.
 */
typedef struct {
  int32_t B, N, D, G, S;
  int32_t dtype, softplus;
  const void* x; int64_t x_stride[2];
  const void* delta; int64_t delta_stride[2];
  const void* gate; int64_t gate_stride[2];
  const void* Bm; int64_t B_stride[3];
  const void* Cm; int64_t C_stride[3];
  const float* A;
  const float* skip;
  const float* delta_bias;
  const int32_t* lengths;
  const float* initial;
  void* y; int64_t y_stride[2];
  float* final;
  float* checkpoints; size_t checkpoint_bytes;   /* 16-byte aligned */
  void* workspace; size_t workspace_bytes;       /* 16-byte aligned */
} dwarf_selective_scan_fwd_args;

size_t dwarf_selective_scan_checkpoint_bytes(const dwarf_selective_scan_fwd_args* args);
size_t dwarf_selective_scan_fwd_workspace_bytes(const dwarf_selective_scan_fwd_args* args);
int dwarf_selective_scan_fwd(const dwarf_selective_scan_fwd_args* args, dwarf_stream_t stream);

/*
 * The gradients for dy (and dfinal, NULL: zero): dx, ddelta, dgate (with a gate) in dtype at the given strides; dB,
 * dC [B][N][G][S] in dtype, contiguous; dA [D][S], dskip [D], ddelta_bias [D] fp32 and dinitial [B][D][S] fp32, each
 * of these four may be NULL.  fwd.checkpoints hold what the forward left there; fwd.y, fwd.final and
 * fwd.workspace are not used.  Sums run in a fixed order.
 */
typedef struct {
  dwarf_selective_scan_fwd_args fwd;
  const void* dy; int64_t dy_stride[2];
  const float* dfinal;
  void* dx; int64_t dx_stride[2];
  void* ddelta; int64_t ddelta_stride[2];
  void* dgate; int64_t dgate_stride[2];
  void* dB;
  void* dC;
  float* dA;
  float* dskip;
  float* ddelta_bias;
  float* dinitial;
  void* workspace; size_t workspace_bytes;       /* 16-byte aligned */
} dwarf_selective_scan_bwd_args;

size_t dwarf_selective_scan_bwd_workspace_bytes(const dwarf_selective_scan_bwd_args* args);
int dwarf_selective_scan_bwd(const dwarf_selective_scan_bwd_args* args, dwarf_stream_t stream);

/*
 * One token of each of R rows against a pool of states [pool][D][S] fp32 (slot stride in elements, each slot
 * contiguous), with the slots' rules of dwarf_causal_conv_step.  x, delta, gate and out [R][D] by row stride, Bm and
 * Cm [R][G][S] by row and group stride.
 */
typedef struct {
  int32_t R, D, G, S, pool;
  int32_t dtype, softplus;
  const void* x; int64_t x_stride;
  const void* delta; int64_t delta_stride;
  const void* gate; int64_t gate_stride;
  const void* Bm; int64_t B_stride[2];
  const void* Cm; int64_t C_stride[2];
  const float* A;
  const float* skip;
  const float* delta_bias;
  const int32_t* slots;
  const float* state;
  float* new_state;
  int64_t slot_stride;
  void* out; int64_t out_stride;
} dwarf_selective_scan_step_args;

int dwarf_selective_scan_step(const dwarf_selective_scan_step_args* args, dwarf_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DWARF_SELECTIVE_H */
