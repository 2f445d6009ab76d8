/*
 * Entry points for a sequence mixer beside the DSQG blocks (libdwarf_dsqg.so,
 * gfx950): layer norm, rotary positions, and linear attention with a decay for
 * each head (prompts and training with gradients, single tokens).
 * Conventions (status codes, strides in elements, dwarf_stream_t) are those of
 * dwarf_dsqg.h.
 */
#ifndef DWARF_MIXER_H
#define DWARF_MIXER_H

#include "dwarf_dsqg.h"

#ifdef __cplusplus
extern "C" {
#endif

/* fp16 elements: a dtype of this header's entry points and dwarf_selective.h's only (with DWARF_BF16 and DWARF_F32). */
#define DWARF_F16 2

/*
 * y = (x - mean) / sqrt(var + eps) * weight[g] + bias[g] over the last D elements of each row, statistics in fp32,
 * one rounding at the end.  x [rows][groups][D] in x_dtype: row stride, group stride, unit element stride; y the
 * same shape and dtype.  weight and bias [groups][D] fp32, contiguous, each may be NULL (1 and 0).
 */
typedef struct {
  int64_t rows;
  int32_t groups, D;
  int32_t dtype;
  float eps;
  const void* x; int64_t x_stride[2];
  const float* weight;
  const float* bias;
  void* y; int64_t y_stride[2];
} dwarf_layer_norm_fwd_args;

int dwarf_layer_norm_fwd(const dwarf_layer_norm_fwd_args* args, dwarf_stream_t stream);

/*
 * The gradients: dx in dtype (may be NULL), dweight and dbias [groups][D] fp32 (each may be NULL), summed over the
 * rows in a fixed order.  The statistics are formed again from x.  fwd.bias and fwd.y are not used.
 */
typedef struct {
  dwarf_layer_norm_fwd_args fwd;
  const void* dy; int64_t dy_stride[2];
  void* dx; int64_t dx_stride[2];
  float* dweight;
  float* dbias;
  void* workspace; size_t workspace_bytes;   /* 16-byte aligned */
} dwarf_layer_norm_bwd_args;

size_t dwarf_layer_norm_bwd_workspace_bytes(const dwarf_layer_norm_bwd_args* args);
int dwarf_layer_norm_bwd(const dwarf_layer_norm_bwd_args* args, dwarf_stream_t stream);

/*
 * Rotary positions of q [B,H,N,D] and, unless it is NULL, k [B,H_kv,N,D]: pair i of the first 2 * pairs elements
 * is turned by the angle 2 pi position turns[i] / 2^64 (backwards where inverse is set) and scaled by magnitude;
 * the other elements are copied.  The pair is (2i, 2i+1) where interleaved is set and (i, i + pairs) where not.
 * turns: the angle per position in 2^-64 turns, so position * turns wraps exactly.  positions: int64, or int32
 * where position_bytes is 4, element [b][n] at the given strides (0 for one position list of the whole batch).
 * Outputs must not overlap the inputs.
 */
typedef struct {
  int32_t B, H, H_kv, N, D, pairs;
  int32_t dtype, interleaved, inverse, position_bytes;
  float magnitude;
  const void* q; int64_t q_stride[4];
  const void* k; int64_t k_stride[4];
  const void* positions; int64_t position_stride[2];
  const uint64_t* turns;
  void* q_out; int64_t q_out_stride[4];
  void* k_out; int64_t k_out_stride[4];
} dwarf_rotary_args;

int dwarf_rotary(const dwarf_rotary_args* args, dwarf_stream_t stream);

/*
 * Linear attention with a decay for each head.  With g = exp(min(log_decay[h], 0)),
 *   S_t = g S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t
 * over the first lengths[b] tokens (all N where lengths is NULL; clamped to [0, N]); the output rows behind them
 * are zero and q, k, v are not used there.  q and out [B,H,N,64], k and v [B,H_kv,N,64], H a multiple of H_kv;
 * S_{-1} = initial [B,H,64,64] fp32 contiguous (NULL: zero), final [B,H,64,64] = the state behind the last live
 * token (may be NULL).  states: [B,H,segments,64,64] fp32, the state in front of each segment of
 * dwarf_linear_attention_segment() tokens, written where there is more than one segment; the backward reads it.
 */
typedef struct {
  int32_t B, H, H_kv, N, head_dim;
  int32_t dtype;
  float scale;
  const void* q; int64_t q_stride[4];
  const void* k; int64_t k_stride[4];
  const void* v; int64_t v_stride[4];
  const float* log_decay;
  const int32_t* lengths;
  const float* initial;
  void* out; int64_t out_stride[4];
  float* final;
  float* states; size_t states_bytes;        /* 16-byte aligned */
} dwarf_linear_attention_fwd_args;

/* Tokens of a segment for these sizes: a rule on B, H and N alone. */
int32_t dwarf_linear_attention_segment(int32_t B, int32_t H, int32_t N);
size_t dwarf_linear_attention_states_bytes(const dwarf_linear_attention_fwd_args* args);
int dwarf_linear_attention_fwd(const dwarf_linear_attention_fwd_args* args, dwarf_stream_t stream);

/*
 * The gradients for dout (and dfinal, NULL: zero): dq, dk, dv in dtype; dlog_decay [H] fp32 and dinitial
 * [B,H,64,64] fp32, each may be NULL.  fwd.states holds what the forward left there; fwd.final the final state
 * where both dfinal and dlog_decay are given; fwd.out is not used.  dlog_decay is 0 where log_decay > 0.
 */
typedef struct {
  dwarf_linear_attention_fwd_args fwd;
  const void* dout; int64_t dout_stride[4];
  const float* dfinal;
  void* dq; int64_t dq_stride[4];
  void* dk; int64_t dk_stride[4];
  void* dv; int64_t dv_stride[4];
  float* dlog_decay;
  float* dinitial;
  void* workspace; size_t workspace_bytes;   /* 16-byte aligned */
} dwarf_linear_attention_bwd_args;

size_t dwarf_linear_attention_bwd_workspace_bytes(const dwarf_linear_attention_bwd_args* args);
int dwarf_linear_attention_bwd(const dwarf_linear_attention_bwd_args* args, dwarf_stream_t stream);

/*
 * One token of each of S rows against a pool of states [pool][H][64][64] fp32 (slot stride in elements, each slot
 * contiguous): row s takes slot slots[s] (s itself where slots is NULL), S' = g S + k v^T, out = scale q S'.  The
 * new state goes to new_state (the pool itself, or another one of the same slot stride).  A slot outside
 * [0, pool) marks a row that pads the batch: no state is touched and its output is zero.  Rows of one slot are
 * consecutive tokens of its sequence, in row order.  q, out [S,H,64], k, v [S,H_kv,64]; out shares no memory with
 * the others.
 */
typedef struct {
  int32_t S, H, H_kv, pool, head_dim;
  int32_t dtype;
  float scale;
  const void* q; int64_t q_stride[3];
  const void* k; int64_t k_stride[3];
  const void* v; int64_t v_stride[3];
  const float* log_decay;
  const int32_t* slots;
  const float* state;
  float* new_state;
  int64_t slot_stride;
  void* out; int64_t out_stride[3];
} dwarf_linear_attention_step_args;

int dwarf_linear_attention_step(const dwarf_linear_attention_step_args* args, dwarf_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DWARF_MIXER_H */
