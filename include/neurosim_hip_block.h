/*
 * neurosim_hip_block.h -- C ABI of the operators of a gated block: the gated projection
 * of rows and its backward pass, and dropout from a counter-based generator.  Conventions
 * (status codes, ns_last_error, caller's stream, no allocation, no synchronisation) are
 * those of neurosim_hip.h; element types are those of neurosim_hip_signal.h.  What a call
 * writes overlaps nothing that it reads.
 */
#ifndef NEUROSIM_HIP_BLOCK_H
#define NEUROSIM_HIP_BLOCK_H

#include <stdint.h>

#include "neurosim_hip_signal.h"   /* NS_TYPE_* */

#ifdef __cplusplus
extern "C" {
#endif

/* Dropout: out[e] = residual[e] + (kept(e) ? x[e] * scale : 0) for e < count, all dense.
 * kept(e) is that number e%8 of the eight 16-bit numbers of counter e/8 is at least
 * `threshold`; scale = 65536 / (65536 - threshold), or 0 for a threshold of 65536.  A
 * counter's numbers are the halves, low before high, of the four words of Philox4x32 with
 * 10 rounds (Salmon, Moraes, Dror and Shaw 2011) of the 128-bit counter (e/8, offset) under
 * the key `seed`, each 64-bit number low word first. */
typedef struct ns_dropout_args {
  int64_t count;
  int32_t type;                /* NS_TYPE_* */
  int32_t threshold;           /* 0 .. 65536 */
  const void* x;
  const void* residual;        /* or NULL */
  void* out;
  const int64_t* seed_data;    /* device: the seed; NULL: `seed` */
  int64_t seed, offset;
} ns_dropout_args;

int ns_dropout(const ns_dropout_args* args, void* stream);

/* Gated projection of M rows of K values to F: g = x gate^T, u = x up^T, y = f(g) u, with
 * f(g) = g sigmoid(g) or g Phi(g), Phi the normal distribution function.  Sums are float32.
 * Rows are dense, at strides in elements.  A backward rounds dg = dy u f'(g) and du = dy f(g) to
 * the type before it multiplies them (float16: as multiples of a power of two per row and column,
 * which keep them in range). */
#define NS_GATE_SILU 0
#define NS_GATE_GELU 1
#define NS_GATED_MAX_COLUMNS (1 << 20)     /* of K and of F */
#define NS_GATED_MAX_ROWS (1 << 21)        /* of a backward */

typedef struct ns_gated_args {
  int64_t rows, columns, width;            /* M, K, F */
  int32_t type;                            /* NS_TYPE_* of x, the weights, y and gradients */
  int32_t activation;                      /* NS_GATE_* */
  const void* x;                           /* [M][K] */
  int64_t x_stride;
  const void* gate;                        /* [F][K] */
  int64_t gate_stride;
  const void* up;                          /* [F][K] */
  int64_t up_stride;
  void* y;                                 /* [M][F] (forward) */
  int64_t y_stride;
  float* pre;                              /* g and u, [2][M][F]: kept by a forward (or NULL),
                                              read by the backward */
  const void* dy;                          /* [M][F] (backward) */
  int64_t dy_stride;
  void* dx;                                /* [M][K] dense, or NULL */
  void* dweights;                          /* [2][F][K] dense: of gate, of up; or NULL */
  void* workspace;                         /* 16-byte aligned */
} ns_gated_args;

/* Bytes of a pass's workspace for these arguments (addresses and strides count). */
int64_t ns_gated_forward_bytes(const ns_gated_args* args);
int64_t ns_gated_backward_bytes(const ns_gated_args* args);
int ns_gated_forward(const ns_gated_args* args, void* stream);
int ns_gated_backward(const ns_gated_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif  /* NEUROSIM_HIP_BLOCK_H */
