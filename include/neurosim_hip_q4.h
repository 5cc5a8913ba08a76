/*
 * neurosim_hip_q4.h -- C ABI of the 4-bit integer operators with a scale per group of
 * columns: quantisation of float rows, reading them back, and the product of float rows
 * with such a matrix.  Conventions (status codes, ns_last_error, caller's stream, no
 * allocation, no synchronisation) are those of neurosim_hip.h.
 *
 * Format: a row of K values is cut into groups of `group` consecutive values (32, 64, or a
 * multiple of 128 up to NS_Q4_MAX_COLUMNS; the last one may be short).  A value is (code - zero) * scale with codes of
 * 0 .. 15, two a byte (even value in the low nibble), rows filled up to whole 16 bytes
 * (ceil(K/32) of them); one scale of a float type and one byte `zero` per group (no zeros: 8).
 * Quantising, with lo = min(0, min x), hi = max(0, max x): scale = hi/15 - lo/15 rounded to its
 * type, zero = round(-lo/scale) in [0, 15], code = round(x/scale) + zero in [0, 15]; without
 * zeros scale = max|x|/7, code = round(x/scale) + 8; ties to even.  A scale of 0 gives values
 * of 0; a group with an infinity or NaN, or whose scale its type cannot hold, has scale NaN
 * and codes 0.
 */
#ifndef NEUROSIM_HIP_Q4_H
#define NEUROSIM_HIP_Q4_H

#include <stdint.h>

#include "neurosim_hip_signal.h"   /* NS_TYPE_* */

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ns_q4_matrix {
  int64_t rows, columns;       /* N, K (up to NS_Q4_MAX_COLUMNS) */
  int64_t group;               /* columns per scale */
  uint8_t* codes;              /* [N][ceil(K/32)][16], 16-byte aligned */
  void* scales;                /* [N][ceil(K/group)] */
  uint8_t* zeros;              /* [N][ceil(K/group)], or NULL */
  int32_t scale_type;          /* NS_TYPE_* of the scales */
  int32_t reserved;
} ns_q4_matrix;

#define NS_Q4_MAX_COLUMNS (1 << 23)

/* Codes, scales and zeros (where `zeros` is given) from float rows x[r*stride + k]. */
int ns_q4_quantize(const ns_q4_matrix* matrix, const void* x, int64_t stride, int32_t type,
                   void* stream);
/* The values of `matrix`, out[r*stride + k], rounded to `type`. */
int ns_q4_dequantize(const ns_q4_matrix* matrix, void* out, int64_t stride, int32_t type,
                     void* stream);

/* y[m][n] = sum_k x[m][k] weight[n][k] + bias[n], sums in float32, rounded to `type`.  The sum of a
 * group (of 128 columns at most) is off by some 2^-24 of scale (16 + zero) sum |x|, in float32 of
 * scale (16 + zero) sum |x - their mean|, columns of weight zero among them.  A row of x that holds
 * an infinity or a NaN gives NaN, and one with values beyond 2^115, 128 of which times a code pass
 * float32, may. */
typedef struct ns_q4_product_args {
  ns_q4_matrix weight;
  int64_t rows;                /* M */
  const void* x;               /* x[m*x_stride + k] */
  int64_t x_stride;
  const float* bias;           /* [N] or NULL */
  void* out;                   /* out[m*stride + n] */
  int64_t stride;
  int32_t type;                /* NS_TYPE_* of x and out */
  int32_t reserved;
  float* workspace;            /* ns_q4_product_floats floats */
} ns_q4_product_args;

/* Floats of a product's workspace (0: none needed). */
int64_t ns_q4_product_floats(int64_t m, int64_t n, int64_t k, int32_t type);
int ns_q4_product(const ns_q4_product_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif  /* NEUROSIM_HIP_Q4_H */
