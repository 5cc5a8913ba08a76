/*
 * neurosim_hip_mx.h -- C ABI of the microscaled 4-bit operators: quantisation of float
 * rows, reading them back, and the product of two quantised matrices.  Conventions
 * (status codes, ns_last_error, caller's stream, no allocation, no synchronisation) are
 * those of neurosim_hip.h.
 *
 * Format (OCP microscaling, MXFP4): a row of K values is cut into ceil(K/32) blocks of 32
 * consecutive values (the last filled up with zeros).  A block has 16 bytes of e2m1 codes
 * (even value in the low nibble; magnitudes 0 .5 1 1.5 2 3 4 6, bit 3 the sign) and one
 * scale byte e: its values are code * 2^(e-127), or NaN where e is 255.
 * Quantising: e - 127 = floor(log2(max|x|)) - 2 clamped to [-127, 127] (max|x| = 0: -127);
 * codes are x 2^(127-e) rounded to nearest, ties to the even code, at most 6 in size.  A
 * block that holds an infinity or a NaN gets e = 255 and codes 0.
 */
#ifndef NEUROSIM_HIP_MX_H
#define NEUROSIM_HIP_MX_H

#include <stdint.h>

#include "neurosim_hip_signal.h"   /* NS_TYPE_* */

#ifdef __cplusplus
extern "C" {
#endif

#define NS_MX_BLOCK 32

/* Rows of one matrix: codes [rows][blocks][16] (16-byte aligned), scales [rows][blocks]. */
typedef struct ns_mx_matrix {
  int64_t rows, columns;       /* columns: K, blocks = ceil(K/32) */
  uint8_t* codes;
  uint8_t* scales;
} ns_mx_matrix;

/* Codes and scales of `matrix` from float rows x[r*stride + k] of type `type`. */
int ns_mx_quantize(const ns_mx_matrix* matrix, const void* x, int64_t stride, int32_t type,
                   void* stream);
/* The values of `matrix`, out[r*stride + k], rounded to `type`. */
int ns_mx_dequantize(const ns_mx_matrix* matrix, void* out, int64_t stride, int32_t type,
                     void* stream);

/* y[m*stride + n] = sum_k a[m,k] b[n,k] + bias[n], summed in float32, rounded to `type`.
 * With float rows `x` for a, they are quantised first (a.codes and a.scales are then not
 * read: the workspace holds them). */
typedef struct ns_mx_product_args {
  ns_mx_matrix a, b;           /* M rows and N rows of K columns (K up to NS_MX_MAX_COLUMNS) */
  const float* bias;           /* [N] or NULL */
  void* out;
  int64_t stride;
  int32_t type;                /* NS_TYPE_* of out */
  int32_t x_type;              /* NS_TYPE_* of x */
  const void* x;               /* optional: a's rows as floats, x[m*x_stride + k] */
  int64_t x_stride;
  void* workspace;             /* ns_mx_product_bytes bytes, 16-byte aligned */
} ns_mx_product_args;

#define NS_MX_MAX_COLUMNS (1 << 23)

/* Bytes of a product's workspace, with float rows for a or without (0: none needed). */
int64_t ns_mx_product_bytes(int64_t m, int64_t n, int64_t k, int32_t float_rows);
int ns_mx_product(const ns_mx_product_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif  /* NEUROSIM_HIP_MX_H */
