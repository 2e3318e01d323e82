/* C-ABI of the orthogonalisation of matrix updates by Newton-Schulz products (libsmel_moe.so, HIP for gfx950).
 *
 * Same conventions as smel_moe.h: raw device pointers, strides in elements, 0 on success or an SMEL_E* / hipError_t
 * code with the message in smel_last_error(), every kernel on `stream`, no allocation, no host synchronisation.
 */
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "smel_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* `batch` matrices x[b][i][j] at x + b x_batch + i x_row + j x_col (elements; x_row or x_col is 1 where that side has
 * more than one element), dtype 0 = bf16, 1 = fp32, 2 = fp16; y: the same matrices, contiguous [batch][rows][cols], of
 * x's dtype. min(rows, cols) <= 128, the longer side under 2^29 (2^30 up to a short side of 32). y overlaps no x of the call. */
typedef struct smel_ortho_job {
  const void* x;
  void* y;
  int64_t batch, rows, cols;
  int64_t x_batch, x_row, x_col;
  int64_t dtype;
} smel_ortho_job;

/* Bytes of the workspace that smel_orthogonalize needs for these jobs, steps and a (-1 for jobs that it does not take). */
int64_t smel_orthogonalize_ws(const smel_ortho_job* jobs, int32_t n_jobs, int32_t steps, double a);

/* Every matrix G of every job: X = G / (|G|_F + eps), then `steps` times X <- a X + b (X X^T) X + c (X X^T)^2 X, to y.
 * 0 <= steps <= 64: up to K steps, the most with a^(2 K) <= 2^24 (6 of the usual coefficients), on the r x r matrices of the short
 * side, G being read twice; up to 2 K in two such passes, more as the formula itself, step by step, the matrices kept in 64 bits in
 * the workspace: the result is the formula's in 64 bits in each (directions that G lacks then hold a^steps times its rounding, as
 * there: from about 28 steps on, anything of their size). ws: device memory of ws_bytes bytes, 16-byte aligned, not shared with a call that may run at the
 * same time. */
int smel_orthogonalize(const smel_ortho_job* jobs, int32_t n_jobs, int32_t steps, double a, double b, double c,
                       double eps, void* ws, int64_t ws_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif
