/* C-ABI of the global gradient norm and the clipping by it (libsmel_moe.so, HIP for gfx950).
 *
 * Same conventions as smel_moe.h: raw device pointers, 0 on success or an SMEL_E* / hipError_t code with the message in
 * smel_last_error(), every kernel on `stream`, no allocation on the device, no host synchronisation.
 */
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "smel_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* n values of dtype (0 bf16, 1 fp32, 2 fp16) at in, and where the scaled ones go (out == in: in place). Element alignment. */
typedef struct smel_clip_job {
  const void* in;
  void* out;
  int64_t n, dtype;
} smel_clip_job;

/* Bytes of the workspace of the calls below for these jobs (-1 for jobs that they do not take). */
int64_t smel_clip_ws(const smel_clip_job* jobs, int32_t n_jobs);

/* *norm = the norm of all values of all jobs together: norm_type 0: sqrt(sum of squares) (64-bit sums, fixed order), 1: the largest
 * magnitude. No values: 0. A NaN gives NaN. `out` is not looked at. ws: device memory of ws_bytes bytes, 16-byte aligned, not
 * shared with a call that may run at the same time. */
int smel_grad_norm(const smel_clip_job* jobs, int32_t n_jobs, int32_t norm_type, float* norm, void* ws, int64_t ws_bytes,
                   hipStream_t stream);

/* The norm as above, and out = round(in c) with c = min(1, max_norm / (norm + eps)), of every job; c = 1 leaves in-place values as they
 * are. An out that overlaps anything but its own job's in, at the same address, is refused. */
int smel_clip_grads(const smel_clip_job* jobs, int32_t n_jobs, int32_t norm_type, double max_norm, double eps, float* norm,
                    void* ws, int64_t ws_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif
