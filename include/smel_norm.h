/* C-ABI of the RMSNorm family around the MoE block, of layer norm and of the norms around a residual add (libsmel_moe.so, HIP for gfx950).
 *
 * Same conventions as smel_moe.h: raw device pointers, element counts and strides in elements, 0 on success or an
 * SMEL_E* / hipError_t code with the message in smel_last_error(), every kernel on `stream`, no allocation, no host
 * synchronisation. Rows of the RMSNorm entry points are 16-bit floats, `dtype` 0 = bf16, 1 = fp16; weights have the rows'
 * dtype and `cols` elements; rstd is one fp32 per row. 1 <= cols <= 16384 (the reference's MAX_COLS). fp32 math with the
 * reference's rounding points; each row's sum is a fixed-order reduction (bitwise repeatable).
 * `w_mode`: 0 = no weight (w may be null), 1 = w, 2 = 1 + w (Qwen3.5/3.6's plus_one).
 */
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "smel_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* y[r] = x[r] rstd[r] w', rstd[r] = 1 / sqrt(mean(x[r]^2) + eps); x rows at stride x_stride (>= cols), y and rstd
 * contiguous. Replaces `_rms_fwd` smel/norm.py:50-62 (launched by `_RMSNorm.forward` :157-171). */
int smel_rmsnorm_fwd(const uint16_t* x, int64_t rows, int64_t cols, int64_t x_stride, const uint16_t* w,
                     int32_t w_mode, float eps, int32_t dtype, uint16_t* y, float* rstd, hipStream_t stream);

/* dx = rstd (g - xhat mean(g xhat)) (+ ds), xhat = x rstd, g = dy w'; x at stride x_stride, dy / ds / dx contiguous,
 * ds may be null. Replaces `_rms_bwd` smel/norm.py:64-82 (`_RMSNorm.backward` :173-183 with ds null,
 * `_AddRMSNorm.backward` :204-219 with x = s and ds = the gradient of s). */
int smel_rmsnorm_bwd(const uint16_t* dy, const uint16_t* x, int64_t rows, int64_t cols, int64_t x_stride,
                     const uint16_t* w, int32_t w_mode, const float* rstd, const uint16_t* ds, int32_t dtype,
                     uint16_t* dx, hipStream_t stream);

/* s = round(h + x) (the residual stream), y = s rstd w' with rstd of s; all contiguous, w_mode 1 or 2 in the
 * reference (0 accepted). Replaces `_add_rms_fwd` smel/norm.py:84-100 (`_AddRMSNorm.forward` :186-202). */
int smel_add_rmsnorm_fwd(const uint16_t* h, const uint16_t* x, int64_t rows, int64_t cols, const uint16_t* w,
                         int32_t w_mode, float eps, int32_t dtype, uint16_t* s, uint16_t* y, float* rstd,
                         hipStream_t stream);

/* y = round(round(w round(x rstd)) silu(z)), the sigmoid on the hardware exp2 and reciprocal (the reference's
 * tl.sigmoid is Triton's fast form too); all contiguous, w required. Replaces `_gated_fwd`
 * smel/norm.py:102-119 (`_GatedRMSNorm.forward` :222-236). */
int smel_gated_rmsnorm_fwd(const uint16_t* x, const uint16_t* z, int64_t rows, int64_t cols, const uint16_t* w,
                           float eps, int32_t dtype, uint16_t* y, float* rstd, hipStream_t stream);

/* dz = dout y silu'(z); dn = round(round(dout silu(z)) w); dx = rstd (dn - xhat mean(dn xhat)); all contiguous.
 * Replaces `_gated_bwd` smel/norm.py:121-145 (`_GatedRMSNorm.backward` :238-249). */
int smel_gated_rmsnorm_bwd(const uint16_t* dout, const uint16_t* x, const uint16_t* z, int64_t rows, int64_t cols,
                           const uint16_t* w, const float* rstd, int32_t dtype, uint16_t* dx, uint16_t* dz,
                           hipStream_t stream);

/* Layer norm, y[r] = (x[r] - m) rstd w + b with m the mean and rstd = 1 / sqrt(mean((x[r] - m)^2) + eps) of the row.
 * `dtype` of the rows: 0 bf16, 1 fp16, 2 fp32; `wtype` of w and b (either may be null: 1 and 0): the rows' dtype or 2
 * (fp32). 1 <= cols <= 16384. h given: the norm of s = round(h + x), written to s (x_stride is both inputs' row stride;
 * h null: s is not touched). y, s contiguous; stats: 2 floats a row (m, rstd) for the backward. Any element alignment. */
int smel_layernorm_fwd(const void* x, const void* h, int64_t rows, int64_t cols, int64_t x_stride, const void* w,
                       const void* b, float eps, int32_t dtype, int32_t wtype, void* s, void* y, float* stats,
                       hipStream_t stream);

/* Floats of the workspace of smel_layernorm_bwd with dw or db (0 rows or columns: 0). */
int64_t smel_layernorm_bwd_ws_floats(int64_t rows, int64_t cols);

/* dx = rstd (g - mean(g) - xhat mean(g xhat)) (+ ds), g = dy w; dw = sum_r dy xhat, db = sum_r dy (fp32 sums, one rounding
 * to wtype). x: the rows that the norm read, at x_stride; dy, ds (may be null), dx contiguous; dx, dw, db may be null (not
 * computed). ws: smel_layernorm_bwd_ws_floats floats where dw or db is given. Each sum has a fixed order. */
int smel_layernorm_bwd(const void* dy, const void* x, int64_t rows, int64_t cols, int64_t x_stride, const void* w,
                       const float* stats, const void* ds, int32_t dtype, int32_t wtype, void* dx, void* dw, void* db,
                       float* ws, int64_t ws_floats, hipStream_t stream);

/* The norm behind a block, its gate, the residual add, the residual scale and the norm before the next block:
 *   n = x r1 w1',  s = round(scale (h + g n)),  y = s r2 w2'        r1, r2 = 1 / sqrt(mean of squares + eps) of x and of s
 * One call's arguments; fields that a call does not have are null or 0. Rows of `dtype` (0 bf16, 1 fp16, 2 fp32), 1 <= cols <= 16384;
 * x, h at row strides x_stride, h_stride, everything else contiguous; any element alignment. w1, w2 (null: 1) and a gate per channel
 * of `wtype` (the rows' dtype or 2); w' = 1 + w where plus_one. pre: with y (0: s alone). gate_kind 0 none, 1 [cols], 2 [rows] (of
 * gate_type: the rows' dtype or 2), 3 [rows][cols] (the rows' dtype); gate_act 1: g = sigmoid(gate), 0: g = gate. The scale is
 * scale_value, or the element at `scale` (of scale_type: the rows' dtype or 2). stats [rows][2]: r1, r2, written forward (null: not), read backward.
 * Backward: dS = ds + r2 (q - shat mean(q shat)), q = dy w2', shat = s r2; dh = scale dS; dn = dh g;
 *   dx = r1 (q1 - xhat mean(q1 xhat)), q1 = dn w1', xhat = x r1; dw1 = sum_r dn xhat, dw2 = sum_r dy shat;
 *   dgate = dh n (times g (1 - g)), summed over what the gate is broadcast over; dscale = sum of dS (h + g n)
 * ds, dy: either may be null; dy null: as without pre. dx, dh, dw1, dw2, dgate, dscale: each may be null (not computed); h is read for
 * dscale alone. Sums in fp32 (dscale's in 64 bits) in a fixed
 * order, one rounding per output. */
typedef struct smel_sandwich {
  const void *h, *x, *w1, *w2, *gate, *scale, *ds, *dy;
  void *s, *y, *dh, *dx, *dw1, *dw2, *dgate, *dscale;
  float* stats;
  int64_t rows, cols, x_stride, h_stride;
  float eps, scale_value;
  int32_t dtype, wtype, gate_kind, gate_type, gate_act, scale_type, plus_one, pre;
} smel_sandwich;

int smel_sandwich_fwd(const smel_sandwich* call, hipStream_t stream);
/* Floats of the workspace (8-byte aligned) of smel_sandwich_bwd for this call (0 where it needs none). */
int64_t smel_sandwich_bwd_ws_floats(const smel_sandwich* call);
int smel_sandwich_bwd(const smel_sandwich* call, float* ws, int64_t ws_floats, hipStream_t stream);

#ifdef __cplusplus
}
#endif
