/*
 * b200_lora.h — low-rank adapters of many requests at once, beside a shared projection.
 *
 * The denoising loop runs every request's tokens through one GEMM per linear
 * (src/transformer.rs:179-196, 326-331 run them request by request).  Requests may carry
 * adapters of their own (W + scale B A, as image-model adapters are distributed): the shared
 * product y = x W^T stays one GEMM, and this adds each request's low-rank part:
 *
 *   out[r, :] = y[r, :] + scale[e] * (x[r, :] A[e]^T) B[e]^T,   e = adapter of r's request
 *
 * x A^T is summed in f32, scaled and rounded to bf16 once; its product with B^T is summed in
 * f32, added to y in f32 and rounded to bf16 once.  One launch; sums in a fixed order.
 *
 * Conventions are those of b200_attn.h.
 */
#ifndef B200_LORA_H
#define B200_LORA_H

#include <stddef.h>
#include <stdint.h>

#include "b200_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200_LORA_MAX_RANK 128
#define B200_LORA_STATUS_BAD_ADAPTER 16

/*
 *   x    device bf16 [rows, k], row stride ldx      a  device bf16 [adapters, rank, k]
 *   y    device bf16 [rows, n], row stride ldy      b  device bf16 [adapters, n, rank]
 *   out  device bf16 [rows, n], row stride ldo; out == y (with ldo == ldy) adds in place.
 *        Otherwise out overlaps y in no element, and in either case a row of out no other row
 *        of x (B200_ERR_INVALID); columns of one buffer that keep apart are no overlap
 *   seg_start   device int32 [segments + 1], non-decreasing: request s has the rows
 *               [seg_start[s], seg_start[s + 1]); limited to [0, rows]
 *   seg_adapter device int32 [segments]: the request's adapter, negative for none (its rows
 *               are copied from y).  An index >= adapters counts as none, and leaves
 *               B200_LORA_STATUS_BAD_ADAPTER in status (optional device int32, if it was 0)
 *   scale       device f32 [adapters], or NULL (1)
 * Rows of no request are not written.  Adapters of a lower rank are padded with zeros.
 * n, k and rank are multiples of 8, rank <= 128, strides multiples of 8; 16-byte alignment.
 */
int b200_lora_add(const void* x, int64_t ldx, const void* a, const void* b, const void* y,
                  int64_t ldy, void* out, int64_t ldo, const int32_t* seg_start,
                  const int32_t* seg_adapter, const float* scale, int32_t rows,
                  int32_t segments, int32_t adapters, int32_t n, int32_t k, int32_t rank,
                  int32_t* status, b200_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* B200_LORA_H */
