/* C ABI of the gfx950 gradient norm and clipping (same library and
 * conventions as mm1_attn.h: the HIP stream as `void*`, caller-owned buffers,
 * no allocation, no synchronisation, return 0 / a negative MM1_E_* code / a
 * positive hipError_t).
 *
 * What the reference's training step does between the backward and the
 * optimizer (CODE/mimans/training/optim.py:114-179).
 *
 * The tensors are given by host arrays of `count` entries, read during the
 * call: in[i] (device pointer, at its element's alignment), f32[i] (1 fp32, 0
 * bf16) and cols[i] consecutive values, or, with `rows` not NULL, rows[i] runs
 * of cols[i] values that lie ld[i] elements apart (ld[i] >= cols[i]).  Empty
 * tensors are skipped and may have NULL pointers.  At most 2^31 - 1 pieces of
 * 4096 values (each run starts one) over all tensors.
 * norm: one fp32 on the device.  Sums are fp64, in a fixed order (bitwise
 * repeatable).
 */
#ifndef MM1_CLIP_H
#define MM1_CLIP_H

#include <stddef.h>

#include "mm1_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MM1_NORM_2 0       /* sqrt of the sum of squares */
#define MM1_NORM_MAX 1     /* largest magnitude (NaN if any value is) */

/* Bytes of scratch for `count` tensors. */
size_t mm1_grad_norm_workspace_size(int count);

/* norm of every value of every tensor (0 where there are none). */
int mm1_grad_norm(int count, const void* const* in, const long* rows, const long* cols, const long* ld,
                  const unsigned char* f32, int norm_type, float* norm, void* workspace, size_t workspace_bytes,
                  void* stream);

/* out[i] = in[i] * min(1, max_norm / (norm + eps)), each value rounded once
 * to its type, and the norm before clipping; a NaN norm makes every value NaN.
 * out NULL: in place (then nothing is written where nothing is clipped); else
 * its tensors have the types, rows and cols of in, runs ld_out[i] apart, and
 * no two tensors that are written may share memory, and out[i] lies at in[i] or in
 * no tensor of in (nor in norm).  norm_known: *norm holds
 * the norm already and is read, not computed.  max_norm >= 0, eps >= 0. */
int mm1_grad_clip(int count, const void* const* in, void* const* out, const long* rows, const long* cols,
                  const long* ld, const long* ld_out, const unsigned char* f32, int norm_type, float max_norm,
                  float eps, int norm_known, float* norm, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MM1_CLIP_H */
