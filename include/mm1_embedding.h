/* C ABI of the gfx950 embedding lookup and its gradient (same library and
 * conventions as mm1_attn.h: the HIP stream as `void*`, caller-owned buffers,
 * no allocation, no synchronisation, return 0 / a negative MM1_E_* code / a
 * positive hipError_t).
 *
 * What the reference leaves to torch's nn.Embedding, whose matrix its tied
 * output head reads (CODE/mimans/model/model.py:53-127,
 * lm_head_tilelang.py:284-338).
 *
 * ids are int64 (ids_wide = 1) or int32 (0).  An id outside [0, vocab) -- the
 * fill of a padded batch, such as -100 -- looks up a row of zeros and adds to
 * no gradient.  Matrices are fp32 (*_f32 = 1) or bf16 (0) with rows of
 * consecutive values, ld* elements apart, at any element alignment; sums and
 * products are fp32, rounded once.
 * Sizes: tokens >= 0, vocab and dim >= 1, vocab <= 2^30, tokens <= 2^26, at
 * most 2^32 - 256 pieces of eight columns over all tokens.
 */
#ifndef MM1_EMBEDDING_H
#define MM1_EMBEDDING_H

#include <stddef.h>

#include "mm1_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* out[t] = scale * weight[ids[t]], out [tokens, dim], weight [vocab, dim]. */
int mm1_embedding(const void* ids, int ids_wide, const void* weight, int weight_f32, long ldw, void* out,
                  int out_f32, long ldo, float scale, long tokens, int vocab, int dim, void* stream);

/* Bytes of scratch mm1_embedding_grad needs (0 also for sizes it refuses). */
size_t mm1_embedding_grad_workspace_size(long tokens, int vocab, int dim);

/* grad[v] = scale * sum of d_out[t] over the tokens with ids[t] == v, in the
 * order of the tokens whatever the scheduling (bitwise repeatable); rows
 * without tokens are cleared.  With accumulate the sums are added to grad, in
 * fp32 with one rounding, and rows without tokens are left as they are.
 * padding_idx: the row that takes no gradient, -1 for none.  ld_d_out may be 0
 * (one gradient row for every token).  grad shares no memory with ids or d_out:
 * it is cleared and written while they are read. */
int mm1_embedding_grad(const void* ids, int ids_wide, const void* d_out, int d_out_f32, long ld_d_out, void* grad,
                       int grad_f32, long ldg, float scale, long padding_idx, int accumulate, void* workspace,
                       size_t workspace_bytes, long tokens, int vocab, int dim, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MM1_EMBEDDING_H */
