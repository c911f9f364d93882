/* C ABI of the gfx950 products with bias, activation and residual in their
 * epilogue, and of the elementwise part of their gradients (same library and
 * conventions as mm1_attn.h and mm1_gemm.h: bf16 tensors as `void*`, the HIP
 * stream as `void*`, caller-owned buffers, no allocation, no synchronisation,
 * return 0 / a negative MM1_E_* code / a positive hipError_t).
 *
 * The output and down projections with the residual stream's addition behind
 * them, which the reference runs as torch products and additions
 * (CODE/mimans/model/attention_tilelang.py:518, swiglu_tilelang.py:284-286,
 * block.py:81-92).
 */
#ifndef MM1_LINEAR_H
#define MM1_LINEAR_H

#include <stddef.h>

#include "mm1_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MM1_ACT_NONE 0
#define MM1_ACT_RELU 1
#define MM1_ACT_GELU 2         /* z Phi(z) */
#define MM1_ACT_GELU_TANH 3    /* z / 2 (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) */
#define MM1_ACT_SILU 4

/* Bytes of scratch mm1_linear needs for these sizes, layouts and activation (0
 * for many, and for those it refuses). */
size_t mm1_linear_workspace_size(int M, int N, int K, int x_layout, int w_layout, int act);

/* z[m][n] = sum_k x(m, k) w(n, k) + bias[n]; out = act(z) + residual; pre =
 * bf16(z), for the backward of an activation (else NULL).  bf16 x and w, fp32 sums and epilogue, one rounding
 * to out's type (fp32, or bf16 where out_f32 = 0).  bias [N] and residual [M, N]
 * may be NULL; *_f32 says their type; ldr, ldp and ldo are the row strides of
 * residual, pre and out, which lie at any element alignment: at most 2^24, and
 * 2^23 for fp32 tensors of more than 64 rows.
 * x and w as in mm1_gemm: MM1_GEMM_ROW or _COL (x ROW with w ROW or COL, or both
 * COL, which takes no activation), strides multiples of 8, 16-byte aligned, but
 * with any M, N and K >= 1 (bounded as in mm1_gemm, K <= 2^28): a row of an operand
 * is readable up to the next multiple of 8 values, and where the row runs along k
 * (ROW) what lies behind K there is zeros.  Deterministic. */
int mm1_linear(const void* x, int x_layout, long ldx, const void* w, int w_layout, long ldw, const void* bias,
               int bias_f32, int act, const void* residual, int residual_f32, long ldr, void* pre, long ldp,
               void* out, int out_f32, long ldo, void* workspace, size_t workspace_bytes, int M, int N, int K,
               void* stream);

/* Bytes of scratch mm1_linear_backward needs for the gradients that it is asked
 * for; dz: whether it has to form dz, which it has not where there is no
 * activation and dy is bf16, 16-byte aligned, with N and ldy multiples of 8. */
size_t mm1_linear_backward_workspace_size(int M, int N, int K, int dz, int dx, int dw, int dbias);

/* The gradients of act(x w^T + bias) from dy [M, N], fp32 or bf16, each written
 * unless it is NULL: with dz = dy act'(z), z from pre (not read without an
 * activation),
 *   dx [M, K] = dz w,  dw = dz^T x in w's own layout ([N, K] for ROW, [K, N] for
 *   COL; contiguous),  dbias [N] = sum over the rows of dz.  N and K as mm1_linear's
 *   strides.
 * dz is fp32; it enters the products rounded to bf16 (dy itself where it is bf16
 * and there is no activation) and dbias as it is.  fp32 sums in a fixed order, one
 * rounding to each result's type.  x [M, K] ROW and w as mm1_linear takes them
 * (not read for the gradients left out). */
int mm1_linear_backward(const void* dy, int dy_f32, long ldy, const void* pre, long ldp, int act, const void* x,
                        long ldx, const void* w, int w_layout, long ldw, void* dx, int dx_f32, void* dw, int dw_f32,
                        void* dbias, int dbias_f32, void* workspace, size_t workspace_bytes, int M, int N, int K,
                        void* stream);

/* dst [rows_out, ldd] bf16 = src [rows, cols] (fp32, rounded to nearest even, or
 * bf16; rows ld elements apart, at any element alignment), and zeros in columns
 * cols .. ldd - 1 and rows rows .. rows_out - 1: an operand at the sizes that
 * the products take.  ldd a multiple of 8, dst 16-byte aligned. */
int mm1_pack_bf16(const void* src, int src_f32, long ld, int rows, int cols, void* dst, long ldd, int rows_out,
                  void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MM1_LINEAR_H */
