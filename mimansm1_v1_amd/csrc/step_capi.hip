// extern "C" entry points of the operators around the step's kernels (the
// embedding, the products with an epilogue, the gradient clip): argument checks, then the launchers.
#include <math.h>
#include <stdint.h>

#include "../../include/mm1_clip.h"
#include "../../include/mm1_embedding.h"
#include "../../include/mm1_linear.h"
#include "embedding.h"
#include "gemm.h"
#include "grad_clip.h"
#include "linear.h"

namespace {

int from_hip(hipError_t e) { return e == hipSuccess ? MM1_OK : static_cast<int>(e); }

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }
bool element_aligned(const void* p, bool f32) { return aligned(p, f32 ? 4 : 2); }

constexpr long kMaxTokens = 1L << 26, kMaxLd = 1L << 40;
constexpr int kMaxVocab = 1 << 30;

// 32-bit piece and thread counts inside the kernels and their grids.
bool embedding_sizes_ok(long tokens, int vocab, int dim) {
  if (tokens < 0 || tokens > kMaxTokens || vocab < 1 || vocab > kMaxVocab || dim < 1) return false;
  const long pieces = ((long)dim + 7) / 8, slabs = ((long)dim + 511) / 512;
  return tokens * pieces <= (1L << 32) - 256 && (tokens + 7) / 8 * slabs < (1L << 24);
}

// A row stride that the epilogue takes: 32-bit byte offsets inside the rows of a wave's block, of
// which it touches no more than M, up to 56 columns into a row.
bool epilogue_ld_ok(long ld, bool f32, int M, int N) {
  const long rows = M < mm1::EPILOGUE_ROWS ? M : mm1::EPILOGUE_ROWS;
  return ld >= N && ld <= (1L << 24) && ((rows - 1) * ld + 64) * (f32 ? 4 : 2) <= (1L << 32);
}

bool linear_sizes_ok(int M, int N, int K) {
  return M >= 1 && N >= 1 && K >= 1 && M <= (1 << 28) && N <= (1 << 28) && K <= (1 << 28) &&
         ((long)M + 255) / 256 * (((long)N + 255) / 256) <= (1L << 24);
}

int ceil8(int n) { return (n + 7) & ~7; }

// Rows of an operand readable to the next multiple of 8 values, 32-bit copies.
bool operand_ok(int layout, long ld, int n, int K) {
  const int n8 = layout == MM1_GEMM_COL ? ceil8(n) : n, k8 = layout == MM1_GEMM_COL ? K : ceil8(K);
  return ld % 8 == 0 && ld >= (layout == MM1_GEMM_COL ? n8 : k8) && mm1::gemm_operand_fits(layout, ld, n8, k8);
}

// Regions of mm1_linear_backward's scratch: dz, then what one launch needs.
struct BackwardScratch {
  size_t dz, bytes;
};
BackwardScratch backward_scratch(int M, int N, int K, bool dz, bool dx, bool dw, bool dbias) {
  BackwardScratch s{};
  if (dz && (dx || dw)) s.dz = ((size_t)M * ceil8(N) * 2 + 255) & ~(size_t)255;
  size_t most = 0;
  auto need = [&](bool asked, size_t bytes) {
    if (asked && bytes > most) most = bytes;
  };
  need(dbias, mm1::linear_grad_workspace_bytes(M, N));
  need(dx, mm1::linear_workspace_bytes(M, K, N, MM1_GEMM_ROW, MM1_GEMM_COL, false));     // enough for a ROW w too
  need(dw, mm1::linear_workspace_bytes(N, K, M, MM1_GEMM_COL, MM1_GEMM_COL, false));
  need(dw, mm1::linear_workspace_bytes(K, N, M, MM1_GEMM_COL, MM1_GEMM_COL, false));
  s.bytes = s.dz + most;
  return s;
}

int check_clip(const mm1::ClipArgs& a, bool writes) {
  if (a.count < 0) return MM1_E_SHAPE;
  if (a.count > 0 && (!a.in || !a.cols || !a.f32 || (a.rows && !a.ld_in) || (a.rows && writes && !a.ld_out)))
    return MM1_E_NULL;
  for (int i = 0; i < a.count; ++i) {
    if (a.cols[i] < 0 || a.cols[i] > kMaxLd) return MM1_E_SHAPE;
    if (a.rows && (a.rows[i] < 0 || a.rows[i] > INT32_MAX || a.ld_in[i] < a.cols[i] || a.ld_in[i] > kMaxLd ||
                   (writes && (a.ld_out[i] < a.cols[i] || a.ld_out[i] > kMaxLd))))
      return MM1_E_SHAPE;
    if (a.cols[i] == 0 || (a.rows && a.rows[i] == 0)) continue;
    if (!a.in[i] || (writes && !a.out[i])) return MM1_E_NULL;
    if (!element_aligned(a.in[i], a.f32[i]) || (writes && !element_aligned(a.out[i], a.f32[i]))) return MM1_E_ALIGN;
  }
  return mm1::clip_sizes_ok(a) ? MM1_OK : MM1_E_SHAPE;
}

}  // namespace

extern "C" {

int mm1_embedding(const void* ids, int ids_wide, const void* weight, int weight_f32, long ldw, void* out,
                  int out_f32, long ldo, float scale, long tokens, int vocab, int dim, void* stream) {
  if (!embedding_sizes_ok(tokens, vocab, dim) || ldw < dim || ldo < dim || ldw > kMaxLd || ldo > kMaxLd)
    return MM1_E_SHAPE;
  if (tokens == 0) return MM1_OK;
  if (!ids || !weight || !out) return MM1_E_NULL;
  if (!aligned(ids, ids_wide ? 8 : 4) || !element_aligned(weight, weight_f32) || !element_aligned(out, out_f32))
    return MM1_E_ALIGN;
  return from_hip(mm1::launch_embedding({ids, ids_wide, weight, weight_f32 != 0, ldw, out, out_f32 != 0, ldo, scale,
                                         tokens, vocab, dim},
                                        static_cast<hipStream_t>(stream)));
}

size_t mm1_embedding_grad_workspace_size(long tokens, int vocab, int dim) {
  return embedding_sizes_ok(tokens, vocab, dim) ? mm1::embedding_grad_workspace_bytes(tokens, vocab, dim) : 0;
}

int mm1_embedding_grad(const void* ids, int ids_wide, const void* d_out, int d_out_f32, long ld_d_out, void* grad,
                       int grad_f32, long ldg, float scale, long padding_idx, int accumulate, void* workspace,
                       size_t workspace_bytes, long tokens, int vocab, int dim, void* stream) {
  if (!embedding_sizes_ok(tokens, vocab, dim) || ldg < dim || ldg > kMaxLd || padding_idx < -1 ||
      padding_idx >= vocab || (ld_d_out < dim && ld_d_out != 0) || ld_d_out > kMaxLd)
    return MM1_E_SHAPE;
  if (!grad || (tokens > 0 && (!ids || !d_out))) return MM1_E_NULL;
  if (!element_aligned(grad, grad_f32) || !element_aligned(d_out, d_out_f32) || !aligned(ids, ids_wide ? 8 : 4) ||
      !aligned(workspace, 16))
    return MM1_E_ALIGN;
  const size_t need = mm1::embedding_grad_workspace_bytes(tokens, vocab, dim);
  if (need > 0 && (!workspace || workspace_bytes < need)) return MM1_E_WORKSPACE;
  if (tokens == 0 && accumulate) return MM1_OK;
  return from_hip(mm1::launch_embedding_grad({ids, ids_wide, d_out, d_out_f32 != 0, ld_d_out, grad, grad_f32 != 0,
                                              ldg, scale, padding_idx, accumulate != 0, workspace, tokens, vocab, dim},
                                             static_cast<hipStream_t>(stream)));
}

size_t mm1_grad_norm_workspace_size(int count) { return count < 0 ? 0 : mm1::clip_workspace_bytes(count); }

int mm1_grad_norm(int count, const void* const* in, const long* rows, const long* cols, const long* ld,
                  const unsigned char* f32, int norm_type, float* norm, void* workspace, size_t workspace_bytes,
                  void* stream) {
  if (!norm) return MM1_E_NULL;
  if (norm_type != MM1_NORM_2 && norm_type != MM1_NORM_MAX) return MM1_E_SHAPE;
  const mm1::ClipArgs a{count, in,  nullptr, rows, cols, ld,      nullptr, f32, norm_type == MM1_NORM_MAX,
                        0.f,   0.f, norm,    workspace, false};
  const int rc = check_clip(a, false);
  if (rc) return rc;
  if (!workspace || workspace_bytes < mm1::clip_workspace_bytes(count)) return MM1_E_WORKSPACE;
  if (!aligned(workspace, 16) || !aligned(norm, 4)) return MM1_E_ALIGN;
  return from_hip(mm1::launch_clip(a, static_cast<hipStream_t>(stream)));
}

int mm1_grad_clip(int count, const void* const* in, void* const* out, const long* rows, const long* cols,
                  const long* ld, const long* ld_out, const unsigned char* f32, int norm_type, float max_norm,
                  float eps, int norm_known, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (!norm) return MM1_E_NULL;
  if ((norm_type != MM1_NORM_2 && norm_type != MM1_NORM_MAX) || !(max_norm >= 0.f) || !(eps >= 0.f) || isinf(eps))
    return MM1_E_SHAPE;
  const bool in_place = out == nullptr;
  const mm1::ClipArgs a{count,    in,  in_place ? const_cast<void* const*>(in) : out, rows, cols, ld,
                        in_place ? ld : ld_out, f32, norm_type == MM1_NORM_MAX, max_norm, eps, norm, workspace,
                        norm_known != 0};
  const int rc = check_clip(a, true);
  if (rc) return rc;
  if (!workspace || workspace_bytes < mm1::clip_workspace_bytes(count)) return MM1_E_WORKSPACE;
  if (!aligned(workspace, 16) || !aligned(norm, 4)) return MM1_E_ALIGN;
  return from_hip(mm1::launch_clip(a, static_cast<hipStream_t>(stream)));
}

static bool layouts_ok(int x_layout, int w_layout) {
  return (x_layout == MM1_GEMM_ROW && (w_layout == MM1_GEMM_ROW || w_layout == MM1_GEMM_COL)) ||
         (x_layout == MM1_GEMM_COL && w_layout == MM1_GEMM_COL);
}

size_t mm1_linear_workspace_size(int M, int N, int K, int x_layout, int w_layout, int act) {
  if (!linear_sizes_ok(M, N, K) || !layouts_ok(x_layout, w_layout)) return 0;
  return mm1::linear_workspace_bytes(M, N, K, x_layout, w_layout, act != MM1_ACT_NONE);
}

int mm1_linear(const void* x, int x_layout, long ldx, const void* w, int w_layout, long ldw, const void* bias,
               int bias_f32, int act, const void* residual, int residual_f32, long ldr, void* pre, long ldp,
               void* out, int out_f32, long ldo, void* workspace, size_t workspace_bytes, int M, int N, int K,
               void* stream) {
  if (!x || !w || !out) return MM1_E_NULL;
  const bool xc = x_layout == MM1_GEMM_COL;
  if (!layouts_ok(x_layout, w_layout)) return MM1_E_SHAPE;
  if (act < MM1_ACT_NONE || act > MM1_ACT_SILU || (xc && (act != MM1_ACT_NONE || pre))) return MM1_E_SHAPE;
  if (!linear_sizes_ok(M, N, K) || !operand_ok(x_layout, ldx, M, K) || !operand_ok(w_layout, ldw, N, K))
    return MM1_E_SHAPE;
  if (!epilogue_ld_ok(ldo, out_f32, M, N) || (residual && !epilogue_ld_ok(ldr, residual_f32, M, N)) ||
      (pre && !epilogue_ld_ok(ldp, false, M, N)))
    return MM1_E_SHAPE;
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(workspace, 16) || !element_aligned(out, out_f32) ||
      !element_aligned(bias, bias_f32) || !element_aligned(residual, residual_f32) || !aligned(pre, 2))
    return MM1_E_ALIGN;
  const size_t need = mm1::linear_workspace_bytes(M, N, K, x_layout, w_layout, act != MM1_ACT_NONE);
  if (need > 0 && (!workspace || workspace_bytes < need)) return MM1_E_WORKSPACE;
  // without an activation z is the output before the residual: nothing keeps it
  if (act == MM1_ACT_NONE && pre) return MM1_E_SHAPE;
  return from_hip(mm1::launch_linear({x, x_layout, ldx, w, w_layout, ldw, bias, bias_f32 != 0, act, residual,
                                      residual_f32 != 0, ldr, pre, ldp, out, out_f32 != 0, ldo, workspace, M, N, K},
                                     static_cast<hipStream_t>(stream)));
}

static bool backward_sizes_ok(int M, int N, int K) {
  return linear_sizes_ok(M, N, K) && linear_sizes_ok(M, K, N) && linear_sizes_ok(N, K, M) && N <= (1 << 24) &&
         K <= (1 << 24);
}

size_t mm1_linear_backward_workspace_size(int M, int N, int K, int dz, int dx, int dw, int dbias) {
  return backward_sizes_ok(M, N, K) ? backward_scratch(M, N, K, dz, dx, dw, dbias).bytes : 0;
}

int mm1_linear_backward(const void* dy, int dy_f32, long ldy, const void* pre, long ldp, int act, const void* x,
                        long ldx, const void* w, int w_layout, long ldw, void* dx, int dx_f32, void* dw, int dw_f32,
                        void* dbias, int dbias_f32, void* workspace, size_t workspace_bytes, int M, int N, int K,
                        void* stream) {
  if (act < MM1_ACT_NONE || act > MM1_ACT_SILU || !backward_sizes_ok(M, N, K)) return MM1_E_SHAPE;
  const bool has_act = act != MM1_ACT_NONE, wc = w_layout == MM1_GEMM_COL;
  if (!dy || (has_act && !pre) || (!dx && !dw && !dbias) || (dx && !w) || (dw && !x)) return MM1_E_NULL;
  if (w_layout != MM1_GEMM_ROW && !wc) return MM1_E_SHAPE;
  if (ldy < N || ldy > kMaxLd || (has_act && (ldp < N || ldp > kMaxLd))) return MM1_E_SHAPE;
  const int x_as = MM1_GEMM_COL, w_as = wc ? MM1_GEMM_ROW : MM1_GEMM_COL;    // as dW's and dX's products read them
  if ((dx && (ldw < (wc ? ceil8(N) : ceil8(K)) || !operand_ok(w_as, ldw, K, N))) ||
      (dw && (ldx < ceil8(K) || !operand_ok(x_as, ldx, K, M))))
    return MM1_E_SHAPE;
  if ((dx && !epilogue_ld_ok(K, dx_f32, M, K)) ||
      (dw && !(wc ? epilogue_ld_ok(N, dw_f32, K, N) : epilogue_ld_ok(K, dw_f32, N, K))))
    return MM1_E_SHAPE;
  if (!element_aligned(dy, dy_f32) || !aligned(pre, 2) || !aligned(x, 16) || !aligned(w, 16) ||
      !element_aligned(dx, dx_f32) || !element_aligned(dw, dw_f32) || !element_aligned(dbias, dbias_f32) ||
      !aligned(workspace, 16))
    return MM1_E_ALIGN;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  // dz is dy where the products take it as it lies
  const bool products = dx || dw;
  const bool ready = !has_act && !dy_f32 && N % 8 == 0 && ldy % 8 == 0 && aligned(dy, 16) &&
                     operand_ok(MM1_GEMM_ROW, ldy, M, N) && operand_ok(MM1_GEMM_COL, ldy, N, M);
  const BackwardScratch scratch = backward_scratch(M, N, K, !ready, dx, dw, dbias);
  if (scratch.bytes > 0 && (!workspace || workspace_bytes < scratch.bytes)) return MM1_E_WORKSPACE;
  char* part = static_cast<char*>(workspace) + scratch.dz;
  const void* dz = ready ? dy : workspace;
  const long ldz = ready ? ldy : ceil8(N);
  if (products && !ready && (!operand_ok(MM1_GEMM_ROW, ldz, M, N) || !operand_ok(MM1_GEMM_COL, ldz, N, M)))
    return MM1_E_SHAPE;
  if (dbias || (products && !ready)) {
    const hipError_t e = mm1::launch_linear_grad({dy, dy_f32 != 0, ldy, pre, ldp, act,
                                                  products && !ready ? workspace : nullptr, ldz, dbias, dbias_f32 != 0,
                                                  part, M, N},
                                                 s);
    if (e != hipSuccess) return from_hip(e);
  }
  auto product = [&](const void* a, int la, long lda, const void* b, int lb, long ldb, void* out, int f32, int m, int n,
                     int k) {
    return mm1::launch_linear({a, la, lda, b, lb, ldb, nullptr, false, MM1_ACT_NONE, nullptr, false, 0, nullptr, 0, out,
                               f32 != 0, n, part, m, n, k},
                              s);
  };
  if (dx) {
    const hipError_t e = product(dz, MM1_GEMM_ROW, ldz, w, w_as, ldw, dx, dx_f32, M, K, N);
    if (e != hipSuccess) return from_hip(e);
  }
  if (dw) {
    const hipError_t e = wc ? product(x, x_as, ldx, dz, MM1_GEMM_COL, ldz, dw, dw_f32, K, N, M)
                            : product(dz, MM1_GEMM_COL, ldz, x, x_as, ldx, dw, dw_f32, N, K, M);
    if (e != hipSuccess) return from_hip(e);
  }
  return MM1_OK;
}

int mm1_pack_bf16(const void* src, int src_f32, long ld, int rows, int cols, void* dst, long ldd, int rows_out,
                  void* stream) {
  if (!src || !dst) return MM1_E_NULL;
  if (rows < 1 || cols < 1 || rows_out < rows || rows_out > (1 << 29) || ld < cols || ld > kMaxLd || ldd < cols ||
      ldd % 8 != 0 || ldd > (1 << 29))
    return MM1_E_SHAPE;
  if (!element_aligned(src, src_f32) || !aligned(dst, 16)) return MM1_E_ALIGN;
  return from_hip(mm1::launch_pack_bf16(src, src_f32 != 0, ld, rows, cols, dst, ldd, rows_out,
                                        static_cast<hipStream_t>(stream)));
}

}  // extern "C"
