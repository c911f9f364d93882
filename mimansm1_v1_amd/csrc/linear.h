// Host interface of the products with an epilogue (linear.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

namespace mm1 {

// Rows of a wave's block at most, whose byte offsets the epilogue forms in 32 bits.
constexpr int EPILOGUE_ROWS = 128;

struct LinearArgs {
  const void* x;
  int x_layout;            // MM1_GEMM_ROW / _COL
  long ldx;
  const void* w;
  int w_layout;
  long ldw;
  const void* bias;        // or nullptr
  bool bias_f32;
  int act;
  const void* residual;    // or nullptr
  bool residual_f32;
  long ldr;
  void* pre;               // bf16 z before the activation, or nullptr
  long ldp;
  void* out;
  bool out_f32;
  long ldo;
  void* workspace;
  int M, N, K;
};

struct LinearGradArgs {
  const void* dy;
  bool dy_f32;
  long ldy;
  const void* pre;
  long ldp;
  int act;
  void* dz;                // bf16 [M, ldz], zeros from column N on; or nullptr
  long ldz;
  void* dbias;             // or nullptr
  bool dbias_f32;
  void* workspace;
  int M, N;
};

size_t linear_workspace_bytes(int M, int N, int K, int x_layout, int w_layout, bool act);
hipError_t launch_linear(const LinearArgs& a, hipStream_t stream);
size_t linear_grad_workspace_bytes(int M, int N);
hipError_t launch_linear_grad(const LinearGradArgs& a, hipStream_t stream);
hipError_t launch_pack_bf16(const void* src, bool src_f32, long ld, int rows, int cols, void* dst, long ldd,
                            int rows_out, hipStream_t stream);

}  // namespace mm1
