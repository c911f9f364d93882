// Products with bias, activation and residual in their epilogue, and the
// elementwise part of their gradients, for gfx950.
//
//   z = X W^T + bias (fp32 sums),  out = act(z) + residual, rounded once
//   dz = dy act'(z),  dbias = column sums of dz   (dX and dW are plain products)
//
// The products run on the GEMM core (gemm_core.h; tiles and splits as
// gemm_plan.h chooses them) with any K: what lies past it reads as zeros.  The
// accumulators go through LDS in fp32, after which a lane holds eight
// neighbouring values of a row: bias, activation and residual meet them there,
// at any element alignment and for any width.  With K split, the kernel that
// adds the partial sums applies the epilogue.
//
// Roundings to fewer bits than the sums': x and w are bf16, the matrix cores' fast type
// (an fp32 one as two bf16 terms would double its products).  z is kept for the
// slope in bf16, half the bytes of a tensor that lives until the backward, and dz
// enters dX's and dW's products in bf16 like every operand, also where dY and W are
// fp32: the arithmetic of bf16 autocast.  Gradients are 2.3e-3 to 2.4e-3 from the exact
// ones, where rounding the bf16 results alone leaves 1.7e-3.
//
// 16384 x 1280 x 3328 with an fp32 residual and output: 148-158 us (880-940 TFLOP/s; the
// 168 MB of the stream come behind the one round of tiles); 4096 x 3328 x 1280 with
// bias, gelu and z kept 51-57; 8192 x 1280 x 1280 with a bf16 residual 41-44.
#include <hip/hip_runtime.h>

#include <atomic>

#include "gemm.h"
#include "gemm_core.h"
#include "gemm_mid.h"
#include "gemm_plan.h"
#include "linear.h"
#include "rows.h"

namespace mm1 {

namespace {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4_any __attribute__((ext_vector_type(4), aligned(2)));

enum Act { NONE, RELU, GELU, GELU_TANH, SILU };

__device__ __forceinline__ float recip(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * 1.44269504f); }

// The normal distribution's upper tail Q(a) for a >= 0 and its density
// exp(-a^2 / 2) (times sqrt(2 pi)): Q = density * t P(t), t = 1 / (1 + 0.265 a), P the
// polynomial of least relative error over a in [0, 13.5] (6.3e-7; fitted to
// erfcx by weighted least squares), beyond which Q is below 2^-126.  The density is 0
// from 15 on, so that arguments clamped to 16 give Q = 0.
__device__ __forceinline__ float upper_tail(float a, float& density) {
  const float t = recip(fmaf(0.265f, a, 1.f));
  float p = -0.0677873029f;
  p = fmaf(p, t, 0.195274021f);
  p = fmaf(p, t, -0.0663641497f);
  p = fmaf(p, t, 0.142494137f);
  p = fmaf(p, t, 0.082946336f);
  p = fmaf(p, t, 0.107836813f);
  p = fmaf(p, t, 0.105599834f);
  density = exp_fast(-0.5f * a * a);
  return density * t * p;
}

constexpr float TANH_C = 0.7978845608f, TANH_A = 0.044715f;      // sqrt(2 / pi)

// sigmoid(x) without overflow: exp of a huge argument is infinite, its reciprocal 0.
__device__ __forceinline__ float sigmoid(float x) { return recip(1.f + exp_fast(-x)); }

template <int ACT>
__device__ __forceinline__ float act1(float z) {
  if constexpr (ACT == RELU) return z < 0.f ? 0.f : z;               // a NaN stays one
  if constexpr (ACT == SILU) return z < -80.f ? 0.f : z * sigmoid(z);      // not -inf * 0
  if constexpr (ACT == GELU_TANH) {
    const float u = 2.f * TANH_C * fmaf(TANH_A * z * z, z, z);
    return u < -80.f ? 0.f : z * sigmoid(u);
  }
  if constexpr (ACT == GELU) {
    const float a = fminf(fabsf(z), 16.f);
    float d;
    return (z < 0.f ? 0.f : z) - a * upper_tail(a, d);       // max(z, 0) - |z| Q(|z|)
  }
  return z;
}

template <int ACT>
__device__ __forceinline__ float slope1(float z) {
  if constexpr (ACT == RELU) return z <= 0.f ? 0.f : 1.f;             // a NaN hands dY on
  if constexpr (ACT == SILU) {
    const float s = sigmoid(z);
    return fabsf(z) > 80.f ? (z > 0.f ? 1.f : 0.f) : s * fmaf(z, 1.f - s, 1.f);
  }
  if constexpr (ACT == GELU_TANH) {
    const float u = 2.f * TANH_C * fmaf(TANH_A * z * z, z, z), s = sigmoid(u);
    const float du = 2.f * TANH_C * fmaf(3.f * TANH_A * z, z, 1.f);
    return fabsf(u) > 80.f ? (z > 0.f ? 1.f : 0.f) : s * fmaf(z * du, 1.f - s, 1.f);
  }
  if constexpr (ACT == GELU) {
    const float a = fminf(fabsf(z), 16.f);
    float d;
    const float q = upper_tail(a, d), t = fmaf(a, -0.3989422804f * d, q);      // Q(a) - a density(a)
    return z < 0.f ? t : z != z ? z : 1.f - t;
  }
  return 1.f;
}

template <int ACT, int N>
__device__ __forceinline__ void apply(float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = act1<ACT>(v[j]);
}
template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {       // act is uniform
  switch (act) {
    case RELU: apply<RELU>(v); break;
    case GELU: apply<GELU>(v); break;
    case GELU_TANH: apply<GELU_TANH>(v); break;
    case SILU: apply<SILU>(v); break;
    default: break;
  }
}

struct Epilogue {
  const void *bias, *residual;
  void* out;
  __bf16* pre;
  long ldr, ldp, ldo;      // offsets in the EPILOGUE_ROWS of a wave's block stay in 32 bits
  int M, N, act;
  bool bias_f32, residual_f32, out_f32;
};

// Eight neighbouring values as they lie in memory (bf16 in `a` alone).
struct Raw {
  u32x4 a, b;
};
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 __attribute__((aligned(2))) u32x2_any;

__device__ __forceinline__ Raw load_raw(const char* p, bool f32) {
  Raw r;
  r.a = *reinterpret_cast<const u32x4_any*>(p);
  if (f32) r.b = *reinterpret_cast<const u32x4_any*>(p + 16);
  return r;
}
__device__ __forceinline__ void unpack(const Raw& r, bool f32, float (&v)[8]) {
  if (f32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = __uint_as_float(r.a[j]);
      v[4 + j] = __uint_as_float(r.b[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(r.a[j] << 16);
      v[2 * j + 1] = __uint_as_float(r.a[j] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void store8(char* p, bool f32, const float (&v)[8]) {
  if (f32) rows::store8(reinterpret_cast<float*>(p), v);
  else rows::store8(reinterpret_cast<__bf16*>(p), v);
}
__device__ __forceinline__ float load1(const void* base, long at, bool f32) {
  return f32 ? static_cast<const float*>(base)[at] : (float)static_cast<const __bf16*>(base)[at];
}
// The first n of eight values (n > 0; eight where it is more).
__device__ __forceinline__ void load_edge(const char* p, bool f32, int n, float (&v)[8]) {
  if (f32) {
    const auto r = rows::load_any(reinterpret_cast<const float*>(p), n);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r[j];
  } else {
    const auto r = rows::load_any(reinterpret_cast<const __bf16*>(p), n);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r[j];
  }
}
__device__ __forceinline__ void store_edge(char* p, bool f32, int n, const float (&v)[8]) {
  if (f32) rows::store_any(reinterpret_cast<float*>(p), n, v);
  else rows::store_any(reinterpret_cast<__bf16*>(p), n, v);
}
__device__ __forceinline__ char* block_at(const void* base, bool f32, long row, long ld, int col) {
  return base ? const_cast<char*>(static_cast<const char*>(base)) + (row * ld + col) * (f32 ? 4 : 2) : nullptr;
}

// A wave's 32 TI rows x 32 TJ columns from val(i, b, q), the f32x4 of columns
// 32b + 8q + 4(lane/32) .. +3 of row 32i + (lane & 31), through STAGE bytes of
// LDS that the wave owns: NB column blocks (two where TJ is even) of as many rows
// as fit at a time, after which a lane holds eight neighbouring columns and
// 4 NB lanes a row.  16-byte chunk c of LDS row r lies at c ^ swizzle(r), which
// keeps the writes and the reads off each other's banks.
template <bool ACT, int STAGE, int TI, int TJ, class Val>
__device__ __forceinline__ void finish(const Epilogue& e, char* lds, int lane, long row0, int col0, Val&& val) {
  constexpr int NB = TJ % 2 == 0 ? 2 : 1, PITCH = 128 * NB;
  constexpr int ROWS = STAGE / PITCH < 32 ? STAGE / PITCH : 32;      // of an exchange
  constexpr int LROWS = 16 / NB, STEPS = ROWS / LROWS;               // rows of an instruction
  static_assert(STEPS * LROWS == ROWS && 32 % ROWS == 0, "whole instructions");
  static_assert(!ACT || TI * TJ <= 8, "an activation takes the smaller tiles");
  static_assert(32 * TI <= EPILOGUE_ROWS, "32-bit offsets");
  __asm__ volatile("" : "+v"(lane));       // made anew here: no address of the epilogue lives through the products
  const int l32 = lane & 31, h = lane >> 5, c8 = lane % (4 * NB), lr = lane / (4 * NB);
  auto swizzle = [](int row) { return NB == 2 ? row & 7 : (row >> 1) & 7; };
  // An fp32 output without an activation: four columns of two rows a lane instead, so that an
  // instruction reads and writes whole lines (16384 x 1280 x 3328 on an fp32 stream 160 us with
  // eight columns, 148 so; 8192 rows 83, 77; but the 192-column tiles 29.7, 31.2 with 4096 x 1280 x 1280).
  const bool quads = !ACT && (NB == 2 || ROWS < 32) && e.out_f32;
  const int c4 = lane % (8 * NB), qr = lane / (8 * NB);
  constexpr int QROWS = 8 / NB;
#pragma unroll
  for (int b0 = 0; b0 < TJ; b0 += NB) {
    const int colb = col0 + 32 * b0;
    if (colb >= e.N || row0 >= e.M) return;                          // uniform
    const bool inside = row0 + 32 * TI <= e.M && colb + 32 * NB <= e.N;
    const char* res = block_at(e.residual, e.residual_f32, row0, e.ldr, colb);
    char* out = block_at(e.out, e.out_f32, row0, e.ldo, colb);
    char* pre = block_at(e.pre, false, row0, e.ldp, colb);
    auto at = [&](int row, long ld, bool f32) { return ((uint32_t)row * (uint32_t)ld + 8u * c8) << (f32 ? 2 : 1); };
    auto at4 = [&](int row, long ld, bool f32) { return ((uint32_t)row * (uint32_t)ld + 4u * c4) << (f32 ? 2 : 1); };
    float bias[8] = {};
    if (inside && e.bias && quads) {
      if (e.bias_f32) {
        const f32x4 b = *reinterpret_cast<const f32x4_any*>(static_cast<const float*>(e.bias) + colb + 4 * c4);
#pragma unroll
        for (int j = 0; j < 4; ++j) bias[j] = b[j];
      } else {
        const bf16x4 b = *reinterpret_cast<const bf16x4_any*>(static_cast<const __bf16*>(e.bias) + colb + 4 * c4);
#pragma unroll
        for (int j = 0; j < 4; ++j) bias[j] = (float)b[j];
      }
    } else if (inside && e.bias)
      unpack(load_raw(block_at(e.bias, e.bias_f32, 0, 0, colb + 8 * c8), e.bias_f32), e.bias_f32, bias);
#pragma unroll
    for (int x0 = 0; x0 < 32 * TI; x0 += ROWS) {
      const int i = x0 / 32, r0 = x0 % 32;
      __builtin_amdgcn_sched_barrier(0);       // an exchange at a time: the accumulators leave few registers
      Raw r[STEPS];
      if (!ACT && inside && res && quads) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const char* p = res + at4(x0 + LROWS * k + QROWS * s + qr, e.ldr, e.residual_f32);
            u32x4& d = s ? r[k].b : r[k].a;
            if (e.residual_f32) {
              d = *reinterpret_cast<const u32x4_any*>(p);
            } else {
              const u32x2 h = *reinterpret_cast<const u32x2_any*>(p);
              d[0] = h[0];
              d[1] = h[1];
            }
          }
        }
      } else if (!ACT && inside && res) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
          r[k] = load_raw(res + at(x0 + LROWS * k + lr, e.ldr, e.residual_f32), e.residual_f32);
      }
      const int wr = l32 - r0;
      if (ROWS == 32 || (wr >= 0 && wr < ROWS)) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(lds + wr * PITCH + (((8 * b + 2 * q + h) ^ swizzle(wr)) << 4)) = val(i, b0 + b, q);
        }
      }
      wave_sync();
      if (inside && quads) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int wrow = LROWS * k + QROWS * s + qr;
            f32x4 v = *reinterpret_cast<const f32x4*>(lds + wrow * PITCH + ((c4 ^ swizzle(wrow)) << 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += bias[j];
            if (res) {
              const u32x4& d = s ? r[k].b : r[k].a;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                v[j] += __uint_as_float(e.residual_f32 ? d[j] : j & 1 ? d[j >> 1] & 0xffff0000u : d[j >> 1] << 16);
            }
            *reinterpret_cast<f32x4_any*>(out + at4(x0 + wrow, e.ldo, true)) = v;
          }
        }
      } else if (inside) {
#pragma unroll(ACT ? 1 : STEPS)
        for (int k = 0; k < STEPS; ++k) {
          const int wrow = LROWS * k + lr, row = x0 + wrow;
          float v[8];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(lds + wrow * PITCH + (((2 * c8 + s) ^ swizzle(wrow)) << 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * s + j] = x[j] + bias[4 * s + j];
          }
          Raw add;
          if constexpr (ACT) {
            if (res) add = load_raw(res + at(row, e.ldr, e.residual_f32), e.residual_f32);
            if (pre) store8(pre + at(row, e.ldp, false), false, v);
            activate(e.act, v);
          } else {
            add = r[k];
          }
          if (res) {
            float a[8];
            unpack(add, e.residual_f32, a);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += a[j];
          }
          store8(out + at(row, e.ldo, e.out_f32), e.out_f32, v);
        }
      } else if constexpr (TI * TJ > 8) {
        // across the edge, value by value: the 320-column tiles have no registers for more
        // (pieces with their parts spilled 80, at 12 us on 16384 x 1280 x 3328)
#pragma unroll 1
        for (int k = lane; k < ROWS * 32 * NB; k += 64) {
          const int wrow = k / (32 * NB), col = k % (32 * NB);
          const long row = x0 + wrow;
          if (row0 + row >= e.M || colb + col >= e.N) continue;
          float v[1] = {*reinterpret_cast<const float*>(lds + wrow * PITCH + (((col >> 2) ^ swizzle(wrow)) << 4) +
                                                        4 * (col & 3))};
          if (e.bias) v[0] += load1(e.bias, colb + col, e.bias_f32);
          if (res) v[0] += load1(res, row * e.ldr + col, e.residual_f32);
          if (e.out_f32) reinterpret_cast<float*>(out)[row * e.ldo + col] = v[0];
          else reinterpret_cast<__bf16*>(out)[row * e.ldo + col] = (__bf16)v[0];
        }
      } else {
        // the same with what lies past the edge left out
        const int n = e.N - colb - 8 * c8;                             // columns from the lane's first on
#pragma unroll 1
        for (int k = 0; k < STEPS; ++k) {
          const int wrow = LROWS * k + lr, row = x0 + wrow;
          if (row0 + row >= e.M || n <= 0) continue;
          float v[8], a[8];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(lds + wrow * PITCH + (((2 * c8 + s) ^ swizzle(wrow)) << 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * s + j] = x[j];
          }
          if (e.bias) {
            load_edge(block_at(e.bias, e.bias_f32, 0, 0, colb + 8 * c8), e.bias_f32, n, a);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += a[j];
          }
          if constexpr (ACT) {
            if (pre) store_edge(pre + at(row, e.ldp, false), false, n, v);
            activate(e.act, v);
          }
          if (res) {
            load_edge(res + at(row, e.ldr, e.residual_f32), e.residual_f32, n, a);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += a[j];
          }
          store_edge(out + at(row, e.ldo, e.out_f32), e.out_f32, n, v);
        }
      }
      wave_sync();
    }
  }
}

// Every tile cut along k into PARTS runs of window pairs, a run for each 8 / PARTS
// XCDs, whose workgroups so walk the same k together and share what they read in
// their L2: a window takes 1.5 us, where SplitTiles' workgroups, each at a k of its
// own, take up to 2.5 (3328 x 1280 x 16384 176 us with SplitTiles, 148 so; 8192 x 1280 x
// 16384 419, 303).  Partial sums of part k of tile t go to slot t * PARTS + k.
template <int PARTS>
struct PartTiles {
  int t0, n_wg, k0, nk, n, j;
  __device__ __forceinline__ PartTiles(int total, int n_kt) {
    constexpr int SHARE = 8 / PARTS;                 // XCDs of a part
    const int xcd = blockIdx.x & 7, part = xcd / SHARE, r = xcd % SHARE;
    n_wg = gridDim.x >> 3;
    j = (int)(blockIdx.x >> 3);
    const int pairs = n_kt / 2;
    k0 = 2 * (int)((long)pairs * part / PARTS);
    nk = 2 * (int)((long)pairs * (part + 1) / PARTS) - k0;
    t0 = (int)((long)total * r / SHARE);
    const int t1 = (int)((long)total * (r + 1) / SHARE);
    n = t0 + j < t1 ? (t1 - t0 - j + n_wg - 1) / n_wg : 0;
  }
  __device__ __forceinline__ int windows() const { return n * nk; }
  __device__ __forceinline__ gemm::Item at(int i) const {
    const int t = t0 + j + i * n_wg;
    return {t, -1, k0, nk, t * PARTS + (int)(blockIdx.x & 7) / (8 / PARTS)};
  }
};

template <class Tiles>
constexpr bool only_parts = false;
template <int PARTS>
constexpr bool only_parts<PartTiles<PARTS>> = true;

template <gemm::Layout LX, gemm::Layout LW, class S, bool ACT, class Tiles, bool RAGGED>
__global__ __launch_bounds__(512, 1) void linear_kernel(const gemm::Problem p, const Epilogue e, float* part) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = w % S::WM, wn = w / S::WM;
  gemm::run<LX, LW, false, S, Tiles, RAGGED>(p, smem, [](int, int) MM1_INLINE {},
                                     [&](int mb, int nb, f32x16 (&acc)[S::TJ][S::TI], int slot) MM1_INLINE {
    if (only_parts<Tiles> || slot >= 0) {
#pragma unroll
      for (int b = 0; b < S::TJ; ++b) {
#pragma unroll
        for (int i = 0; i < S::TI; ++i) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(part + part_index<S>(slot, w, b, i, q, lane)) = quad(acc[b][i], q);
        }
      }
      return;
    }
    finish<ACT, S::STAGE_BYTES, S::TI, S::TJ>(e, smem + S::RING + S::STAGE_BYTES * w, lane,
                                              (long)mb * gemm::BM + 32 * S::TI * wm, nb * S::BN + 32 * S::TJ * wn,
                                              [&](int i, int b, int q) { return quad(acc[b][i], q); });
  });
}

// Leftover tile blockIdx.x / 8, wave blockIdx.x % 8 of it, row block = wave of
// this workgroup: the sum of its partial tiles in workgroup order, then the
// epilogue.
template <class S, bool ACT>
__global__ __launch_bounds__(64 * S::TI) void linear_sum_kernel(const float* __restrict__ part, const Epilogue e,
                                                                int n_mblk, int n_nblk, int left0, int left, int upt,
                                                                int n_g) {
  __shared__ __attribute__((aligned(16))) char smem[S::TI * S::STAGE_BYTES];
  const int lane = threadIdx.x & 63, i = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = blockIdx.x >> 3, w = blockIdx.x & 7;
  const int wm = w % S::WM, wn = w / S::WM;
  auto unit = [&](int g) { return gemm::SplitTiles::unit(g, left, upt, n_g); };
  int g = (int)((long)l * n_g / left);
  while (g > 0 && unit(g) > (long)l * upt) --g;
  while (unit(g + 1) <= (long)l * upt) ++g;
  f32x4 sum[S::TJ][4] = {};
  for (; g < n_g && unit(g) < (long)(l + 1) * upt; ++g) {
    if (unit(g + 1) == unit(g)) continue;   // an empty run wrote nothing
#pragma unroll
    for (int b = 0; b < S::TJ; ++b) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        sum[b][q] += *reinterpret_cast<const f32x4*>(part + part_index<S>(g + l, w, b, i, q, lane));
    }
  }
  int mb, nb;
  gemm::tile_coords(left0 + l, n_mblk, n_nblk, mb, nb);
  finish<ACT, S::STAGE_BYTES, 1, S::TJ>(e, smem + S::STAGE_BYTES * i, lane, (long)mb * gemm::BM + 32 * (S::TI * wm + i),
                          nb * S::BN + 32 * S::TJ * wn, [&](int, int b, int q) { return sum[b][q]; });
}

// The same for PartTiles: tile blockIdx.x / 8, its parts in order.
template <class S>
__global__ __launch_bounds__(64 * S::TI) void linear_part_sum_kernel(const float* __restrict__ part, const Epilogue e,
                                                                     int n_mblk, int n_nblk, int parts) {
  __shared__ __attribute__((aligned(16))) char smem[S::TI * S::STAGE_BYTES];
  const int lane = threadIdx.x & 63, i = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x >> 3, w = blockIdx.x & 7, wm = w % S::WM, wn = w / S::WM;
  f32x4 sum[S::TJ][4] = {};
  for (int g = 0; g < parts; ++g) {
#pragma unroll
    for (int b = 0; b < S::TJ; ++b) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        sum[b][q] += *reinterpret_cast<const f32x4*>(part + part_index<S>(t * parts + g, w, b, i, q, lane));
    }
  }
  int mb, nb;
  gemm::tile_coords(t, n_mblk, n_nblk, mb, nb);
  finish<false, S::STAGE_BYTES, 1, S::TJ>(e, smem + S::STAGE_BYTES * i, lane, (long)mb * gemm::BM + 32 * (S::TI * wm + i),
                          nb * S::BN + 32 * S::TJ * wn, [&](int, int b, int q) { return sum[b][q]; });
}

// Small tiles, split along k as in gemm.hip's small kernel.
template <gemm::Layout LX, gemm::Layout LW, bool ACT>
__global__ __launch_bounds__(256) void linear_small_kernel(const gemm::Problem p, const Epilogue e, float* part,
                                                           int splits) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tiles = p.n_mblk * p.n_nblk, total = tiles * splits, per = (total + 7) / 8;
  const int j = (int)(blockIdx.x >> 3), item = (int)(blockIdx.x & 7) * per + j;
  if (j >= per || item >= total) return;
  const int split = item / tiles, t = item - split * tiles;
  const int nb = t / p.n_mblk, mb = t - nb * p.n_mblk;
  const int n_win = (p.K + gemm::BK - 1) / gemm::BK;
  const int w0 = (int)((long)split * n_win / splits), w1 = (int)((long)(split + 1) * n_win / splits);
  f32x16 acc[1];
  gemm::run_small<LX, LW, false, true>(p, smem, mb, nb, w0, w1 - w0, acc);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (splits > 1) {
    float* dst = part + ((((long)t * splits + split) * 4 + w) * 4 * 64 + lane) * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<f32x4*>(dst + q * 256) = quad(acc[0], q);
    return;
  }
  finish<ACT, 2048, 1, 1>(e, smem + 2048 * w, lane, (long)mb * gemm::SMALL + 32 * (w & 1),
                      nb * gemm::SMALL + 32 * (w >> 1), [&](int, int, int q) { return quad(acc[0], q); });
}

template <bool ACT>
__global__ __launch_bounds__(256) void linear_small_sum_kernel(const float* __restrict__ part, const Epilogue e,
                                                               int n_mblk, int splits) {
  __shared__ __attribute__((aligned(16))) char smem[4 * 2048];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x, nb = t / n_mblk, mb = t - nb * n_mblk;
  f32x4 sum[4] = {};
  for (int s = 0; s < splits; ++s) {
    const float* src = part + ((((long)t * splits + s) * 4 + w) * 4 * 64 + lane) * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) sum[q] += *reinterpret_cast<const f32x4*>(src + q * 256);
  }
  finish<ACT, 2048, 1, 1>(e, smem + 2048 * w, lane, (long)mb * gemm::SMALL + 32 * (w & 1),
                      nb * gemm::SMALL + 32 * (w >> 1), [&](int, int, int q) { return sum[q]; });
}

// Partial tile of the mid tiles: [wave][column block][row block][q][lane] x 4 floats.
template <class S>
__device__ __forceinline__ long mid_part(long tile, int w, int b, int i, int q, int lane) {
  return (((((tile * 4 + w) * S::TJ + b) * S::TI + i) * 4 + q) * 64 + lane) * 4;
}

// Mid tiles (gemm_mid.h), split along k like the small ones.
template <gemm::Layout LX, gemm::Layout LW, class S, bool ACT>
__global__ __launch_bounds__(256) void linear_mid_kernel(const gemm::Problem p, const Epilogue e, float* part,
                                                         int splits) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tiles = p.n_mblk * p.n_nblk, total = tiles * splits, per = (total + 7) / 8;
  const int j = (int)(blockIdx.x >> 3), item = (int)(blockIdx.x & 7) * per + j;
  if (j >= per || item >= total) return;
  const int split = item / tiles, t = item - split * tiles;
  int mb, nb;
  gemm::tile_coords(t, p.n_mblk, p.n_nblk, mb, nb);
  const int n_win = (p.K + gemm::BK - 1) / gemm::BK;
  const int w0 = (int)((long)split * n_win / splits), w1 = (int)((long)(split + 1) * n_win / splits);
  f32x16 acc[S::TJ][S::TI];
  gemm::run_mid<LX, LW, S>(p, smem, mb, nb, w0, w1 - w0, acc);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (splits > 1) {
#pragma unroll
    for (int b = 0; b < S::TJ; ++b) {
#pragma unroll
      for (int i = 0; i < S::TI; ++i) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(part + mid_part<S>((long)t * splits + split, w, b, i, q, lane)) = quad(acc[b][i], q);
      }
    }
    return;
  }
  finish<ACT, 8192, S::TI, S::TJ>(e, smem + 8192 * w, lane, (long)mb * S::ROWS + 64 * (w & 1),
                                  nb * S::COLS + 32 * S::TJ * (w >> 1),
                                  [&](int i, int b, int q) { return quad(acc[b][i], q); });
}

// Tile blockIdx.x / 4, wave blockIdx.x % 4 of it, row block = wave of this
// workgroup: the splits' sum in their order, then the epilogue.
template <class S, bool ACT>
__global__ __launch_bounds__(128) void linear_mid_sum_kernel(const float* __restrict__ part, const Epilogue e,
                                                             int n_mblk, int n_nblk, int splits) {
  __shared__ __attribute__((aligned(1024))) char smem[S::TI * 8192];
  const int lane = threadIdx.x & 63, i = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x >> 2, w = blockIdx.x & 3;
  f32x4 sum[S::TJ][4] = {};
  for (int s = 0; s < splits; ++s) {
#pragma unroll
    for (int b = 0; b < S::TJ; ++b) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        sum[b][q] += *reinterpret_cast<const f32x4*>(part + mid_part<S>((long)t * splits + s, w, b, i, q, lane));
    }
  }
  int mb, nb;
  gemm::tile_coords(t, n_mblk, n_nblk, mb, nb);
  finish<ACT, 8192, 1, S::TJ>(e, smem + 8192 * i, lane, (long)mb * S::ROWS + 64 * (w & 1) + 32 * i,
                              nb * S::COLS + 32 * S::TJ * (w >> 1), [&](int, int b, int q) { return sum[b][q]; });
}

// Up to 16 rows against a k-contiguous W: sixteen columns a workgroup, whose
// sixteen waves each take every sixteenth 32 k with 16 x 16 x 32 products straight from
// memory, and one sum in LDS.  Bound by the latency of a few loads and of the one launch
// (4 x 1280 x 1280 3.6 us in a graph; the small tiles, split along k and summed by a second
// launch, 7.5).
constexpr int FEW_ROWS = 16, FEW_WAVES = 16;

template <bool ACT>
__device__ __forceinline__ void finish_few(const Epilogue& e, int m, int col, float z) {
  if (m >= e.M || col >= e.N) return;
  float v[1] = {z};
  if (e.bias) v[0] += load1(e.bias, col, e.bias_f32);
  if constexpr (ACT) {
    if (e.pre) e.pre[m * e.ldp + col] = (__bf16)v[0];
    activate(e.act, v);
  }
  if (e.residual) v[0] += load1(e.residual, m * e.ldr + col, e.residual_f32);
  if (e.out_f32) static_cast<float*>(e.out)[m * e.ldo + col] = v[0];
  else static_cast<__bf16*>(e.out)[m * e.ldo + col] = (__bf16)v[0];
}

template <bool ACT>
__global__ __launch_bounds__(64 * FEW_WAVES) void linear_few_kernel(const __bf16* __restrict__ x, long ldx,
                                                                    const __bf16* __restrict__ w, long ldw, int K,
                                                                    const Epilogue e) {
  __shared__ float sums[FEW_WAVES][FEW_ROWS][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, n0 = blockIdx.x * 16;
  const __bf16* xr = x + (long)min(r, e.M - 1) * ldx;
  const __bf16* wr = w + (long)min(n0 + r, e.N - 1) * ldw;
  const bf16x8 zero = {};
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 32 * wave + 8 * (lane >> 4); k - 8 * (lane >> 4) < K; k += 32 * FEW_WAVES) {
    const bf16x8 a = k < K ? *reinterpret_cast<const bf16x8*>(wr + k) : zero;
    const bf16x8 b = k < K ? *reinterpret_cast<const bf16x8*>(xr + k) : zero;
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);     // columns of W down, rows of x across
  }
  *reinterpret_cast<f32x4*>(&sums[wave][r][4 * (lane >> 4)]) = acc;
  __syncthreads();
  const int m = threadIdx.x >> 4, n = threadIdx.x & 15;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < FEW_WAVES; ++i) v += sums[i][m][n];
  finish_few<ACT>(e, m, n0 + n, v);
}

// The same against a k-major W, as single tokens meet the feed-forward's down projection
// and as their dX meets a k-contiguous one: thirty-two columns a workgroup, a lane holding two
// neighbouring ones of eight k, whose halves make two products' operands.  Neighbouring
// workgroups, which share lines of W, run on one XCD.  4 x 3328 x 1280 6.2 us.
template <bool ACT>
__global__ __launch_bounds__(64 * FEW_WAVES) void linear_few_col_kernel(const __bf16* __restrict__ x, long ldx,
                                                                        const __bf16* __restrict__ w, long ldw, int K,
                                                                        const Epilogue e) {
  __shared__ __attribute__((aligned(16))) float sums[FEW_WAVES][FEW_ROWS][36];      // 32 columns
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int n0 = 32 * (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3));
  if (n0 >= e.N) return;
  const __bf16* xr = x + (long)min(r, e.M - 1) * ldx;
  const __bf16* wc = w + min(n0 + 2 * r, ((e.N + 7) & ~7) - 2);
  const bf16x8 zero = {};
  f32x4 acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
#pragma unroll 2
  for (int k = 32 * wave + 8 * g; k - 8 * g < K; k += 32 * FEW_WAVES) {
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? *reinterpret_cast<const uint32_t*>(wc + (long)(k + i) * ldw) : 0;
    const bf16x8 b = k < K ? *reinterpret_cast<const bf16x8*>(xr + k) : zero;
    u32x4 a0, a1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a0[i] = (v[2 * i + 1] << 16) | (v[2 * i] & 0xffffu);
      a1[i] = (v[2 * i + 1] & 0xffff0000u) | (v[2 * i] >> 16);
    }
    acc0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a0), b, acc0, 0, 0, 0);
    acc1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a1), b, acc1, 0, 0, 0);
  }
  *reinterpret_cast<f32x4*>(&sums[wave][r][8 * g]) = f32x4{acc0[0], acc1[0], acc0[1], acc1[1]};
  *reinterpret_cast<f32x4*>(&sums[wave][r][8 * g + 4]) = f32x4{acc0[2], acc1[2], acc0[3], acc1[3]};
  __syncthreads();
  if (threadIdx.x >= FEW_ROWS * 32) return;
  const int m = threadIdx.x >> 5, n = threadIdx.x & 31;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < FEW_WAVES; ++i) v += sums[i][m][n];
  finish_few<ACT>(e, m, n0 + n, v);
}

// ---------------------------------------------------------------------------
// dz and the column sums of dz before its rounding.  Workgroup (slab, block):
// 512 columns, eight per lane, and `rows` rows, its waves taking rows in turn;
// its column sums go to part[block], which colsum_kernel adds in block order.
// Bound by HBM: 16384 x 1280 fp32 to bf16 28.7 us (126 MB, 4.4 TB/s); 4096 x 3328 bf16
// with gelu's slope and column sums 22.6 + 4.9 (82 MB).
constexpr int GRAD_SLAB = 512, GRAD_AHEAD = 4;

template <class G, int ACT>
__global__ __launch_bounds__(256) void linear_grad_kernel(const G* __restrict__ dy, long ldy,
                                                          const __bf16* __restrict__ pre, long ldp,
                                                          __bf16* __restrict__ dz, long ldz, float* __restrict__ part,
                                                          int M, int N, int rows) {
  __shared__ float sums[4][GRAD_SLAB];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int col = blockIdx.x * GRAD_SLAB + 8 * lane, n = N - col;
  const long r0 = (long)blockIdx.y * rows, r1 = min((long)M, r0 + rows);
  float acc[8] = {};
  const bool out = dz && col < ldz;
  for (long r = r0 + w; r < r1; r += 4 * GRAD_AHEAD) {
    rows::Raw8<G> g[GRAD_AHEAD];
    rows::Raw8<__bf16> z[GRAD_AHEAD];
#pragma unroll
    for (int a = 0; a < GRAD_AHEAD; ++a) {
      const long row = r + 4 * a;
      if (n > 0 && row < r1) {
        g[a] = rows::load_any(dy + row * ldy + col, n);
        if constexpr (ACT != NONE) z[a] = rows::load_any(pre + row * ldp + col, n);
      }
    }
#pragma unroll
    for (int a = 0; a < GRAD_AHEAD; ++a) {
      const long row = r + 4 * a;
      if (row >= r1) break;
      float v[8] = {};
      if (n > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // columns past N: dy and z are zeros there
          v[j] = g[a][j];
          if constexpr (ACT != NONE) v[j] *= slope1<ACT>(z[a][j]);
          acc[j] += v[j];
        }
      }
      if (out) rows::store8(dz + row * ldz + col, v);      // ldz is a multiple of 8
    }
  }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[w][8 * lane + j] = acc[j];
  __syncthreads();
  for (int c = threadIdx.x; c < GRAD_SLAB; c += 256) {
    const int at = blockIdx.x * GRAD_SLAB + c;
    if (at < N) part[(long)blockIdx.y * N + at] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
  }
}

// 64 columns per workgroup, 16 groups of partial rows, then the groups in order.
template <class B>
__global__ __launch_bounds__(1024) void colsum_kernel(const float* __restrict__ part, int blocks, int N,
                                                      B* __restrict__ out) {
  __shared__ float sums[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6;
  float s = 0.f;
  if (c < N) {
#pragma unroll 4
    for (int b = g; b < blocks; b += 16) s += part[(long)b * N + c];
  }
  sums[g][threadIdx.x & 63] = s;
  __syncthreads();
  if (g > 0 || c >= N) return;
  for (int i = 1; i < 16; ++i) s += sums[i][threadIdx.x];
  out[c] = (B)s;
}

// bf16 copy of a matrix with rows and columns of zeros behind its own.
template <class T>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ src, long ld, int rows, int cols,
                                                   __bf16* __restrict__ dst, int pieces, long total) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long row = i / pieces;
    const int col = 8 * (int)(i - row * pieces);
    float v[8] = {};
    if (row < rows && col < cols) {
      const auto x = rows::load_any(src + row * ld + col, cols - col);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = x[j];
    }
    rows::store8(dst + 8 * i, v);
  }
}

// ---------------------------------------------------------------------------
struct Launch {
  const LinearArgs& a;
  const Plan& plan;
  int mid;
  const gemm::Problem& p;
  const Epilogue& e;
  hipStream_t stream;
};

// Allows a kernel its LDS, once per device (`done`: the devices that have it).
template <class K>
hipError_t allow_lds(K kern, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err != hipSuccess) return err;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
  err = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (err == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return err;
}

template <gemm::Layout LX, gemm::Layout LW, class S, bool ACT, class Tiles, bool RAGGED>
hipError_t launch_r(const Launch& l) {
  static std::atomic<uint64_t> done{0};
  auto kern = linear_kernel<LX, LW, S, ACT, Tiles, RAGGED>;
  const hipError_t err = allow_lds(kern, S::LDS_BYTES, done);
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(kern, dim3(l.plan.grid), dim3(512), S::LDS_BYTES, l.stream, l.p, l.e,
                     static_cast<float*>(l.a.workspace));
  return hipGetLastError();
}

// Checking every copy against K costs the large tiles up to a third of their
// rate with a k-contiguous x (4096 x 1280 x 3328 84 us, unchecked 70).
template <gemm::Layout LX, gemm::Layout LW, class S, bool ACT, class Tiles>
hipError_t launch_t(const Launch& l) {
  if constexpr (LX == gemm::ROW) {
    if (l.a.K % 128 == 0) return launch_r<LX, LW, S, ACT, Tiles, false>(l);
  }
  return launch_r<LX, LW, S, ACT, Tiles, true>(l);
}

template <gemm::Layout LX, gemm::Layout LW, bool ACT>
hipError_t launch_small(const Launch& l) {
  static std::atomic<uint64_t> done{0};
  auto kern = linear_small_kernel<LX, LW, ACT>;
  const hipError_t err = allow_lds(kern, gemm::SMALL_LDS, done);
  if (err != hipSuccess) return err;
  auto part = static_cast<float*>(l.a.workspace);
  hipLaunchKernelGGL(kern, dim3(l.plan.grid), dim3(256), gemm::SMALL_LDS, l.stream, l.p, l.e, part, l.plan.splits);
  if (l.plan.splits > 1)
    hipLaunchKernelGGL((linear_small_sum_kernel<ACT>), dim3(l.plan.n_mblk * l.plan.n_nblk), dim3(256), 0, l.stream,
                       static_cast<const float*>(part), l.e, l.plan.n_mblk, l.plan.splits);
  return hipGetLastError();
}

template <gemm::Layout LX, gemm::Layout LW, class S, bool ACT>
hipError_t launch_mid(const Launch& l) {
  static std::atomic<uint64_t> done{0};
  auto kern = linear_mid_kernel<LX, LW, S, ACT>;
  const hipError_t err = allow_lds(kern, S::LDS_BYTES, done);
  if (err != hipSuccess) return err;
  auto part = static_cast<float*>(l.a.workspace);
  hipLaunchKernelGGL(kern, dim3(l.plan.grid), dim3(256), S::LDS_BYTES, l.stream, l.p, l.e, part, l.plan.splits);
  if (l.plan.splits > 1)
    hipLaunchKernelGGL((linear_mid_sum_kernel<S, ACT>), dim3(4 * l.plan.n_mblk * l.plan.n_nblk), dim3(128), 0, l.stream,
                       static_cast<const float*>(part), l.e, l.plan.n_mblk, l.plan.n_nblk, l.plan.splits);
  return hipGetLastError();
}

template <gemm::Layout LX, gemm::Layout LW, class S, bool ACT>
hipError_t launch_s(const Launch& l) {
  if (l.plan.left == 0) return launch_t<LX, LW, S, ACT, gemm::WholeTiles>(l);
  const hipError_t err = launch_t<LX, LW, S, ACT, gemm::SplitTiles>(l);
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((linear_sum_kernel<S, ACT>), dim3(l.plan.left * 8), dim3(64 * S::TI), 0, l.stream,
                     static_cast<const float*>(l.a.workspace), l.e, l.plan.n_mblk, l.plan.n_nblk,
                     l.plan.n_mblk * l.plan.n_nblk - l.plan.left, l.plan.left, gemm::windows_of(l.a.K) / 2,
                     l.plan.grid);
  return hipGetLastError();
}

template <class S, int PARTS>
hipError_t launch_parts(const Launch& l) {
  const hipError_t err = launch_r<gemm::COL, gemm::COL, S, false, PartTiles<PARTS>, true>(l);
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((linear_part_sum_kernel<S>), dim3(8 * l.plan.n_mblk * l.plan.n_nblk), dim3(64 * S::TI), 0, l.stream,
                     static_cast<const float*>(l.a.workspace), l.e, l.plan.n_mblk, l.plan.n_nblk, PARTS);
  return hipGetLastError();
}
template <class S>
hipError_t launch_parts_s(const Launch& l, int parts) {
  return parts == 2 ? launch_parts<S, 2>(l) : parts == 4 ? launch_parts<S, 4>(l) : launch_parts<S, 8>(l);
}

template <gemm::Layout LX, gemm::Layout LW>
hipError_t launch_l(const Launch& l) {
  typedef gemm::Mid<2> Mid128;
  typedef gemm::Mid<3> Mid192;
  if constexpr (LX == gemm::ROW) {             // no activation behind two k-major operands
    if (l.a.act != NONE && l.mid)
      return l.mid == 2 ? launch_mid<LX, LW, Mid128, true>(l) : launch_mid<LX, LW, Mid192, true>(l);
    if (l.a.act != NONE)
      return l.plan.splits > 0 ? launch_small<LX, LW, true>(l) : launch_s<LX, LW, gemm::Wide256, true>(l);
  }
  if (l.mid) return l.mid == 2 ? launch_mid<LX, LW, Mid128, false>(l) : launch_mid<LX, LW, Mid192, false>(l);
  if (l.plan.splits > 0) return launch_small<LX, LW, false>(l);
  return l.plan.wide320 ? launch_s<LX, LW, gemm::Wide320, false>(l) : launch_s<LX, LW, gemm::Wide256, false>(l);
}

int cus_or_default() {
  int cus = 0;
  return cu_count(cus) == hipSuccess ? cus : 256;
}

// Times of the mid tiles in us, for 128 and 192 columns: a tile alone on its CU and
// two that share it (launch, first fill and epilogue; a window), and the sum of the
// splits (its launch, a tile's epilogue, its bytes).  Fitted to 37 products of 100 to
// 16384 rows.
struct MidTimes {
  double fixed, window;
};
constexpr MidTimes MID_ALONE[2] = {{4.3, 0.67}, {9.5, 0.74}}, MID_SHARED[2] = {{8, 1.0}, {11, 1.34}};
constexpr double MID_SUM = 3.5, MID_SUM_TILE = 0.045, MID_BYTES = 2e7;
// ... and by how much they have to beat the model of the core's tiles, which is up to
// a tenth too high itself.
constexpr double MID_MARGIN = 0.93;

// Times of PartTiles and, where SplitTiles does not give every tile a whole number of
// workgroups, of SplitTiles, in us: fixed, a window of a 256-column tile, a byte of the
// partial sums.  Fitted to 18 products of K from 4096 on.
constexpr double PART_FIXED = 8, PART_WINDOW = 1.55, PART_BYTE = 0.36e-6, LOOSE_FIXED = 18, LOOSE_WINDOW = 2.4;

struct LinearPlan {
  Plan plan;
  int mid;                 // column blocks of the mid tiles (2, 3), 0: the core's tiles
  int parts;               // of PartTiles (2, 4, 8), 0: none
};

// PartTiles for two k-major operands where one round of them takes less than the plan.
void plan_parts(int M, int N, int K, int n_g, LinearPlan& best) {
  const int n_win = gemm::windows_of(K);
  double us = best.plan.cost * WINDOW_US;
  if (!best.mid && best.plan.left > 0 && n_g % best.plan.left != 0) {
    const long total = (long)best.plan.n_mblk * best.plan.n_nblk;
    const double tile = (double)n_win * (best.plan.wide320 ? 1.25 : 1);
    us = LOOSE_FIXED + (double)(total / n_g) * tile * PART_WINDOW + (double)best.plan.left / n_g * tile * LOOSE_WINDOW;
  }
  for (int bn = 256; bn <= 320; bn += 64) {
    for (int parts = 2; parts <= 8; parts *= 2) {
      Plan p{};
      p.wide320 = bn == 320;
      p.n_mblk = (M + gemm::BM - 1) / gemm::BM;
      p.n_nblk = (N + bn - 1) / bn;
      p.grid = n_g;
      const long tiles = (long)p.n_mblk * p.n_nblk;
      if (n_win < 8 * parts || (tiles * parts + 7) / 8 > n_g / 8) continue;
      p.part_bytes = (size_t)(tiles * parts) * gemm::BM * bn * 4;
      const int each = (n_win / 2 + parts - 1) / parts * 2;
      const double t = PART_FIXED + each * PART_WINDOW * bn / 256 + (double)p.part_bytes * PART_BYTE;
      if (t >= us) continue;
      us = t;
      p.cost = t / WINDOW_US;
      best = {p, 0, parts};
    }
  }
}

// The tiles and splits of least modelled time; the model has no term for the bytes of
// residual, z and output, which weigh most behind a lone round of large tiles (4096 x
// 3328 x 1280 with gelu and z 51 us, 33 for the library's plain product).  An activation takes no 320-column
// tiles: their accumulators leave it no registers.
LinearPlan plan_for(int M, int N, int K, bool k_major, bool act, int cus) {
  const int n_g = ((cus > 0 ? cus : 256) + 7) & ~7;
  LinearPlan best{};
  if (act) {
    const Plan large = plan_of(256, M, N, K, k_major, n_g), small = small_plan(M, N, K, n_g);
    best.plan = small.cost < large.cost ? small : large;
  } else {
    best.plan = make_plan(M, N, K, k_major, cus, false);
  }
  const int n_win = (K + gemm::BK - 1) / gemm::BK;
  for (int tj = 2; tj <= 3; ++tj) {
    Plan p{};
    p.n_mblk = (M + 127) / 128;
    p.n_nblk = (N + 64 * tj - 1) / (64 * tj);
    const long tiles = (long)p.n_mblk * p.n_nblk;
    for (int s = 1; s <= 16 && (s == 1 || (s * 8 <= n_win && s * tiles <= 2 * n_g)); ++s) {
      const long n = tiles * s, rest = n % (2 * n_g);
      const double win = (n_win + s - 1) / s;
      auto us_of = [&](const MidTimes& t) { return t.fixed + t.window * win; };
      const double full = (double)(n / (2 * n_g)) * us_of(MID_SHARED[tj - 2]);
      const double last = rest == 0 ? 0 : us_of(rest > n_g ? MID_SHARED[tj - 2] : MID_ALONE[tj - 2]);
      const size_t bytes = s > 1 ? (size_t)n * 128 * 64 * tj * 4 : 0;
      const double us = full + last + (s > 1 ? MID_SUM + MID_SUM_TILE * tiles + (double)bytes / MID_BYTES : 0);
      if (us / WINDOW_US >= (best.mid ? 1 : MID_MARGIN) * best.plan.cost) continue;
      p.splits = s;
      p.cost = us / WINDOW_US;
      p.grid = (int)((tiles * s + 7) / 8 * 8);
      p.part_bytes = bytes;
      best = {p, tj, 0};
    }
  }
  if (k_major) plan_parts(M, N, K, n_g, best);
  return best;
}

int ceil8(int n) { return (n + 7) & ~7; }

// Rows of a workgroup of linear_grad_kernel: about 4 workgroups a CU, at least
// 16 rows each and, for the sum of their partials, at most 1024 of them in a column.
int grad_rows(int M, int N) {
  const long slabs = (N + GRAD_SLAB - 1) / GRAD_SLAB;
  long rows = (M * slabs + 1023) / 1024;
  const long least = ((long)M + 1023) / 1024;
  rows = rows < least ? least : rows;
  rows = rows < 16 ? 16 : rows;
  return (int)((rows + 15) / 16 * 16);
}

template <class G, int ACT>
void launch_grad_t(const LinearGradArgs& a, int rows, hipStream_t stream) {
  const int width = a.dz && a.ldz > a.N ? (int)a.ldz : a.N;
  const dim3 grid((width + GRAD_SLAB - 1) / GRAD_SLAB, (a.M + rows - 1) / rows);
  hipLaunchKernelGGL((linear_grad_kernel<G, ACT>), grid, dim3(256), 0, stream, static_cast<const G*>(a.dy), a.ldy,
                     static_cast<const __bf16*>(a.pre), a.ldp, static_cast<__bf16*>(a.dz), a.ldz,
                     a.dbias ? static_cast<float*>(a.workspace) : nullptr, a.M, a.N, rows);
}

template <class G>
void launch_grad_g(const LinearGradArgs& a, int rows, hipStream_t stream) {
  switch (a.act) {
    case RELU: launch_grad_t<G, RELU>(a, rows, stream); break;
    case GELU: launch_grad_t<G, GELU>(a, rows, stream); break;
    case GELU_TANH: launch_grad_t<G, GELU_TANH>(a, rows, stream); break;
    case SILU: launch_grad_t<G, SILU>(a, rows, stream); break;
    default: launch_grad_t<G, NONE>(a, rows, stream); break;
  }
}

}  // namespace

// A workgroup walks all of k, so long sums go to the tiles, which split them, and with
// thousands of columns the tiles read W as fast (4 rows, k-major W, us here and with tiles:
// 1280 x 1280 3.8, 7.5; 1280 x 3328 6.2, 10.7; 3328 x 1280 3.9, 8.5; 1280 x 16384 33, 16;
// 16384 x 3328 21.7, 21.0; 16 rows 22.8, 19.6).
static bool few(int M, int N, int K, int x_layout) {
  return M <= FEW_ROWS && N <= 8192 && K <= 6144 && x_layout == gemm::ROW;
}

size_t linear_workspace_bytes(int M, int N, int K, int x_layout, int w_layout, bool act) {
  if (few(M, N, K, x_layout)) return 0;
  return plan_for(M, N, K, x_layout == gemm::COL, act, cus_or_default()).plan.part_bytes;
}

// The plain products of whole pieces run on gemm.hip's kernels, which round
// before the exchange and so exchange half as often (16384 x 3328 x 1280 126 us, 148
// here).
static bool plain(const LinearArgs& a) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.out);
  return !a.bias && !a.residual && a.act == NONE && a.N % 8 == 0 && a.ldo % 8 == 0 && at % 16 == 0 &&
         (a.x_layout == gemm::COL ? a.M % 8 == 0 : a.K % 128 == 0);
}

hipError_t launch_linear(const LinearArgs& a, hipStream_t stream) {
  int cus = 0;
  const hipError_t err = cu_count(cus);
  if (err != hipSuccess) return err;
  const bool xc = a.x_layout == gemm::COL, wc = a.w_layout == gemm::COL;
  const Epilogue e{a.bias, a.residual, a.out, static_cast<__bf16*>(a.pre), a.ldr, a.ldp, a.ldo, a.M, a.N, a.act,
                   a.bias_f32, a.residual_f32, a.out_f32};
  if (few(a.M, a.N, a.K, a.x_layout)) {
    auto kern = wc ? (a.act == NONE ? linear_few_col_kernel<false> : linear_few_col_kernel<true>)
                   : (a.act == NONE ? linear_few_kernel<false> : linear_few_kernel<true>);
    hipLaunchKernelGGL(kern, dim3(wc ? ((a.N + 31) / 32 + 7) / 8 * 8 : (a.N + 15) / 16), dim3(64 * FEW_WAVES), 0, stream, static_cast<const __bf16*>(a.x), a.ldx,
                       static_cast<const __bf16*>(a.w), a.ldw, a.K, e);
    return hipGetLastError();
  }
  const LinearPlan chosen = plan_for(a.M, a.N, a.K, xc, a.act != NONE, cus);
  const Plan& plan = chosen.plan;
  if (!chosen.mid && !chosen.parts && plain(a))
    return launch_gemm({a.x, a.ldx, a.x_layout, a.w, a.ldw, a.w_layout, nullptr, 0, a.out, nullptr, 0, a.ldo, a.out_f32,
                        a.workspace, a.M, a.N, a.K},
                       stream);
  // a k-major operand is read in pieces of 8 columns
  const gemm::Problem p{{static_cast<const __bf16*>(a.x), a.ldx, xc ? ceil8(a.M) : a.M},
                        {static_cast<const __bf16*>(a.w), a.ldw, wc ? ceil8(a.N) : a.N},
                        nullptr, 0, a.K, plan.n_mblk, plan.n_nblk};
  const Launch l{a, plan, chosen.mid, p, e, stream};
  if (chosen.parts)
    return plan.wide320 ? launch_parts_s<gemm::Wide320>(l, chosen.parts) : launch_parts_s<gemm::Wide256>(l, chosen.parts);
  if (xc) return launch_l<gemm::COL, gemm::COL>(l);
  return wc ? launch_l<gemm::ROW, gemm::COL>(l) : launch_l<gemm::ROW, gemm::ROW>(l);
}

size_t linear_grad_workspace_bytes(int M, int N) {
  const int rows = grad_rows(M, N);
  return (size_t)((M + rows - 1) / rows) * N * sizeof(float);
}

hipError_t launch_linear_grad(const LinearGradArgs& a, hipStream_t stream) {
  const int rows = grad_rows(a.M, a.N);
  if (a.dy_f32) launch_grad_g<float>(a, rows, stream);
  else launch_grad_g<__bf16>(a, rows, stream);
  if (a.dbias) {
    const dim3 grid((a.N + 63) / 64), block(1024);
    const int blocks = (a.M + rows - 1) / rows;
    const float* part = static_cast<const float*>(a.workspace);
    if (a.dbias_f32)
      hipLaunchKernelGGL((colsum_kernel<float>), grid, block, 0, stream, part, blocks, a.N, static_cast<float*>(a.dbias));
    else
      hipLaunchKernelGGL((colsum_kernel<__bf16>), grid, block, 0, stream, part, blocks, a.N,
                         static_cast<__bf16*>(a.dbias));
  }
  return hipGetLastError();
}

hipError_t launch_pack_bf16(const void* src, bool src_f32, long ld, int rows, int cols, void* dst, long ldd,
                            int rows_out, hipStream_t stream) {
  const int pieces = (int)(ldd / 8);
  const long total = (long)rows_out * pieces, need = (total + 255) / 256;
  const dim3 grid((unsigned)(need < 16384 ? need : 16384)), block(256);
  if (src_f32)
    hipLaunchKernelGGL((pack_kernel<float>), grid, block, 0, stream, static_cast<const float*>(src), ld, rows, cols,
                       static_cast<__bf16*>(dst), pieces, total);
  else
    hipLaunchKernelGGL((pack_kernel<__bf16>), grid, block, 0, stream, static_cast<const __bf16*>(src), ld, rows, cols,
                       static_cast<__bf16*>(dst), pieces, total);
  return hipGetLastError();
}

}  // namespace mm1
