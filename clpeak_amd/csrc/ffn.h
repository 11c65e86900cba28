// Shared by the feed-forward operators (mi355_glu_*, mi355_gemm_i8_scaled, mi355_quantize_i8): what a product's kernel
// does with a finished sum, and the activations.  The sums are fp32 (int32 for int8 operands); every kernel finishes
// them in registers, so that nothing but the operator's own outputs goes to memory.
#pragma once
#include "internal.h"
#include "mfma_common.h"
#include "gemm_quad.h"

// What becomes of the sums.
enum FfnEpi {
  kEpiPlain = 0,        // C = sum, rounded to the operands' 16-bit type
  kEpiScaled = 1,       // int8 operands: C = sum * scale_a[row] * scale_b[col] (+ bias[col])
  kEpiGated = 2,        // 16-bit operands, two products: H = act(gate) * up, the two sums kept where asked for
  kEpiGatedScaled = 3,  // int8 operands, two products, each sum scaled first
};
constexpr bool epi_is_gated(int epi) { return epi == kEpiGated || epi == kEpiGatedScaled; }

struct FfnOut {
  void *c;               // C or H, rows of ldc elements
  uint64_t ldc;
  void *g, *u;           // kEpiGated: where the two sums are kept (both or neither)
  uint64_t ldg;
  const float *sa, *sb, *sb2, *bias;
  int type;              // of C / H: MI355_TYPE_*
  int act;               // MI355_GLU_*
};

// One product of rows: A[M][K] with the rows of B (gated: of B and of B2, both N rows).  Strides and K in bytes, K a
// multiple of 128; strides and addresses multiples of 16.
struct FfnProduct {
  const uint8_t *a, *b, *b2;
  uint64_t lda, ldb;
  uint32_t m, n, k_bytes;
  FfnOut out;
};

// ffn_rows.hip: any shape; the kernel for few rows.  op: kQuadBf16 / kQuadF16 / kQuadI8.
int mi355_launch_ffn_rows(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p);

// ffn.hip: the kernel that suits the product.
int mi355_ffn_product(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p);

// ffn_backward.hip (arguments checked by the caller).
int mi355_glu_backward_limits(mi355_dev *dev, const char *what, uint32_t T, uint32_t F);
size_t mi355_glu_backward_bytes(uint32_t T, uint32_t F, uint32_t D);
int mi355_launch_glu_backward(mi355_dev *dev, int type, int act, const void *dH, uint64_t lddh, const void *X, uint64_t ldx, const void *Wg,
                              const void *Wu, uint64_t ldw, const void *G, const void *U, uint64_t ldg, void *dX, uint64_t lddx, void *dWg,
                              void *dWu, uint64_t lddw, uint32_t T, uint32_t F, uint32_t D, uint8_t *workspace);

// ---- activations -------------------------------------------------------------------------------------------------
// In fp32 from the unrounded sums.  sigmoid(x) = 1 / (1 + 2^(-x log2 e)): the exponential and the reciprocal are one
// instruction each, off by about an ulp, which the 16-bit roundings behind them (2^-9 and coarser) do not see; what the
// rounding of x log2 e adds is |x| 2^-24 relative, and where |x| is large enough for that to count, sigmoid is 0 or 1.
__device__ __forceinline__ float ffn_sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f));
}
// 2 y of gelu's tanh form, act = x sigmoid(2 y), y = sqrt(2/pi) (x + 0.044715 x^3).  |x| is held to 16, where sigmoid
// has long been 0 or 1 (2 y = 317): the cube of a far larger one would overflow and meet a zero in the derivative.
__device__ __forceinline__ float ffn_gelu_tanh_arg(float x) {
  const float c = fminf(fmaxf(x, -16.0f), 16.0f);
  return 1.59576912160573071f * c * fmaf(0.044715f * c, c, 1.0f);
}
__device__ __forceinline__ float ffn_act(int act, float x) {
  if (act == MI355_GLU_SILU) return x * ffn_sigmoid(x);
  if (act == MI355_GLU_GELU_TANH) return x * ffn_sigmoid(ffn_gelu_tanh_arg(x));
  if (act == MI355_GLU_GELU) return 0.5f * x * (1.0f + erff(x * 0.707106781186547524f));
  return x < 0.0f ? 0.0f : x;   // (a NaN stays one)
}
// The activation and its derivative.
__device__ __forceinline__ void ffn_act_grad(int act, float x, float &a, float &da) {
  if (act == MI355_GLU_SILU) {
    const float p = ffn_sigmoid(x);
    a = x * p;
    da = fmaf(a, 1.0f - p, p);
  } else if (act == MI355_GLU_GELU_TANH) {
    const float p = ffn_sigmoid(ffn_gelu_tanh_arg(x));
    const float c = fminf(fmaxf(x, -16.0f), 16.0f);
    a = x * p;
    da = fmaf(a * (1.0f - p), 1.59576912160573071f * fmaf(0.134145f * c, c, 1.0f), p);
  } else if (act == MI355_GLU_GELU) {
    const float cdf = 0.5f * (1.0f + erff(x * 0.707106781186547524f));
    a = x * cdf;
    const float c = fminf(fmaxf(x, -16.0f), 16.0f);
    da = fmaf(c * 0.398942280401432678f, __builtin_amdgcn_exp2f(c * c * -0.72134752044448170f), cdf);
  } else {
    a = x < 0.0f ? 0.0f : x;
    da = x > 0.0f ? 1.0f : x <= 0.0f ? 0.0f : x;
  }
}

// ---- stores of narrow values -----------------------------------------------------------------------------------------
// Rounded once, to nearest even, from fp32.
__device__ __forceinline__ void ffn_store1(void *base, uint64_t at, int type, float x) {
  if (type == MI355_TYPE_F32) { static_cast<float *>(base)[at] = x; return; }
  const uint32_t p = type == MI355_TYPE_F16 ? mi355_pack_f16x2(x, 0.0f) : mi355_pack_bf16x2(x, 0.0f);
  static_cast<uint16_t *>(base)[at] = (uint16_t)p;
}
__device__ __forceinline__ float ffn_load1(const void *base, uint64_t at, int type) {
  if (type == MI355_TYPE_F32) return static_cast<const float *>(base)[at];
  if (type == MI355_TYPE_F16) return (float)static_cast<const _Float16 *>(base)[at];
  const uint32_t bits = (uint32_t)static_cast<const uint16_t *>(base)[at] << 16;
  return __builtin_bit_cast(float, bits);
}

// int32 sum -> value.  The sum is rounded to fp32 (exact below 2^24), then multiplied by the two scales in turn, so that
// neither product of a small and a large scale leaves the range before the sum is in it.
__device__ __forceinline__ float ffn_scaled(int32_t sum, float sa, float sb) { return (float)sum * sa * sb; }

// One element of the output from its sum (gated: from its two sums), as raw bits of fp32 or int32.
template <int EPI>
__device__ __forceinline__ void ffn_finish1(const FfnOut &o, uint32_t row, uint32_t col, int32_t s0, int32_t s1) {
  const uint64_t at = (uint64_t)row * o.ldc + col;
  if constexpr (EPI == kEpiPlain) {
    ffn_store1(o.c, at, o.type, __builtin_bit_cast(float, s0));
  } else if constexpr (EPI == kEpiScaled) {
    float v = ffn_scaled(s0, o.sa[row], o.sb[col]);
    if (o.bias) v += o.bias[col];
    ffn_store1(o.c, at, o.type, v);
  } else if constexpr (EPI == kEpiGated) {
    const float g = __builtin_bit_cast(float, s0), u = __builtin_bit_cast(float, s1);
    ffn_store1(o.c, at, o.type, ffn_act(o.act, g) * u);
    if (o.g) {
      const uint64_t kept = (uint64_t)row * o.ldg + col;
      ffn_store1(o.g, kept, o.type, g);
      ffn_store1(o.u, kept, o.type, u);
    }
  } else {
    const float sa = o.sa[row];
    ffn_store1(o.c, at, o.type, ffn_act(o.act, ffn_scaled(s0, sa, o.sb[col])) * ffn_scaled(s1, sa, o.sb2[col]));
  }
}
