// Shared by the feed-forward operators (mi355_glu_*, mi355_gemm_i8_scaled, mi355_quantize_i8): what a product's kernel
// does with a finished sum, and the activations.  The sums are fp32 (int32 for int8 operands); every kernel finishes
// them in registers, so that nothing but the operator's own outputs goes to memory.
#pragma once
#include "internal.h"
#include "mfma_common.h"
#include "gemm_quad.h"
#include "gemm_ring.h"

// What becomes of the sums.
enum FfnEpi {
  kEpiPlain = 0,        // C = sum, rounded to the operands' 16-bit type
  kEpiScaled = 1,       // int8 operands: C = sum * scale_a[row] * scale_b[col] (+ bias[col])
  kEpiGated = 2,        // 16-bit operands, two products: H = act(gate) * up, the two sums kept where asked for
  kEpiGatedScaled = 3,  // int8 operands, two products, each sum scaled first
  kEpiPartial = 4,      // the sums of a slice of K, as they are (32 bits each)
};
constexpr bool epi_is_gated(int epi) { return epi == kEpiGated || epi == kEpiGatedScaled; }

struct FfnOut {
  void *c;               // C or H, rows of ldc elements
  uint64_t ldc;
  void *g, *u;           // kEpiGated: where the two sums are kept (both or neither)
  uint64_t ldg;
  const float *sa, *sb, *sb2, *bias;   // (kEpiPlain of fp16: one value at sa, which C's sums are multiplied by)
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

// ffn_rows.hip: at most 64 rows of A.  op: kQuadBf16 / kQuadF16 / kQuadI8.
int mi355_launch_ffn_rows(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p);

// ffn_quad.hip / ffn_small.hip: on 256x256 and on 128x128 (tall: 256x128) tiles of sums (gated: half as many columns of outputs).
int mi355_launch_ffn_quad(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p);
// ffn_mid.hip: on 64x64 tiles of sums (gated: of 64x32 outputs), for some dozens of rows.
// slices > 1 (kEpiScaled): K is cut into so many, `workspace` holds `slices` matrices of m rows of
// mi355_ffn_slice_row(n) 32-bit sums, on 16 bytes.
int mi355_launch_ffn_small(mi355_dev *dev, int op, int epi, const char *what, bool tall, const FfnProduct &p, uint32_t slices, void *workspace);
int mi355_launch_ffn_mid(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p, uint32_t slices, void *workspace);
// kEpiPlain, on either: up to three products of 16-bit operands in one launch, each in slices of its own number.
struct FfnGroup {
  struct One {
    const uint8_t *a, *b;
    uint64_t lda, ldb, ldc;
    void *c;
    uint32_t m, n, k_bytes, slices;
    uint32_t pairs;                     // 1: the result is the sum of the upper and the lower half of the rows
    uint32_t tiles_m, tiles_n, first;   // (the launch's: the number of the product's first workgroup)
  } of[3];
  uint32_t count;
  int type;
  const float *sa;                      // (FfnOut's)
};
struct FfnGroupChoice {
  int kernel;             // (ffn.hip's number of it)
  uint32_t slices[3];
  double us;
};
// (ffn.hip: the longest walks first; tiles of rows x cols sums)
int mi355_ffn_lay_out_group(mi355_dev *dev, const char *what, FfnGroup &g, uint32_t rows, uint32_t cols, uint32_t &blocks);
int mi355_launch_ffn_small_group(mi355_dev *dev, int op, const char *what, bool tall, const FfnGroup &g);
int mi355_launch_ffn_mid_group(mi355_dev *dev, int op, const char *what, const FfnGroup &g);
// ffn_join.hip: the second launch of products in slices, up to three of them.
struct FfnJoin {
  FfnOut out;
  const int32_t *partial;
  uint64_t ldp;
  uint32_t m, n, slices, first;   // (first: the launch's)
};
int mi355_launch_ffn_join(mi355_dev *dev, int op, int epi, const char *what, FfnJoin *parts, uint32_t count);
inline uint64_t mi355_ffn_slice_row(uint32_t n) { return (n + 3ull) / 4u * 4u; }
// The product whose outputs are the sums of the slices, in the workspace.
inline FfnProduct mi355_ffn_slices_of(const FfnProduct &p, void *workspace) {
  FfnProduct q = p;
  q.out.c = workspace;
  q.out.ldc = mi355_ffn_slice_row(p.n);
  q.out.type = MI355_TYPE_F32;
  return q;
}
// (pairs: each slice's matrix is two of half as many rows)
inline FfnJoin mi355_ffn_join_of(const FfnProduct &p, uint32_t slices, bool pairs, const void *workspace) {
  return {p.out, static_cast<const int32_t *>(workspace), mi355_ffn_slice_row(p.n), pairs ? p.m / 2u : p.m, p.n, pairs ? 2u * slices : slices, 0};
}

// What the kernels on 64x64 and 128x128 tiles are given, and what a workgroup makes of it: a tile of a product, and a slice
// of its K.
struct FfnWork {
  FfnProduct p;
  uint32_t tiles_m, tiles_n, tile, slice, slices;
};
template <int EPI>
struct FfnLaunch {
  FfnProduct p;
  uint32_t tiles_m, tiles_n;
  __device__ __forceinline__ FfnWork work() const {
    FfnWork w{p, tiles_m, tiles_n, blockIdx.x, 0, 1};
    if constexpr (EPI == kEpiPartial) {   // (the sums go to p.out.c as matrix number blockIdx.y there)
      w.slice = blockIdx.y; w.slices = gridDim.y;
      w.p.out.c = static_cast<float *>(p.out.c) + (uint64_t)blockIdx.y * p.m * p.out.ldc;
    }
    return w;
  }
};
template <>
struct FfnLaunch<kEpiPlain> {
  FfnGroup g;
  __device__ __forceinline__ FfnWork work() const {
    // member by member, with no index that varies: the addresses have to stay in scalar registers
    const bool second = blockIdx.x >= g.of[1].first, third = blockIdx.x >= g.of[2].first;
    FfnGroup::One o;
#define MI355_PICK(x) o.x = third ? g.of[2].x : second ? g.of[1].x : g.of[0].x
    MI355_PICK(a); MI355_PICK(b); MI355_PICK(lda); MI355_PICK(ldb); MI355_PICK(ldc); MI355_PICK(c);
    MI355_PICK(m); MI355_PICK(n); MI355_PICK(k_bytes); MI355_PICK(slices); MI355_PICK(pairs); MI355_PICK(tiles_m); MI355_PICK(tiles_n); MI355_PICK(first);
#undef MI355_PICK
    const uint32_t at = blockIdx.x - o.first, tiles = o.tiles_m * o.tiles_n;
    FfnWork w{};
    w.p.a = o.a; w.p.b = o.b; w.p.lda = o.lda; w.p.ldb = o.ldb;
    w.p.m = o.m; w.p.n = o.n; w.p.k_bytes = o.k_bytes;
    w.tiles_m = o.tiles_m; w.tiles_n = o.tiles_n;
    w.slice = at / tiles; w.tile = at - w.slice * tiles; w.slices = o.slices;
    w.p.out.ldc = o.ldc;
    w.p.out.sa = g.sa;
    w.p.out.type = o.slices > 1u || o.pairs ? MI355_TYPE_F32 : g.type;
    w.p.out.c = static_cast<uint8_t *>(o.c) + (o.slices > 1u ? (uint64_t)w.slice * o.m * o.ldc * 4u : 0u);
    return w;
  }
};

// The number of a kernel among those on one shape of tile (256x256 ones apart).
constexpr int ffn_kind(int op, int epi) {
  return op != kQuadI8 ? (op - kQuadBf16) * 2 + epi_is_gated(epi) : 4 + (epi == kEpiPartial ? 2 : epi_is_gated(epi));
}

// ffn.hip: the product on the kernel that suits it, and the workspace that it can use.
int mi355_ffn_product(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p, void *workspace, size_t workspace_bytes);
size_t mi355_ffn_workspace(const mi355_dev *dev, int epi, uint32_t m, uint32_t n, uint32_t k_bytes);
// A group's tiling and slices (of its products m, n and k_bytes are looked at) and its launches, slices joined; the
// workspace that the slices need; the time expected of a product on ffn_rows.hip (more than 64 rows: forever).
FfnGroupChoice mi355_choose_ffn_group(const mi355_dev *dev, const FfnGroup &g);
size_t mi355_ffn_group_workspace(const FfnGroup &g, const FfnGroupChoice &c);
int mi355_ffn_group(mi355_dev *dev, int op, const char *what, const FfnGroup &g, const FfnGroupChoice &c, uint8_t *workspace);
double mi355_ffn_rows_us(const mi355_dev *dev, int epi, uint32_t m, uint32_t n, uint32_t k_bytes);

// ffn_backward.hip (arguments checked by the caller).
int mi355_glu_backward_limits(mi355_dev *dev, const char *what, uint32_t T, uint32_t F);
size_t mi355_glu_backward_bytes(const mi355_dev *dev, uint32_t T, uint32_t F, uint32_t D);
int mi355_launch_glu_backward(mi355_dev *dev, int type, int act, const void *dH, uint64_t lddh, const void *X, uint64_t ldx, const void *Wg,
                              const void *Wu, uint64_t ldw, const void *G, const void *U, uint64_t ldg, void *dX, uint64_t lddx, void *dWg,
                              void *dWu, uint64_t lddw, uint32_t T, uint32_t F, uint32_t D, uint8_t *workspace);

// ---- activations -------------------------------------------------------------------------------------------------
// In fp32 from the unrounded sums, each right relative to itself, also where it is small: some outputs are fp32.
// sigmoid(x) = 1 / (1 + 2^(-x log2 e)): the exponential and the reciprocal are one instruction each, off by about an ulp;
// the roundings of x log2 e add 2 |x| 2^-24 relative, as much as a rounding of x itself does there.  (Exponentials out of
// fp32's normal range are 0 or infinite: a silu or gelu below 2^-100 may be 0.)
__device__ __forceinline__ float ffn_sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f));
}
// 2 y of gelu's tanh form, act = x sigmoid(2 y), y = sqrt(2/pi) (x + 0.044715 x^3).  |x| is held to 16, where sigmoid
// has long been 0 or 1 (2 y = 317): the cube of a far larger one would overflow and meet a zero in the derivative.
__device__ __forceinline__ float ffn_gelu_tanh_arg(float x) {
  const float c = fminf(fmaxf(x, -16.0f), 16.0f);
  return 1.59576912160573071f * c * fmaf(0.044715f * c, c, 1.0f);
}
// The normal distribution's function, 1/2 (1 + erf(x / sqrt 2)), and e = exp(-x^2 / 2), its density times sqrt(2 pi).  The
// smaller tail is e t P(t), t = 1 / (1 + 0.35 |x|), P the polynomial of eighth degree nearest to the quotient relative to it
// (fitted to scipy's scaled complementary error function over 0 .. 14: 3.2e-8, in fp32 3e-7); the larger one is 1 less
// that.  Left of 0 nothing cancels, as it would in 1 + erf.
__device__ __forceinline__ float ffn_normal(float x, float &e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, fabsf(x), 1.0f));
  float p = -0.0291459389f;
  p = fmaf(p, t, 0.1439717392f);
  p = fmaf(p, t, -0.2557143386f);
  p = fmaf(p, t, 0.1591742553f);
  p = fmaf(p, t, -0.0231098999f);
  p = fmaf(p, t, 0.1055080313f);
  p = fmaf(p, t, 0.1198328607f);
  p = fmaf(p, t, 0.1398618706f);
  p = fmaf(p, t, 0.1396214042f);
  e = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
  const float tail = p * t * e;
  return x < 0.0f ? tail : 1.0f - tail;
}
__device__ __forceinline__ float ffn_act(int act, float x) {
  if (act == MI355_GLU_SILU) return x * ffn_sigmoid(x);
  if (act == MI355_GLU_GELU_TANH) return x * ffn_sigmoid(ffn_gelu_tanh_arg(x));
  if (act == MI355_GLU_GELU) {
    float e;
    return x * ffn_normal(x, e);
  }
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
    float e;
    const float cdf = ffn_normal(x, e);
    a = x * cdf;
    da = fmaf(fminf(fmaxf(x, -16.0f), 16.0f) * 0.398942280401432678f, e, cdf);   // (past 16 e is 0)
  } else {
    a = x < 0.0f ? 0.0f : x;
    da = x > 0.0f ? 1.0f : x <= 0.0f ? 0.0f : x;
  }
}

// ---- the order of the tiles --------------------------------------------------------------------------------------------
// tile_at's, and where the number of tiles is no multiple of the XCDs' (8) still consecutive tiles for each XCD: neighbours
// share rows of both operands, and where rows of C do not start on lines also the lines between them, which an L2 can
// only complete if both are its own (gated 7525x8347x1024 fp16: 266 -> 236 us).
__device__ __forceinline__ void ffn_tile_at(const TileGrid &g, uint32_t round, uint32_t &tm, uint32_t &tn) {
  if (g.total % 8u == 0u) return tile_at(g, round, tm, tn);
  const uint32_t id = g.first + round * g.stride, xcd = id % 8u, rest = g.total % 8u;
  const uint32_t lin = xcd * (g.total / 8u) + min(xcd, rest) + id / 8u;
  const uint32_t per_group = 4u * g.tiles_n, group = lin / per_group, in_group = lin - group * per_group;
  const uint32_t rows_here = min(4u, g.tiles_m - group * 4u);
  tn = in_group / rows_here;
  tm = group * 4u + in_group - tn * rows_here;
}

// ---- stores of narrow values -----------------------------------------------------------------------------------------
// Rounded once, to nearest even, from fp32.
__device__ __forceinline__ void ffn_store1(void *base, uint64_t at, int type, float x) {
  if (type == MI355_TYPE_F32) { static_cast<float *>(base)[at] = x; return; }
  const uint32_t p = type == MI355_TYPE_F16 ? mi355_pack_f16x2(x, 0.0f) : mi355_pack_bf16x2(x, 0.0f);
  static_cast<uint16_t *>(base)[at] = (uint16_t)p;
}

// int32 sum -> value.  The sum is rounded to fp32 (exact below 2^24), then multiplied by the two scales in turn.  The first
// product never loses bits below the range (the sum is a whole number) and leaves it above only for scale_a of 2^97 and
// more, which the header rules out: to take the smaller scale first would cost three operations a sum.
__device__ __forceinline__ float ffn_scaled(int32_t sum, float sa, float sb) { return (float)sum * sa * sb; }
// (the addition as one operation with the second product, in every kernel alike)
__device__ __forceinline__ float ffn_scaled_plus(int32_t sum, float sa, float sb, float bias) { return fmaf((float)sum * sa, sb, bias); }

// ---- finished tiles --------------------------------------------------------------------------------
// A wave's sums are tiles of 16x16, and a lane holds 4 consecutive columns of one row of a tile: row lane % 16, columns
// 4 (lane / 16) on (the products are issued transposed).  Two neighbouring tiles are finished together: of 16-bit
// outputs the two first trade halves (v_permlane16_swap exchanges the odd lane groups of the first tile with the even
// ones of the second), after which a lane holds 8 consecutive columns, 16 bytes.
struct FfnPair {
  float x[2][4];
};
// Rows end at m, columns at n.  Addresses are aligned to the elements only: the part's vector stores take that.
__device__ __forceinline__ void ffn_store_pair(void *base, uint64_t ld, int type, uint32_t row, uint32_t col0, uint32_t lane, uint32_t m, uint32_t n,
                                               const FfnPair &v) {
  const uint32_t g = lane / 16u;
  if (type == MI355_TYPE_F32) {
    if (row < m) {
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const uint32_t col = col0 + 16u * t + 4u * g;
        float *to = static_cast<float *>(base) + (uint64_t)row * ld + col;
        if (col + 4u <= n) {
          __builtin_memcpy(__builtin_assume_aligned(to, 4), v.x[t], 16);
        } else {   // (a loop, so that this rare case stays short code)
          float x0 = v.x[t][0], x1 = v.x[t][1], x2 = v.x[t][2];
#pragma unroll 1
          for (uint32_t c = col; c < n; c++) {
            *to++ = x0;
            x0 = x1; x1 = x2;
          }
        }
      }
    }
    return;
  }
  uint32_t p[2][2];
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int h = 0; h < 2; h++)
      p[t][h] = type == MI355_TYPE_F16 ? mi355_pack_f16x2(v.x[t][2 * h], v.x[t][2 * h + 1]) : mi355_pack_bf16x2(v.x[t][2 * h], v.x[t][2 * h + 1]);
  const auto q01 = __builtin_amdgcn_permlane16_swap(p[0][0], p[1][0], false, false);
  const auto q23 = __builtin_amdgcn_permlane16_swap(p[0][1], p[1][1], false, false);
  const uint32_t w[4] = {q01[0], q23[0], q01[1], q23[1]};
  const uint32_t col = col0 + 16u * (g & 1u) + 8u * (g >> 1);
  if (row < m) {
    uint16_t *to = static_cast<uint16_t *>(base) + (uint64_t)row * ld + col;
    if (col + 8u <= n) {
      __builtin_memcpy(__builtin_assume_aligned(to, 2), w, 16);
    } else {   // (a loop, so that this rare case stays short code)
      uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
#pragma unroll 1
      for (uint32_t c = col; c < n; c++) {
        *to++ = (uint16_t)lo;
        lo = lo >> 16 | hi << 48;
        hi >>= 16;
      }
    }
  }
}

// Four neighbouring elements (the first `count` of them).
__device__ __forceinline__ void ffn_store4(void *base, uint64_t at, int type, const float (&x)[4], uint32_t count) {
  if (type == MI355_TYPE_F32) {
    float *to = static_cast<float *>(base) + at;
    if (count >= 4u) {
      __builtin_memcpy(__builtin_assume_aligned(to, 4), x, 16);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 3; e++)
        if (e < count) to[e] = x[e];
    }
    return;
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; h++) w[h] = type == MI355_TYPE_F16 ? mi355_pack_f16x2(x[2 * h], x[2 * h + 1]) : mi355_pack_bf16x2(x[2 * h], x[2 * h + 1]);
  uint16_t *to = static_cast<uint16_t *>(base) + at;
  if (count >= 4u) {
    __builtin_memcpy(__builtin_assume_aligned(to, 2), w, 8);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 3; e++)
      if (e < count) to[e] = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
  }
}

// One matrix instruction on 16-byte fragments, K half by K half; issued transposed (B first): a lane then holds 4
// consecutive columns of one row.
template <int OP>
__device__ __forceinline__ i32x4v ffn_mfma(const i32x4v &b, const i32x4v &a, const i32x4v &c) {
  if constexpr (OP == kQuadI8) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, c, 0, 0, 0);
  } else if constexpr (OP == kQuadBf16) {
    return __builtin_bit_cast(i32x4v, __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, b), __builtin_bit_cast(bf16x8v, a),
                                                                           __builtin_bit_cast(f32x4v, c), 0, 0, 0));
  } else {
    return __builtin_bit_cast(i32x4v, __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, b), __builtin_bit_cast(half8v, a),
                                                                          __builtin_bit_cast(f32x4v, c), 0, 0, 0));
  }
}

// The type of an output: that of 16-bit operands but for a slice's sums.
template <int OP, int EPI>
__device__ __forceinline__ int ffn_type_out(const FfnOut &o) {
  if (EPI == kEpiPartial || (EPI == kEpiPlain && o.type == MI355_TYPE_F32)) return MI355_TYPE_F32;
  return OP == kQuadBf16 ? MI355_TYPE_BF16 : OP == kQuadF16 ? MI355_TYPE_F16 : o.type;
}

// kEpiPlain: 32-bit sums (a slice's, and rows that are added later) are kept as they are.
__device__ __forceinline__ float ffn_plain_factor(const FfnOut &o) { return o.sa && o.type != MI355_TYPE_F32 ? *o.sa : 1.0f; }

// What a lane needs for its columns of a pair of tiles, and for a row.
template <int EPI>
struct FfnColumns {
  float sb[2][4], sb2[2][4], bias[2][4];
  float plain;   // (kEpiPlain of fp16)
  __device__ __forceinline__ void load(const FfnOut &o, uint32_t col0, uint32_t lane, uint32_t n) {
    if constexpr (EPI == kEpiScaled || EPI == kEpiGatedScaled) {
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t col = min(col0 + 16u * t + 4u * (lane / 16u) + e, n - 1u);
          sb[t][e] = o.sb[col];
          if constexpr (EPI == kEpiGatedScaled) sb2[t][e] = o.sb2[col];
          else bias[t][e] = o.bias ? o.bias[col] : 0.0f;
        }
    }
    if constexpr (EPI == kEpiPlain) plain = ffn_plain_factor(o);
  }
};

// A pair of finished tiles (gated: of the gate, s, and of the other product, s2), as raw bits of fp32 or int32.
template <int OP, int EPI>
__device__ __forceinline__ void ffn_finish_pair(const FfnOut &o, uint32_t row, uint32_t col0, uint32_t lane, uint32_t m, uint32_t n, float sa,
                                                const FfnColumns<EPI> &c, const i32x4v (&s)[2], const i32x4v (&s2)[2]) {
  const int type = ffn_type_out<OP, EPI>(o);
  FfnPair a, b;
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int32_t v = s[t][e], v2 = s2[t][e];   // (through a scalar: __builtin_bit_cast of a vector's element reads element 0)
      if constexpr (EPI == kEpiPartial) {
        a.x[t][e] = __builtin_bit_cast(float, v);
      } else if constexpr (OP == kQuadI8) {
        a.x[t][e] = EPI == kEpiScaled && o.bias ? ffn_scaled_plus(v, sa, c.sb[t][e], c.bias[t][e]) : ffn_scaled(v, sa, c.sb[t][e]);
        if constexpr (EPI == kEpiGatedScaled) b.x[t][e] = ffn_scaled(v2, sa, c.sb2[t][e]);
      } else {
        a.x[t][e] = __builtin_bit_cast(float, v);
        if constexpr (OP == kQuadF16 && EPI == kEpiPlain) a.x[t][e] *= c.plain;
        if constexpr (EPI == kEpiGated) b.x[t][e] = __builtin_bit_cast(float, v2);
      }
    }
  if constexpr (epi_is_gated(EPI)) {
    if constexpr (EPI == kEpiGated)
      if (o.g) {
        ffn_store_pair(o.g, o.ldg, type, row, col0, lane, m, n, a);
        ffn_store_pair(o.u, o.ldg, type, row, col0, lane, m, n, b);
      }
    // one branch on the activation for the 8 values
    if (o.act == MI355_GLU_SILU) {
#pragma unroll
      for (int i = 0; i < 8; i++) a.x[i / 4][i % 4] = ffn_act(MI355_GLU_SILU, a.x[i / 4][i % 4]) * b.x[i / 4][i % 4];
    } else if (o.act == MI355_GLU_GELU_TANH) {
#pragma unroll
      for (int i = 0; i < 8; i++) a.x[i / 4][i % 4] = ffn_act(MI355_GLU_GELU_TANH, a.x[i / 4][i % 4]) * b.x[i / 4][i % 4];
    } else if (o.act == MI355_GLU_GELU) {
#pragma unroll
      for (int i = 0; i < 8; i++) a.x[i / 4][i % 4] = ffn_act(MI355_GLU_GELU, a.x[i / 4][i % 4]) * b.x[i / 4][i % 4];
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) a.x[i / 4][i % 4] = ffn_act(MI355_GLU_RELU, a.x[i / 4][i % 4]) * b.x[i / 4][i % 4];
    }
  }
  ffn_store_pair(o.c, o.ldc, type, row, col0, lane, m, n, a);
}

// Four neighbouring columns of one row (of them, those below n) from their sums (gated: from both sums each).
template <int OP, int EPI>
__device__ __forceinline__ void ffn_finish4(const FfnOut &o, uint32_t row, uint32_t col, uint32_t n, const i32x4v &s, const i32x4v &s2) {
  if (col >= n) return;
  const int type = ffn_type_out<OP, EPI>(o);
  float x[4], y[4];
  float sa = EPI == kEpiScaled || EPI == kEpiGatedScaled ? o.sa[row] : 0.0f;
  if constexpr (OP == kQuadF16 && EPI == kEpiPlain) sa = ffn_plain_factor(o);
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int32_t v = s[e], v2 = s2[e];   // (through a scalar: __builtin_bit_cast of a vector's element reads element 0)
    const uint32_t c = min(col + e, n - 1u);
    if constexpr (EPI == kEpiScaled) {
      x[e] = o.bias ? ffn_scaled_plus(v, sa, o.sb[c], o.bias[c]) : ffn_scaled(v, sa, o.sb[c]);
    } else if constexpr (EPI == kEpiGatedScaled) {
      x[e] = ffn_scaled(v, sa, o.sb[c]);
      y[e] = ffn_scaled(v2, sa, o.sb2[c]);
    } else {
      x[e] = __builtin_bit_cast(float, v);
      y[e] = __builtin_bit_cast(float, v2);
      if constexpr (OP == kQuadF16 && EPI == kEpiPlain) x[e] *= sa;
    }
  }
  if constexpr (EPI == kEpiGated)
    if (o.g) {
      ffn_store4(o.g, (uint64_t)row * o.ldg + col, type, x, n - col);
      ffn_store4(o.u, (uint64_t)row * o.ldg + col, type, y, n - col);
    }
  if constexpr (epi_is_gated(EPI)) {
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = ffn_act(o.act, x[e]) * y[e];
  }
  ffn_store4(o.c, (uint64_t)row * o.ldc + col, type, x, n - col);
}

// One element of the output from its sum (gated: from its two sums), as raw bits of fp32 or int32.
template <int EPI>
__device__ __forceinline__ void ffn_finish1(const FfnOut &o, uint32_t row, uint32_t col, int32_t s0, int32_t s1) {
  const uint64_t at = (uint64_t)row * o.ldc + col;
  if constexpr (EPI == kEpiPlain) {
    ffn_store1(o.c, at, o.type, __builtin_bit_cast(float, s0) * ffn_plain_factor(o));
  } else if constexpr (EPI == kEpiScaled) {
    const float sa = o.sa[row], sb = o.sb[col];
    ffn_store1(o.c, at, o.type, o.bias ? ffn_scaled_plus(s0, sa, sb, o.bias[col]) : ffn_scaled(s0, sa, sb));
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
