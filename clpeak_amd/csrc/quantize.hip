// Rows to int8 with a scale each:  scale[m] = amax / 127,  q[m][k] = 127 x[m][k] / amax to the nearest whole number
// (ties to even), amax the row's largest magnitude.
//
// The quotient is computed in fp32 (one product with 127 / amax) and is off by less than 4e-5 there, so it decides
// everything but values that close to the border between two whole numbers.  Those are decided exactly: 254 |x| against
// (2k + 1) amax, both exact in fp64.  The result is the definition's for every finite input of every type.
//
// One pass over memory: a row is held in registers between the maximum and the rounding, 8 elements per lane and chunk.
// A row of up to 2048 elements belongs to one wave (no barrier, four rows per workgroup), a longer one to a workgroup;
// past 16384 elements the row is read again, from the caches.  Bound by the 2 (4) bytes read and the byte written.
#include "ffn.h"

namespace {

constexpr int kThreads = 256, kVec = 8;

template <int TYPE> struct Elem { using type = uint16_t; };
template <> struct Elem<MI355_TYPE_F32> { using type = uint32_t; };

// 8 elements as fp32 from an address that is element-aligned only; past the end of the row: 0, which changes no maximum.
template <int TYPE>
__device__ __forceinline__ void load8(const typename Elem<TYPE>::type *row, uint32_t at, uint32_t K, float (&x)[kVec]) {
  typename Elem<TYPE>::type raw[kVec];
  if (at + kVec <= K) {
    __builtin_memcpy(raw, row + at, sizeof(raw));
  } else {
#pragma unroll
    for (int e = 0; e < kVec; e++) raw[e] = at + e < K ? row[at + e] : 0;
  }
#pragma unroll
  for (int e = 0; e < kVec; e++) {
    if constexpr (TYPE == MI355_TYPE_F32) x[e] = __builtin_bit_cast(float, raw[e]);
    else if constexpr (TYPE == MI355_TYPE_F16) x[e] = (float)__builtin_bit_cast(_Float16, raw[e]);
    else x[e] = __builtin_bit_cast(float, (uint32_t)raw[e] << 16);
  }
}

struct RowScale {
  float inv;      // 127 / amax
  double amax;
  float up;       // a power of two both are taken times, where 127 / amax would overflow
};

__device__ __forceinline__ int quantize1(float x, const RowScale &s) {
  const float xs = x * s.up, t = xs * s.inv, k = rintf(t);
  if (__builtin_expect(fabsf(t - k) < 0.4999f, 1)) return (int)k;
  const float low = floorf(fabsf(t) - 0.25f);   // the border is low + 0.5
  const double left = 254.0 * (double)fabsf(xs), border = (2.0 * (double)low + 1.0) * s.amax;
  const int q = (int)low + (left > border || (left == border && ((int)low & 1)) ? 1 : 0);
  return t < 0.0f ? -q : q;
}

// kv: columns written, K of them quantised, the rest 0.
__device__ __forceinline__ void store8(int8_t *row, uint32_t at, uint32_t K, uint32_t kv, const float (&x)[kVec], const RowScale &s, bool finite) {
  int8_t q[kVec];
#pragma unroll
  for (int e = 0; e < kVec; e++) q[e] = finite && at + e < K ? (int8_t)quantize1(x[e], s) : (int8_t)0;
  if (at + kVec <= kv) {
    __builtin_memcpy(row + at, q, kVec);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; e++)
      if (at + e < kv) row[at + e] = q[e];
  }
}

// The largest magnitude as bits of fp32: whole numbers order them, infinities above every finite value and NaNs above
// those, so one maximum also says whether the row is finite.
__device__ __forceinline__ uint32_t top8(uint32_t top, const float (&x)[kVec]) {
#pragma unroll
  for (int e = 0; e < kVec; e++) top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
  return top;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}

// LANES: lanes per row (a wave or the workgroup).  CH > 0: the row is at most CH chunks of LANES * 8 elements and is held in
// registers.  CH == 0: any length, read twice.
template <int TYPE, int LANES, int CH>
__global__ void __launch_bounds__(kThreads) quantize_i8_kernel(const void *X, uint64_t ldx, int8_t *Q, uint64_t ldq, float *scale,
                                                               uint32_t M, uint32_t K, uint32_t kv) {
  using E = typename Elem<TYPE>::type;
  constexpr uint32_t kRows = kThreads / LANES, kStep = LANES * kVec;
  const uint32_t lane = threadIdx.x % LANES;
  const uint32_t m = blockIdx.x * kRows + threadIdx.x / LANES;
  if (LANES == 64 && m >= M) return;   // (a whole wave; with one row per workgroup every row exists)
  const E *row = static_cast<const E *>(X) + (uint64_t)m * ldx;
  int8_t *out = Q + (uint64_t)m * ldq;

  float x[CH ? CH : 1][kVec];
  uint32_t top = 0;
  if constexpr (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; c++) load8<TYPE>(row, lane * kVec + c * kStep, K, x[c]);
#pragma unroll
    for (int c = 0; c < CH; c++) top = top8(top, x[c]);
  } else {
    for (uint64_t at = lane * kVec; at < K; at += kStep) {
      load8<TYPE>(row, (uint32_t)at, K, x[0]);
      top = top8(top, x[0]);
    }
  }
  top = wave_max(top);
  if constexpr (LANES > 64) {
    __shared__ uint32_t tops[kThreads / 64];
    if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  }
  const bool finite = top < 0x7f800000u;
  const float amax = __builtin_bit_cast(float, top);
  RowScale s;
  s.up = amax < 0x1p-64f ? 0x1p64f : 1.0f;
  s.amax = (double)(amax * s.up);
  s.inv = top ? 127.0f / (amax * s.up) : 0.0f;
  // a row that holds an infinity or a NaN has no scale: NaN, so that what is computed from it shows it
  if (lane == 0) scale[m] = finite ? amax / 127.0f : __builtin_nanf("");
  if constexpr (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; c++) store8(out, lane * kVec + c * kStep, K, kv, x[c], s, finite);
    for (uint64_t at = (uint64_t)lane * kVec + CH * kStep; at < kv; at += kStep) {   // padding past what the registers held
      const float none[kVec] = {};
      store8(out, (uint32_t)at, K, kv, none, s, false);
    }
  } else {
    for (uint64_t at = lane * kVec; at < kv; at += kStep) {
      load8<TYPE>(row, (uint32_t)at, K, x[0]);
      store8(out, (uint32_t)at, K, kv, x[0], s, finite);
    }
  }
}

template <int TYPE>
void launch(mi355_dev *dev, const void *X, uint64_t ldx, int8_t *Q, uint64_t ldq, float *scale, uint32_t M, uint32_t K, uint32_t kv) {
  const uint32_t by_wave = M / 4u + (M % 4u != 0u);
#define GO(lanes, ch, grid) quantize_i8_kernel<TYPE, lanes, ch><<<grid, kThreads, 0, dev->stream>>>(X, ldx, Q, ldq, scale, M, K, kv)
  if (K <= 512u) GO(64, 1, by_wave);
  else if (K <= 2048u) GO(64, 4, by_wave);
  else if (K <= 4096u) GO(256, 2, M);
  else if (K <= 8192u) GO(256, 4, M);
  else if (K <= 16384u) GO(256, 8, M);
  else GO(256, 0, M);
#undef GO
}

}  // namespace

extern "C" int mi355_quantize_i8(mi355_dev *dev, int type, const void *X, uint64_t ldx, int8_t *Q, uint64_t ldq, float *scale,
                                 uint32_t M, uint32_t K, uint32_t k_pad) {
  MI355_HANDLE(dev);
  MI355_REQUIRE(dev, type == MI355_TYPE_BF16 || type == MI355_TYPE_F16 || type == MI355_TYPE_F32, "quantize_i8: unknown type %d", type);
  MI355_REQUIRE(dev, K > 0, "quantize_i8: empty rows");
  MI355_REQUIRE(dev, K <= 0x40000000u && k_pad >= K && k_pad <= 0x40000000u, "quantize_i8: %u columns written from rows of %u (at most 2^30)", k_pad, K);
  MI355_REQUIRE(dev, ldx >= K && ldq >= k_pad, "quantize_i8: rows of %u / %u elements do not fit strides of %llu / %llu", K, k_pad,
                (unsigned long long)ldx, (unsigned long long)ldq);
  MI355_REQUIRE(dev, ldx <= (1ull << 40) && ldq <= (1ull << 40) && M <= 0x7fffffffu, "quantize_i8: strides of %llu / %llu elements or %u rows are too many",
                (unsigned long long)ldx, (unsigned long long)ldq, M);
  if (M == 0) return MI355_OK;
  MI355_REQUIRE(dev, X && Q && scale, "quantize_i8: null buffer");
  const uintptr_t e = type == MI355_TYPE_F32 ? 4 : 2;
  MI355_REQUIRE(dev, (uintptr_t)X % e == 0 && (uintptr_t)scale % 4 == 0, "quantize_i8: X and the scales must be aligned to their elements");
  MI355_SET_DEVICE(dev);
  if (type == MI355_TYPE_BF16) launch<MI355_TYPE_BF16>(dev, X, ldx, Q, ldq, scale, M, K, k_pad);
  else if (type == MI355_TYPE_F16) launch<MI355_TYPE_F16>(dev, X, ldx, Q, ldq, scale, M, K, k_pad);
  else launch<MI355_TYPE_F32>(dev, X, ldx, Q, ldq, scale, M, K, k_pad);
  MI355_LAUNCH_CHECK(dev, "quantize_i8");
  return MI355_OK;
}
