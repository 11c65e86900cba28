// Rows to int8 with a scale each:  scale[m] = amax / 127,  q[m][k] = 127 x[m][k] / amax to the nearest whole number
// (ties to even), amax the row's largest magnitude.
//
// The quotient is computed in fp32 (one fused product with 127 / amax; off by less than 2e-5) and rounded by adding
// 1.5 * 2^23, whose last bit is 1: the low byte of the sum is q.  Where that may be on the wrong side of the border between
// two whole numbers it is decided exactly, 254 |x| against (2k + 1) amax, both exact in fp64.
//   fp32: where a quotient is within 1e-4 of a border.
//   bf16, fp16: quotients that are not on a border are farther from it than the error.  With x = mx 2^s and amax = ma (mx,
// ma whole, below 2^11) a quotient of 1/2 or more has s >= -8 and is |254 mx 2^s - (2k + 1) ma| / (2 ma) from the border,
// that is at least 2^(s - 11), where the error is below 2^(s - 13).  On a border 127 mx 2^(s + 1) = (2k + 1) ma, 127 a
// prime: either 2k + 1 = 127, where the even neighbour is the larger one and 127 / amax rounded up gives it; or 127
// divides ma, and 127 / amax is exact where ma / 127 is a power of two.  The rows of what remains (amax = 127 c 2^n, c =
// 9 .. 15 but for powers of two) are decided exactly throughout.
// The result is the definition's for every finite input of every type.
//
// One pass over memory: a row is held in registers between the maximum and the rounding, 8 elements per lane and chunk.
// A row of up to 2048 elements belongs to one wave (no barrier, four rows per workgroup), a longer one to a workgroup of 4, 8
// or 16 waves; past 65536 elements the row is read again, from the caches.  Bound by the 2 (4) bytes read and the byte written:
// 8191 x 8200 bf16, 202 MB, in 34.7 us (5.8 TB/s); a single row 1.9 us.
#include "ffn.h"
#include <algorithm>

namespace {

constexpr int kVec = 8;

template <int TYPE> struct Elem { using type = uint16_t; };
template <> struct Elem<MI355_TYPE_F32> { using type = uint32_t; };

// 8 elements of a row, as their bits: 16-bit types two to a word.
template <int TYPE>
struct Chunk {
  static constexpr int kWords = TYPE == MI355_TYPE_F32 ? 8 : 4;
  uint32_t w[kWords];

  // From an address that is element-aligned only; past the end of the row: 0, which changes no maximum.
  __device__ __forceinline__ void load(const typename Elem<TYPE>::type *row, uint32_t at, uint32_t K) {
    if (at + kVec <= K) {
      __builtin_memcpy(w, row + at, sizeof(w));
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i++) w[i] = 0;
#pragma unroll
      for (int e = 0; e < kVec; e++) {
        if (at + e >= K) break;
        if constexpr (TYPE == MI355_TYPE_F32) w[e] = row[at + e];
        else w[e / 2] |= (uint32_t)row[at + e] << (16 * (e % 2));
      }
    }
  }
  __device__ __forceinline__ float value(int e) const {
    if constexpr (TYPE == MI355_TYPE_F32) return __builtin_bit_cast(float, w[e]);
    else if constexpr (TYPE == MI355_TYPE_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e / 2] >> (16 * (e % 2))));
    else return __builtin_bit_cast(float, e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
  }
  // The largest magnitude so far, as bits: whole numbers order them, infinities above every finite value and NaNs above
  // those, so one maximum also says whether the row is finite.  16-bit types: two maxima, one in each half.
  __device__ __forceinline__ uint32_t top(uint32_t t) const {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < kWords; i++) {
      if constexpr (TYPE == MI355_TYPE_F32)
        t = max(t, w[i] & 0x7fffffffu);
      else
        t = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, t), __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu)));
    }
    return t;
  }
};
// Bits of the largest magnitude of a row (its two halves joined) as fp32; not finite: 0x7f800000 or more.
template <int TYPE>
__device__ __forceinline__ uint32_t top_as_f32(uint32_t t) {
  if constexpr (TYPE == MI355_TYPE_F32) return t;
  t = max(t & 0xffffu, t >> 16);
  if constexpr (TYPE == MI355_TYPE_BF16) return t << 16;
  return t >= 0x7c00u ? 0x7f800000u : __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)t));
}

struct RowScale {
  float inv;      // 127 / amax, rounded up
  float amax;
  bool exactly;   // every quotient of the row is decided exactly
};

// From the largest magnitude of a row, finite.
template <int TYPE>
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale s;
  s.amax = amax;
  s.exactly = !(amax > 0x1p-118f);   // (127 / 2^-118 is below 2^125; zeros go there too)
  s.inv = s.exactly ? 0.0f : 127.0f / amax;
  const float over = fmaf(s.inv, amax, -127.0f);
  if (over < 0.0f && !s.exactly) s.inv = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, s.inv) + 1u);
  if constexpr (TYPE != MI355_TYPE_F32) {
    const uint32_t ma = (__builtin_bit_cast(uint32_t, amax) & 0x7fffffu | 0x800000u) >> 13;   // 11 bits (of bf16: 8, and zeros)
    if (ma % 127u == 0u && over != 0.0f) s.exactly = true;
  }
  return s;
}

constexpr float kRound = 12582912.0f;   // 1.5 * 2^23

// Decided by comparing 254 |x| with (2k + 1) amax.
__device__ __noinline__ uint32_t quantize_exactly(float x, float amax) {
  const double a = (double)fabsf(x) * 254.0, m = (double)amax;
  double k = floor(a / (2.0 * m));         // within one of the truth; the border above it is k + 1/2
  if (2.0 * k * m > a) k -= 1.0;
  const double border = (2.0 * k + 1.0) * m;
  const int q = (int)k + (a > border || (a == border && ((int)k & 1)) ? 1 : 0);
  return (uint32_t)(x < 0.0f ? -q : q);
}

// kv: columns written, K of them quantised, the rest 0.
template <int TYPE>
__device__ __forceinline__ void store8(int8_t *row, uint32_t at, uint32_t kv, const Chunk<TYPE> &c, const RowScale &s) {
  uint32_t q[kVec];
  float off = 0.0f;
#pragma unroll
  for (int e = 0; e < kVec; e++) {
    const float x = c.value(e), v = fmaf(x, s.inv, kRound);
    q[e] = __builtin_bit_cast(uint32_t, v);
    if constexpr (TYPE == MI355_TYPE_F32) off = fmaxf(off, fabsf(fmaf(x, s.inv, kRound - v)));
  }
  if (__builtin_expect(off > 0.4999f || s.exactly, 0)) {
#pragma unroll
    for (int e = 0; e < kVec; e++) q[e] = s.amax > 0.0f ? quantize_exactly(c.value(e), s.amax) : 0u;
  }
  // the low bytes of each four
  const uint32_t p0 = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u) | __builtin_amdgcn_perm(q[3], q[2], 0x04000c0cu);
  const uint32_t p1 = __builtin_amdgcn_perm(q[5], q[4], 0x0c0c0400u) | __builtin_amdgcn_perm(q[7], q[6], 0x04000c0cu);
  if (at + kVec <= kv) {
    const uint32_t p[2] = {p0, p1};
    __builtin_memcpy(row + at, p, kVec);
  } else {
    uint64_t rest = (uint64_t)p1 << 32 | p0;
    for (uint32_t k = at; k < kv; k++, rest >>= 8) row[k] = (int8_t)rest;
  }
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}

// LANES: lanes per row (a wave or the workgroup).  CH > 0: the row is at most CH chunks of LANES * 8 elements and is held in
// registers.  CH == 0: any length, read twice.
template <int TYPE, int LANES, int CH>
__global__ void __launch_bounds__(LANES > 64 ? LANES : 256) quantize_i8_kernel(const void *X, uint64_t ldx, int8_t *Q, uint64_t ldq, float *scale,
                                                               uint32_t M, uint32_t K, uint32_t kv) {
  using E = typename Elem<TYPE>::type;
  constexpr uint32_t kRows = LANES > 64 ? 1 : 4, kStep = LANES * kVec;
  const uint32_t lane = threadIdx.x % LANES;
  const uint32_t m = blockIdx.x * kRows + threadIdx.x / LANES;
  if (LANES == 64 && m >= M) return;   // (a whole wave; with one row per workgroup every row exists)
  const E *row = static_cast<const E *>(X) + (uint64_t)m * ldx;
  int8_t *out = Q + (uint64_t)m * ldq;

  Chunk<TYPE> x[CH ? CH : 1];
  uint32_t top = 0;
  if constexpr (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; c++) x[c].load(row, lane * kVec + c * kStep, K);
#pragma unroll
    for (int c = 0; c < CH; c++) top = x[c].top(top);
  } else {
    for (uint32_t at = lane * kVec; at < K; at += kStep) {
      x[0].load(row, at, K);
      top = x[0].top(top);
    }
  }
  top = wave_max(top_as_f32<TYPE>(top));
  if constexpr (LANES > 64) {
    __shared__ uint32_t tops[LANES / 64];
    if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LANES / 64; i++) top = max(top, tops[i]);
  }
  // a row that holds an infinity or a NaN has no scale: NaN, so that what is computed from it shows it; and zeros
  const bool finite = top < 0x7f800000u;
  const RowScale s = row_scale<TYPE>(finite ? __builtin_bit_cast(float, top) : 0.0f);
  if (lane == 0) scale[m] = finite ? s.amax / 127.0f : __builtin_nanf("");
  if constexpr (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; c++) store8<TYPE>(out, lane * kVec + c * kStep, kv, x[c], s);
    for (uint32_t at = lane * kVec + CH * kStep; at < kv; at += kStep)   // padding past what the registers held
      for (uint32_t k = at; k < at + kVec && k < kv; k++) out[k] = 0;
  } else {
    for (uint32_t at = lane * kVec; at < kv; at += kStep) {
      x[0].load(row, at, K);
      store8<TYPE>(out, at, kv, x[0], s);
    }
  }
}

template <int TYPE>
void launch(mi355_dev *dev, const void *X, uint64_t ldx, int8_t *Q, uint64_t ldq, float *scale, uint32_t M, uint32_t K, uint32_t kv) {
#define GO(lanes, ch) quantize_i8_kernel<TYPE, lanes, ch><<<lanes > 64 ? M : (M + 3u) / 4u, lanes > 64 ? lanes : 256, 0, dev->stream>>>(X, ldx, Q, ldq, scale, M, K, kv)
  if (K <= 512u) GO(64, 1);
  else if (K <= 1024u) GO(64, 2);
  else if (K <= 2048u) GO(64, 4);
  else if (K <= 4096u) GO(256, 2);
  else if (K <= 8192u) GO(256, 4);
  else if (K <= 16384u) GO(512, 4);
  else if (K <= 32768u) GO(1024, 4);
  else if (K <= 65536u) GO(1024, 8);
  else GO(1024, 0);
#undef GO
}

constexpr uint32_t kMaxLaunchRows = 1u << 21;   // (a launch has less than 2^32 threads, a row at most 1024)

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
  for (uint32_t m = 0; m < M; m += kMaxLaunchRows) {
    const uint32_t rows = std::min(M - m, kMaxLaunchRows);
    const uint8_t *x = static_cast<const uint8_t *>(X) + m * ldx * e;
    if (type == MI355_TYPE_BF16) launch<MI355_TYPE_BF16>(dev, x, ldx, Q + m * ldq, ldq, scale + m, rows, K, k_pad);
    else if (type == MI355_TYPE_F16) launch<MI355_TYPE_F16>(dev, x, ldx, Q + m * ldq, ldq, scale + m, rows, K, k_pad);
    else launch<MI355_TYPE_F32>(dev, x, ldx, Q + m * ldq, ldq, scale + m, rows, K, k_pad);
    MI355_LAUNCH_CHECK(dev, "quantize_i8");
  }
  return MI355_OK;
}
