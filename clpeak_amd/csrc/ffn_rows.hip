// Products of few rows (generated tokens, one or some of each stream): every weight is read once and used for a handful
// of rows, so the time is that of reading the weights.
//
// A workgroup of eight waves owns 16 rows of B (gated: 16 of the gate's and the same 16 of the other projection's) and
// all rows of A (16 MT of them, at most 64), over the whole of K.  K is cut into windows of 128 bytes, which the waves
// take in turn: a wave reads its window's fragments straight from memory into registers (nothing is shared between the
// waves, so LDS would only add a trip), the workgroup's eight windows are 1 KiB of every row, and the waves' sums meet in
// LDS at the end, added in the order of the waves: results do not depend on timing.  No sum is split over workgroups:
// N = 4096 rows are 256 workgroups, one for each CU.
//
// Measured: the gated projection of one token, 2 x 8192 rows of 4096 bf16, 134 MB in 23.0 us (5.8 TB/s); gated 7 x 8192 x
// 4096 int8, 67 MB in 12.4 us (5.4 TB/s); 1x4096x4096 int8 5.4 us, on 64x64 tiles (ffn_mid.hip) 9.9 us.  With more rows the
// vector caches bound it: every workgroup reads all of A.
#include "ffn.h"

namespace {

constexpr int kRowWaves = 8, kRowThreads = 64 * kRowWaves;

// U windows: the fragments of both K halves (16 bytes at 16 * (lane / 16), and 64 bytes on).
template <int OP, int MT, int NB, int U>
struct RowStage {
  i32x4v a[U][MT][2], b[U][NB][2];
  // `at`: byte offset along K of window number i of this wave
  template <class At>
  __device__ __forceinline__ void load(const uint8_t *const (&pa)[MT], const uint8_t *const (&pb)[NB], uint32_t i, At at) {
#pragma unroll
    for (int k = 0; k < U; k++) {
      const uint32_t o = at(i + k);
#pragma unroll
      for (int j = 0; j < NB; j++)
#pragma unroll
        for (int h = 0; h < 2; h++) b[k][j][h] = *reinterpret_cast<const i32x4v *>(pb[j] + o + 64 * h);
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) a[k][t][h] = *reinterpret_cast<const i32x4v *>(pa[t] + o + 64 * h);
    }
    __builtin_amdgcn_sched_barrier(0);   // (the loads go out here, not where their values are needed)
  }
  __device__ __forceinline__ void multiply(i32x4v (&acc)[MT][NB], uint32_t windows = U) const {
#pragma unroll
    for (int k = 0; k < U; k++) {
      if ((uint32_t)k >= windows) break;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int j = 0; j < NB; j++) acc[t][j] = ffn_mfma<OP>(b[k][j][h], a[k][t][h], acc[t][j]);
    }
  }
};

// Windows per stage, two stages in flight: as many as leave room for the sums, and for one token few enough that two
// workgroups share a CU (1x16384x4096 int8: 13.1 us with two windows and 128 registers, 15.1 us with four and 154).
constexpr int rows_unroll(int mt, int nb) { return mt == 1 ? (nb == 1 ? 2 : 1) : mt == 4 || mt * nb > 4 ? (nb == 1 ? 2 : 1) : 2; }

template <int OP, int EPI, int MT>
__global__ void __launch_bounds__(kRowThreads, MT == 1 ? 4 : 2) ffn_rows_kernel(FfnProduct p) {
  constexpr int NB = epi_is_gated(EPI) ? 2 : 1;
  constexpr int U = rows_unroll(MT, NB);
  __shared__ int32_t sums[kRowWaves][MT][NB][16][16];   // [row][column]
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t r = lane % 16, g = lane / 16;
  const uint32_t tn = blockIdx.x, n0 = tn * 16u;

  // Rows past the last one are read as the last one; what they give is never stored.
  const uint8_t *pa[MT], *pb[NB];
#pragma unroll
  for (int i = 0; i < MT; i++) pa[i] = p.a + (uint64_t)min(16u * i + r, p.m - 1u) * p.lda + 16u * g;
  const uint64_t b_row = (uint64_t)min(n0 + r, p.n - 1u) * p.ldb + 16u * g;
  pb[0] = p.b + b_row;
  if constexpr (NB == 2) pb[1] = p.b2 + b_row;

  i32x4v acc[MT][NB];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NB; j++) acc[i][j] = (i32x4v){0, 0, 0, 0};

  // This wave's windows are numbers wave, wave + 8, .. of a walk over K that starts at a place of the workgroup's own: rows
  // are a power of two apart as a rule, and workgroups that all read the same few columns of their rows would all read
  // from the same few memory channels.
  const uint32_t windows = p.k_bytes / 128u, begin = (tn / 8u * kRowWaves + tn % 8u * (windows / 8u)) % windows;
  const uint32_t mine = wave < windows ? (windows - wave - 1u) / kRowWaves + 1u : 0u;
  auto at = [&](uint32_t i) {
    const uint32_t w = min(wave + kRowWaves * i, windows - 1u) + begin;   // (past the end: a window that is not multiplied)
    return (w >= windows ? w - windows : w) * 128u;
  };
  // Two stages of U windows, one in flight while the other is multiplied.
  RowStage<OP, MT, NB, U> s0, s1;
  if (mine > 0) {
    s0.load(pa, pb, 0, at);
    uint32_t i = 0;
    for (; i + 2 * U < mine; i += 2 * U) {
      s1.load(pa, pb, i + U, at);
      s0.multiply(acc);
      s0.load(pa, pb, i + 2 * U, at);
      s1.multiply(acc);
    }
    if (i + U < mine) {
      s1.load(pa, pb, i + U, at);
      s0.multiply(acc);
      s1.multiply(acc, mine - i - U);
    } else {
      s0.multiply(acc, mine - i);
    }
  }

#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NB; j++) *reinterpret_cast<i32x4v *>(&sums[wave][i][j][r][4 * g]) = acc[i][j];
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < MT * 256u; e += kRowThreads) {
    const uint32_t i = e / 256u, row = e / 16u % 16u, col = e % 16u;
    int32_t s[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < NB; j++) {
      if constexpr (OP == kQuadI8) {
#pragma unroll
        for (int v = 0; v < kRowWaves; v++) s[j] += sums[v][i][j][row][col];
      } else {
        float f = 0.0f;
#pragma unroll
        for (int v = 0; v < kRowWaves; v++) f += __builtin_bit_cast(float, sums[v][i][j][row][col]);
        s[j] = __builtin_bit_cast(int32_t, f);
      }
    }
    if (16u * i + row < p.m && n0 + col < p.n) ffn_finish1<EPI>(p.out, 16u * i + row, n0 + col, s[0], s[1]);
  }
}

template <int OP, int EPI, int MT>
int launch(mi355_dev *dev, const char *what, const FfnProduct &p) {
  ffn_rows_kernel<OP, EPI, MT><<<(p.n + 15u) / 16u, kRowThreads, 0, dev->stream>>>(p);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}
template <int OP, int EPI>
int launch_by_rows(mi355_dev *dev, const char *what, const FfnProduct &p) {
  if (p.m <= 16u) return launch<OP, EPI, 1>(dev, what, p);
  if (p.m <= 32u) return launch<OP, EPI, 2>(dev, what, p);
  if (p.m <= 48u) return launch<OP, EPI, 3>(dev, what, p);
  return launch<OP, EPI, 4>(dev, what, p);
}

}  // namespace

int mi355_launch_ffn_rows(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p) {
  if (op == kQuadI8) return epi == kEpiScaled ? launch_by_rows<kQuadI8, kEpiScaled>(dev, what, p) : launch_by_rows<kQuadI8, kEpiGatedScaled>(dev, what, p);
  if (op == kQuadBf16) return epi == kEpiPlain ? launch_by_rows<kQuadBf16, kEpiPlain>(dev, what, p) : launch_by_rows<kQuadBf16, kEpiGated>(dev, what, p);
  return epi == kEpiPlain ? launch_by_rows<kQuadF16, kEpiPlain>(dev, what, p) : launch_by_rows<kQuadF16, kEpiGated>(dev, what, p);
}
