// Products whose sum was cut into slices along K: the slices' sums, 32 bits each, are added in the order of the slices and
// finished.  int8 sums are exact however they are cut; fp32 ones depend on the cut, which depends on the sizes alone.
// Bound by the workspace it reads, 4 bytes per slice and output, and by being a launch (4 slices of 48x4096: 4.0 us).
#include "ffn.h"

namespace {

template <int OP, int EPI>
__global__ void __launch_bounds__(256) ffn_join_kernel(FfnOut o, const int32_t *partial, uint32_t slices, uint64_t ldp, uint32_t m, uint32_t n) {
  const uint64_t quads = (n + 3u) / 4u, at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  if (at >= quads * m) return;
  const uint32_t row = (uint32_t)(at / quads), col = (uint32_t)(at % quads) * 4u;
  const int32_t *from = partial + (uint64_t)row * ldp + col;
  i32x4v s = *reinterpret_cast<const i32x4v *>(from);
#pragma unroll 4
  for (uint32_t k = 1; k < slices; k++) {
    const i32x4v t = *reinterpret_cast<const i32x4v *>(from + (uint64_t)k * m * ldp);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int32_t x = s[e], y = t[e];
      if constexpr (OP == kQuadI8) s[e] = x + y;
      else s[e] = __builtin_bit_cast(int32_t, __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y));
    }
  }
  ffn_finish4<OP, EPI>(o, row, col, n, s, s);
}

template <int OP, int EPI>
int launch(mi355_dev *dev, const char *what, const FfnProduct &p, uint32_t slices, const void *workspace) {
  const uint64_t blocks = ((p.n + 3ull) / 4u * p.m + 255u) / 256u;
  MI355_REQUIRE(dev, blocks <= 0xffffffull, "%s: %u x %u outputs are more than one launch takes", what, p.m, p.n);
  ffn_join_kernel<OP, EPI><<<(uint32_t)blocks, 256, 0, dev->stream>>>(p.out, (const int32_t *)workspace, slices, mi355_ffn_slice_row(p.n), p.m, p.n);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}

}  // namespace

int mi355_launch_ffn_join(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p, uint32_t slices, const void *workspace) {
  if (op == kQuadI8 && epi == kEpiScaled) return launch<kQuadI8, kEpiScaled>(dev, what, p, slices, workspace);
  return op == kQuadBf16 ? launch<kQuadBf16, kEpiPlain>(dev, what, p, slices, workspace) : launch<kQuadF16, kEpiPlain>(dev, what, p, slices, workspace);
}
