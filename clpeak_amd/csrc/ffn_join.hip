// Products whose sum was cut into slices along K: the slices' sums, 32 bits each, are added in the order of the slices and
// finished.  int8 sums are exact however they are cut; fp32 ones depend on the cut, which depends on the sizes alone.
// Bound by the workspace it reads, 4 bytes per slice and output, and by being a launch (4 slices of 48x4096: 4.0 us).
#include "ffn.h"

namespace {

template <int OP, int EPI>
__global__ void __launch_bounds__(256) ffn_join_kernel(FfnJoin j0, FfnJoin j1, FfnJoin j2) {
  FfnJoin j = j0;
  if (blockIdx.x >= j1.first) j = j1;
  if (blockIdx.x >= j2.first) j = j2;
  const uint64_t quads = (j.n + 3u) / 4u, at = (uint64_t)(blockIdx.x - j.first) * 256u + threadIdx.x;
  if (at >= quads * j.m) return;
  const uint32_t row = (uint32_t)(at / quads), col = (uint32_t)(at % quads) * 4u;
  const int32_t *from = j.partial + (uint64_t)row * j.ldp + col;
  i32x4v s = *reinterpret_cast<const i32x4v *>(from);
#pragma unroll 4
  for (uint32_t k = 1; k < j.slices; k++) {
    const i32x4v t = *reinterpret_cast<const i32x4v *>(from + (uint64_t)k * j.m * j.ldp);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int32_t x = s[e], y = t[e];
      if constexpr (OP == kQuadI8) s[e] = x + y;
      else s[e] = __builtin_bit_cast(int32_t, __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y));
    }
  }
  ffn_finish4<OP, EPI>(j.out, row, col, j.n, s, s);
}

template <int OP, int EPI>
void launch(mi355_dev *dev, const FfnJoin (&j)[3], uint32_t blocks) {
  ffn_join_kernel<OP, EPI><<<blocks, 256, 0, dev->stream>>>(j[0], j[1], j[2]);
}

}  // namespace

int mi355_launch_ffn_join(mi355_dev *dev, int op, int epi, const char *what, FfnJoin *parts, uint32_t count) {
  FfnJoin j[3] = {};
  uint64_t blocks = 0;
  for (uint32_t i = 0; i < 3; i++) {
    if (i < count) j[i] = parts[i];
    j[i].first = i < count ? (uint32_t)blocks : 0xffffffffu;
    if (i < count) blocks += ((j[i].n + 3ull) / 4u * j[i].m + 255u) / 256u;
    MI355_REQUIRE(dev, blocks <= 0xffffffull, "%s: %u x %u outputs are more than one launch takes", what, j[i].m, j[i].n);
  }
  if (op == kQuadI8 && epi == kEpiScaled) launch<kQuadI8, kEpiScaled>(dev, j, (uint32_t)blocks);
  else if (op == kQuadBf16) launch<kQuadBf16, kEpiPlain>(dev, j, (uint32_t)blocks);
  else launch<kQuadF16, kEpiPlain>(dev, j, (uint32_t)blocks);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}
