// ffn_across.hip: products whose sum runs over the rows of B, and of A too where that is asked for.
#pragma once
#include "ffn.h"

// C[m][n] = sum over k of A * B[k][n], k = 0 .. 64 steps - 1, 16-bit operands, 256x256 tiles of sums.
//   B: up to four stretches of rows, one behind the other along k, each a multiple of 64 rows.
//   A: [m][k] (a row of k lda bytes apart from the next), or across: [k][parts x part], parts times m columns, each part
//      padded to `part` columns (a multiple of 64); part 0 is C's, part 1 that of c2.
// n is a multiple of 64; addresses and strides (bytes) are multiples of 16, strides at most 64 MiB.
struct FfnAcross {
  const uint8_t *a;
  uint64_t lda;
  uint32_t m, n, steps, parts, part, stretches;
  struct Stretch {
    const uint8_t *rows;
    uint32_t ld, slabs;   // (slabs of 64 rows)
  } b[4];
  FfnOut out;             // c, ldc, type
  void *c2;
  bool pairs;             // C is the sum of the upper and the lower half of the m rows
};
// slices > 1: the sum is cut into so many; then, and where C is one of pairs, `workspace` holds slices x parts matrices of m rows of n 32-bit sums, on 16 bytes.
int mi355_launch_ffn_across(mi355_dev *dev, int op, bool across_a, const char *what, const FfnAcross &p, uint32_t slices, uint8_t *workspace);

// How such a product is best launched (ffn.hip), and the time expected of it: the rows behind main_rows (if that is not 0)
// are a launch of their own; each launch in slices.
struct AcrossChoice {
  uint32_t main_rows, slices, rest_slices;
  double us;
};
AcrossChoice mi355_choose_ffn_across(const mi355_dev *dev, uint32_t m, uint32_t parts, uint32_t n, uint32_t steps);
