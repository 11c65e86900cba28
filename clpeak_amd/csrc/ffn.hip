// The entry points of the feed-forward products: their checks, and which kernel a product runs on.
#include "ffn.h"
#include "ffn_across.h"
#include <algorithm>
#include <cmath>

namespace {

constexpr uint32_t kMaxRows = 1u << 30, kMaxCols = 1u << 26;   // of a matrix: indices and a launch's threads stay within 32 bits
constexpr uint64_t kMaxRow = 64ull << 20;         // bytes between two rows of an operand (32-bit offsets within 64 rows)
constexpr uint64_t kMaxStride = 1ull << 40;       // elements between two rows of any other matrix

// An operand of a product: rows of K elements, `ld` apart.
int check_operand(mi355_dev *dev, const char *what, const char *name, const void *p, uint64_t ld, uint32_t k, uint32_t elem) {
  MI355_REQUIRE(dev, p, "%s: %s is null", what, name);
  MI355_REQUIRE(dev, ((uintptr_t)p & 15u) == 0, "%s: %s must be 16-byte aligned", what, name);
  MI355_REQUIRE(dev, ld >= k && ld <= kMaxRow / elem && ld * elem % 16u == 0, "%s: rows of %s are %llu elements apart: at least %u, a multiple of %u and at most 64 MiB are wanted",
                what, name, (unsigned long long)ld, k, 16u / elem);
  return MI355_OK;
}
// Any other matrix.
int check_matrix(mi355_dev *dev, const char *what, const char *name, const void *p, uint64_t ld, uint32_t cols, uint32_t elem) {
  MI355_REQUIRE(dev, p, "%s: %s is null", what, name);
  MI355_REQUIRE(dev, (uintptr_t)p % elem == 0, "%s: %s must be aligned to its elements of %u bytes", what, name, elem);
  MI355_REQUIRE(dev, ld >= cols && ld <= kMaxStride, "%s: rows of %s are %llu elements apart: at least %u are wanted", what, name, (unsigned long long)ld, cols);
  return MI355_OK;
}
int check_vector(mi355_dev *dev, const char *what, const char *name, const float *p) {
  MI355_REQUIRE(dev, p && (uintptr_t)p % 4u == 0, "%s: %s is null or not aligned to its elements", what, name);
  return MI355_OK;
}
int check_16bit(mi355_dev *dev, const char *what, int type, int act) {
  MI355_REQUIRE(dev, type == MI355_TYPE_BF16 || type == MI355_TYPE_F16, "%s: type %d is neither bf16 nor fp16", what, type);
  MI355_REQUIRE(dev, act >= MI355_GLU_SILU && act <= MI355_GLU_RELU, "%s: unknown activation %d", what, act);
  return MI355_OK;
}
// rows x cols outputs, sums over k.
int check_sizes(mi355_dev *dev, const char *what, uint32_t rows, uint32_t cols, uint32_t k, uint32_t elem) {
  MI355_REQUIRE(dev, cols > 0 && k > 0, "%s: empty problem", what);
  MI355_REQUIRE(dev, rows <= kMaxRows && cols <= kMaxCols, "%s: %u rows and %u columns: at most 2^30 and 2^26 are taken", what, rows, cols);
  MI355_REQUIRE(dev, (uint64_t)k * elem % 128u == 0 && (uint64_t)k * elem <= kMaxRow, "%s: sums over %u elements: a multiple of %u and at most 64 MiB are wanted", what, k, 128u / elem);
  return MI355_OK;
}

}  // namespace

// Which kernel: the one whose time, by what was measured of it, is least.  Each has its own limit.
//   rows   what the workgroups of one CU read, their weights and all rows of A each, at 33 KB a microsecond through
//          its vector cache, and what surrounds a walk; at least the weights at 5.5 TB/s from memory;
//   tiles  of 64x64, 128x128, 256x128 or 256x256 sums: rounds of tiles over the CUs, each the steps of K (128 bytes) times a step's
//          time and what surrounds the walk (the 256x256 tiles' workgroups go on to their next tile without a break).  A
//          step takes longer as the part fills up and its clock falls.  At least the time of the weights, more where CUs
//          are idle and fewer bytes are in flight.
// K in slices where the tiles leave CUs idle: shorter walks, for a second launch and the sums' way through memory.
// Rows that would make the CUs go round once more for a few tiles are a product of their own: 4099 x 8190 x 8192 int8 as
// 4096 rows in two full rounds of 256x256 tiles and 3 rows by themselves.
// mi355_gemm_tiling pins a tiling, whatever the number of rows.
namespace {

enum Kernel { kOnRows, kOn64, kOn128, kOn256x128, kOn256 };
struct Choice {
  Kernel kernel = kOn256;
  uint32_t slices = 1;
  double us = 1e30;
};
struct Tiling {
  Kernel kernel;
  int pin;
  double rows, cols, step_us, full_step_us, round_us, once_us, weights;   // (the weights' bytes per us)
};
constexpr Tiling kTilings[] = {{kOn64, MI355_GEMM_TILING_64, 64, 64, 0.20, 0.32, 4.0, 1.0, 5.5e6},
                               {kOn128, MI355_GEMM_TILING_128, 128, 128, 0.30, 0.47, 5.0, 0.0, 5.5e6},
                               {kOn256x128, MI355_GEMM_TILING_256X128, 256, 128, 0.55, 0.85, 7.0, 0.0, 4.5e6},
                               {kOn256, MI355_GEMM_TILING_256, 256, 256, 0.85, 1.30, 4.0, 10.0, 4.5e6}};
constexpr const Tiling &tiling_of(Kernel k) { return kTilings[k - kOn64]; }

constexpr uint32_t kMostSlices = 16;

double count_of_cus(const mi355_dev *dev) { return dev->props.num_cus > 0 ? dev->props.num_cus : 1; }
double columns_of_sums(int epi, uint32_t n) { return epi_is_gated(epi) ? 2.0 * n : (double)n; }

double tiling_us(const Tiling &t, double cus, uint32_t m, uint32_t n, double sums_n, uint32_t k_bytes, uint32_t slices) {
  const double steps = std::ceil(k_bytes / 128u / (double)slices), weights_us = sums_n * k_bytes / t.weights;
  const double tiles = std::ceil(m / t.rows) * std::ceil(sums_n / t.cols) * slices;
  const double busy = std::min(1.0, tiles / cus), rounds = std::ceil(tiles / cus);
  const double step = t.step_us + (t.full_step_us - t.step_us) * busy;
  double us = t.once_us + std::max(weights_us * (1.6 - 0.6 * busy) + t.round_us, rounds * (steps * step + t.round_us));
  if (slices > 1) us += 4.0 + (double)m * n * (slices * 8.0 + 2.0) / 4e6;
  return us;
}

Choice choose(const mi355_dev *dev, int epi, uint32_t m, uint32_t n, uint32_t k_bytes, bool can_slice) {
  const double cus = count_of_cus(dev), sums_n = columns_of_sums(epi, n);
  Choice best;
  auto take = [&](Kernel k, uint32_t slices, double us) {
    if (us < best.us) { best.kernel = k; best.slices = slices; best.us = us; }
  };
  const int pin = dev->gemm_tiling;
  if (pin == MI355_GEMM_TILING_AUTO) take(kOnRows, 1, mi355_ffn_rows_us(dev, epi, m, n, k_bytes));
  for (const Tiling &t : kTilings) {
    if (pin != MI355_GEMM_TILING_AUTO && pin != t.pin) continue;
    const uint32_t most = can_slice && epi == kEpiScaled && t.kernel != kOn256 ? kMostSlices : 1;
    for (uint32_t s = 1; s <= most && (s == 1 || s * 4u <= k_bytes / 128u); s++) take(t.kernel, s, tiling_us(t, cus, m, n, sums_n, k_bytes, s));
  }
  return best;
}

// A product as one launch, or (main_rows > 0) as two by rows, the first on 256x256 tiles.
struct Division {
  Choice whole, rest;
  uint32_t main_rows = 0;
  double us = 0.0;
};
Division divide(const mi355_dev *dev, int epi, uint32_t m, uint32_t n, uint32_t k_bytes, bool can_slice) {
  Division d;
  d.whole = choose(dev, epi, m, n, k_bytes, can_slice);
  d.us = d.whole.us;
  if (dev->gemm_tiling != MI355_GEMM_TILING_AUTO) return d;
  const double cus = count_of_cus(dev), sums_n = columns_of_sums(epi, n), tiles_n = std::ceil(sums_n / 256.0);
  const double rounds = std::ceil(std::ceil(m / 256.0) * tiles_n / cus);
  const double rows = std::floor((rounds - 1.0) * cus / tiles_n) * 256.0;   // in one round less
  if (rows < 256.0 || rows >= m) return d;
  const uint32_t main_rows = (uint32_t)rows;
  const Choice rest = choose(dev, epi, m - main_rows, n, k_bytes, can_slice);
  const double us = tiling_us(tiling_of(kOn256), cus, main_rows, n, sums_n, k_bytes, 1) + rest.us;
  if (us < d.us) { d.main_rows = main_rows; d.rest = rest; d.us = us; }
  return d;
}

size_t slices_bytes(const Choice &c, uint32_t m, uint32_t n) {
  return c.slices > 1 ? (size_t)(c.slices * (uint64_t)m * mi355_ffn_slice_row(n) * 4u) : 0;
}
size_t division_bytes(const Division &d, uint32_t m, uint32_t n) {
  return d.main_rows ? slices_bytes(d.rest, m - d.main_rows, n) : slices_bytes(d.whole, m, n);
}

int launch(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p, const Choice &c, void *workspace) {
  if (c.kernel == kOnRows) return mi355_launch_ffn_rows(dev, op, epi, what, p);
  if (c.kernel == kOn64) return mi355_launch_ffn_mid(dev, op, epi, what, p, c.slices, workspace);
  if (c.kernel == kOn256) return mi355_launch_ffn_quad(dev, op, epi, what, p);
  return mi355_launch_ffn_small(dev, op, epi, what, c.kernel == kOn256x128, p, c.slices, workspace);
}

}  // namespace

double mi355_ffn_rows_us(const mi355_dev *dev, int epi, uint32_t m, uint32_t n, uint32_t k_bytes) {
  if (m > 64u) return 1e30;
  const double a_rows = m <= 16u ? m : (m + 15u) / 16u * 16u, sums_n = columns_of_sums(epi, n);
  const double on_one_cu = std::ceil(std::ceil(n / 16.0) / count_of_cus(dev)), read = (16.0 * sums_n / n + a_rows) * k_bytes;
  return 2.5 + std::max(sums_n * k_bytes / 5.5e6, on_one_cu * (read / 3.3e4 + (m <= 16u ? 0.4 : 0.9)));
}

namespace {

// When the last of so many workgroups ends, each CU taking the next when it is done with one; the longest come first.
struct Workgroups {
  double count, us;
};
double last_end(double cus, Workgroups (&w)[3], uint32_t kinds) {
  std::sort(w, w + kinds, [](const Workgroups &a, const Workgroups &b) { return a.us > b.us; });
  struct { double at, cus; } busy[16] = {{0.0, cus}};   // (a kind splits one of them at most, and leaves the rest whole)
  uint32_t n = 1;
  double end = 0.0;
  for (uint32_t k = 0; k < kinds; k++) {
    double left = w[k].count;
    if (left > 8.0 * cus) {   // (many rounds: as many on every CU)
      const double whole = std::floor(left / cus) - 4.0;
      for (uint32_t i = 0; i < n; i++) busy[i].at += whole * w[k].us;
      left -= whole * cus;
    }
    while (left > 0.0) {
      uint32_t first = 0;
      for (uint32_t i = 1; i < n; i++)
        if (busy[i].at < busy[first].at) first = i;
      if (left < busy[first].cus && n < 16u) {
        busy[n++] = {busy[first].at, busy[first].cus - left};
        busy[first].cus = left;
      }
      busy[first].at += w[k].us;
      left -= busy[first].cus;
    }
  }
  for (uint32_t i = 0; i < n; i++) end = std::max(end, busy[i].at);
  return end;
}

}  // namespace

// Slices of about as many steps for all of them, so that no walk outlasts the others.
FfnGroupChoice mi355_choose_ffn_group(const mi355_dev *dev, const FfnGroup &g) {
  const double cus = count_of_cus(dev);
  FfnGroupChoice best{kOn128, {1, 1, 1}, 1e30};
  uint32_t longest = 1;
  for (uint32_t i = 0; i < g.count; i++) longest = std::max(longest, g.of[i].k_bytes / 128u);
  for (const Tiling &t : kTilings) {
    if (t.kernel == kOn256 || (dev->gemm_tiling != MI355_GEMM_TILING_AUTO && dev->gemm_tiling != t.pin)) continue;
    double weights_us = 0.0, tiles[3] = {};
    for (uint32_t i = 0; i < g.count; i++) {
      weights_us += (double)g.of[i].n * g.of[i].k_bytes / t.weights;
      tiles[i] = std::ceil(g.of[i].m / t.rows) * std::ceil(g.of[i].n / t.cols);
    }
    for (uint32_t s = 1; s <= kMostSlices && (s == 1 || s * 4u <= longest); s++) {
      FfnGroupChoice c{t.kernel, {1, 1, 1}, 0.0};
      Workgroups w[3] = {};
      double steps_of[3] = {}, join = 0.0;
      for (uint32_t i = 0; i < g.count; i++) {
        const uint32_t steps = g.of[i].k_bytes / 128u;
        c.slices[i] = std::max(1u, (steps * s + longest / 2u) / longest);
        while (c.slices[i] > 1u && c.slices[i] * 4u > steps) c.slices[i]--;
        if (c.slices[i] > 1u || g.of[i].pairs) join += (double)g.of[i].m * g.of[i].n * (c.slices[i] * 6.0 + 2.0) / 4e6;
        steps_of[i] = std::ceil(steps / (double)c.slices[i]);
      }
      double step = t.full_step_us, end = 0.0;
      for (int again = 0; again < 2; again++) {   // (a step is as long as the part is busy, over all of the launch)
        double work = 0.0;
        for (uint32_t i = 0; i < g.count; i++) {
          w[i] = {tiles[i] * c.slices[i], steps_of[i] * step + t.round_us};
          work += w[i].count * w[i].us;
        }
        end = last_end(cus, w, g.count);
        step = t.step_us + (t.full_step_us - t.step_us) * work / (cus * end);
      }
      c.us = t.once_us + std::max(weights_us, end) + (join > 0.0 ? 3.0 + join : 0.0);
      if (c.us < best.us) best = c;
    }
  }
  return best;
}

size_t mi355_ffn_group_workspace(const FfnGroup &g, const FfnGroupChoice &c) {
  uint64_t bytes = 0;
  for (uint32_t i = 0; i < g.count; i++)
    if (c.slices[i] > 1u || g.of[i].pairs) bytes += c.slices[i] * (uint64_t)g.of[i].m * mi355_ffn_slice_row(g.of[i].n) * 4u;
  return (size_t)bytes;
}

int mi355_ffn_lay_out_group(mi355_dev *dev, const char *what, FfnGroup &g, uint32_t rows, uint32_t cols, uint32_t &blocks) {
  std::stable_sort(g.of, g.of + g.count, [](const FfnGroup::One &a, const FfnGroup::One &b) { return a.k_bytes / a.slices > b.k_bytes / b.slices; });
  uint64_t first = 0;
  for (uint32_t i = 0; i < 3; i++) {
    FfnGroup::One &o = g.of[i];
    o.first = i < g.count ? (uint32_t)first : 0xffffffffu;
    if (i >= g.count) continue;
    const uint64_t tiles_m = (o.m + (uint64_t)rows - 1u) / rows, tiles_n = (o.n + (uint64_t)cols - 1u) / cols;
    MI355_REQUIRE(dev, tiles_m * tiles_n <= 0xffffffull && first + tiles_m * tiles_n * o.slices <= 0xffffffull, "%s: %u x %u outputs are more than one launch takes", what, o.m, o.n);
    o.tiles_m = (uint32_t)tiles_m; o.tiles_n = (uint32_t)tiles_n;
    first += tiles_m * tiles_n * o.slices;
  }
  blocks = (uint32_t)first;
  return MI355_OK;
}

int mi355_ffn_group(mi355_dev *dev, int op, const char *what, const FfnGroup &group, const FfnGroupChoice &c, uint8_t *workspace) {
  FfnGroup g = group;
  FfnJoin join[3];
  uint32_t joins = 0;
  for (uint32_t i = 0; i < g.count; i++) {
    FfnGroup::One &o = g.of[i];
    o.slices = c.slices[i];
    if (o.slices <= 1u && !o.pairs) continue;
    FfnProduct p{};
    p.m = o.m; p.n = o.n;
    p.out.c = o.c; p.out.ldc = o.ldc; p.out.type = g.type; p.out.sa = g.sa;
    join[joins++] = mi355_ffn_join_of(p, o.slices, o.pairs, workspace);
    o.c = workspace;
    o.ldc = mi355_ffn_slice_row(o.n);
    workspace += o.slices * (uint64_t)o.m * o.ldc * 4u;
  }
  if (int rc = c.kernel == kOn64 ? mi355_launch_ffn_mid_group(dev, op, what, g) : mi355_launch_ffn_small_group(dev, op, what, c.kernel == kOn256x128, g)) return rc;
  return joins ? mi355_launch_ffn_join(dev, op, kEpiPlain, what, join, joins) : MI355_OK;
}

AcrossChoice mi355_choose_ffn_across(const mi355_dev *dev, uint32_t m, uint32_t parts, uint32_t n, uint32_t steps) {
  const double cus = count_of_cus(dev);
  const Tiling &t = tiling_of(kOn256);
  auto best = [&](uint32_t rows, uint32_t &slices) {
    double least = 1e30;
    for (uint32_t s = 1; s <= 16u && (s == 1 || s * 4u <= steps); s++) {
      // (the parts' tiles side by side; rows of a tile that do not exist cost as much as others, but not the join)
      const double all = parts * std::ceil(rows / 256.0) * 256.0;
      const double us = tiling_us(t, cus, (uint32_t)all, n, n, steps * 128u, s) - (s > 1 ? (all - parts * (double)rows) * n * (s * 8.0 + 2.0) / 4e6 : 0.0);
      if (us < least) { least = us; slices = s; }
    }
    return least;
  };
  AcrossChoice c{0, 1, 1, 0.0};
  c.us = best(m, c.slices);
  const double tiles_n = std::ceil(n / 256.0), rounds = std::ceil(std::ceil(m / 256.0) * tiles_n / cus);
  const double rows = std::floor((rounds - 1.0) * cus / tiles_n) * 256.0;
  if (parts == 1 && rows >= 256.0 && rows < m) {
    uint32_t main_slices = 1, rest_slices = 1;
    const double us = best((uint32_t)rows, main_slices) + best(m - (uint32_t)rows, rest_slices);
    if (us < c.us) c = {(uint32_t)rows, main_slices, rest_slices, us};
  }
  return c;
}

size_t mi355_ffn_workspace(const mi355_dev *dev, int epi, uint32_t m, uint32_t n, uint32_t k_bytes) {
  return division_bytes(divide(dev, epi, m, n, k_bytes, true), m, n);
}

// The caller has checked everything.
int mi355_ffn_product(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p, void *workspace, size_t workspace_bytes) {
  Division d = divide(dev, epi, p.m, p.n, p.k_bytes, true);
  const size_t need = division_bytes(d, p.m, p.n);
  if (need > 0 && (!workspace || workspace_bytes < need)) d = divide(dev, epi, p.m, p.n, p.k_bytes, false);
  if (d.main_rows == 0) return launch(dev, op, epi, what, p, d.whole, workspace);
  FfnProduct first = p, rest = p;
  first.m = d.main_rows;
  const uint64_t elem = p.out.type == MI355_TYPE_F32 ? 4 : 2;
  rest.m = p.m - d.main_rows;
  rest.a += (uint64_t)d.main_rows * p.lda;
  rest.out.c = static_cast<uint8_t *>(p.out.c) + d.main_rows * p.out.ldc * elem;
  if (p.out.sa) rest.out.sa += d.main_rows;
  if (p.out.g) {
    rest.out.g = static_cast<uint8_t *>(p.out.g) + d.main_rows * p.out.ldg * elem;
    rest.out.u = static_cast<uint8_t *>(p.out.u) + d.main_rows * p.out.ldg * elem;
  }
  if (int rc = launch(dev, op, epi, what, first, Choice{}, nullptr)) return rc;
  return launch(dev, op, epi, what, rest, d.rest, workspace);
}

extern "C" int mi355_glu_forward(mi355_dev *dev, int type, int act, const void *X, uint64_t ldx, const void *Wg, const void *Wu, uint64_t ldw,
                                 void *H, uint64_t ldh, void *G, void *U, uint64_t ldg, uint32_t T, uint32_t F, uint32_t D) {
  MI355_HANDLE(dev);
  const char *what = "glu_forward";
  if (int rc = check_16bit(dev, what, type, act)) return rc;
  if (int rc = check_sizes(dev, what, T, F, D, 2)) return rc;
  if (T == 0) return MI355_OK;
  if (int rc = check_operand(dev, what, "X", X, ldx, D, 2)) return rc;
  if (int rc = check_operand(dev, what, "Wg", Wg, ldw, D, 2)) return rc;
  if (int rc = check_operand(dev, what, "Wu", Wu, ldw, D, 2)) return rc;
  if (int rc = check_matrix(dev, what, "H", H, ldh, F, 2)) return rc;
  MI355_REQUIRE(dev, (G != nullptr) == (U != nullptr), "%s: G and U are kept together or not at all", what);
  if (G) {
    if (int rc = check_matrix(dev, what, "G", G, ldg, F, 2)) return rc;
    if (int rc = check_matrix(dev, what, "U", U, ldg, F, 2)) return rc;
  }
  MI355_SET_DEVICE(dev);
  FfnProduct p{};
  p.a = (const uint8_t *)X; p.b = (const uint8_t *)Wg; p.b2 = (const uint8_t *)Wu;
  p.lda = ldx * 2; p.ldb = ldw * 2;
  p.m = T; p.n = F; p.k_bytes = D * 2;
  p.out.c = H; p.out.ldc = ldh; p.out.g = G; p.out.u = U; p.out.ldg = ldg; p.out.type = type; p.out.act = act;
  return mi355_ffn_product(dev, type == MI355_TYPE_BF16 ? kQuadBf16 : kQuadF16, kEpiGated, what, p, nullptr, 0);
}

extern "C" int mi355_glu_backward_workspace(mi355_dev *dev, uint32_t T, uint32_t F, uint32_t D, size_t *bytes) {
  MI355_HANDLE(dev);
  MI355_REQUIRE(dev, bytes, "glu_backward_workspace: null out pointer");
  *bytes = 0;
  if (int rc = check_sizes(dev, "glu_backward_workspace", T, F, D, 2)) return rc;
  if (int rc = mi355_glu_backward_limits(dev, "glu_backward_workspace", T, F)) return rc;
  *bytes = mi355_glu_backward_bytes(dev, T, F, D);
  return MI355_OK;
}

extern "C" int mi355_glu_backward(mi355_dev *dev, int type, int act, const void *dH, uint64_t lddh, const void *X, uint64_t ldx,
                                  const void *Wg, const void *Wu, uint64_t ldw, const void *G, const void *U, uint64_t ldg,
                                  void *dX, uint64_t lddx, void *dWg, void *dWu, uint64_t lddw, uint32_t T, uint32_t F, uint32_t D,
                                  void *workspace, size_t workspace_bytes) {
  MI355_HANDLE(dev);
  const char *what = "glu_backward";
  if (int rc = check_16bit(dev, what, type, act)) return rc;
  if (int rc = check_sizes(dev, what, T, F, D, 2)) return rc;
  if (int rc = mi355_glu_backward_limits(dev, what, T, F)) return rc;
  MI355_REQUIRE(dev, (dWg != nullptr) == (dWu != nullptr), "%s: dWg and dWu are computed together or not at all", what);
  if (T > 0) {
    if (int rc = check_matrix(dev, what, "dH", dH, lddh, F, 2)) return rc;
    if (int rc = check_matrix(dev, what, "G", G, ldg, F, 2)) return rc;
    if (int rc = check_matrix(dev, what, "U", U, ldg, F, 2)) return rc;
    if (dX) {
      if (int rc = check_operand(dev, what, "Wg", Wg, ldw, D, 2)) return rc;
      if (int rc = check_operand(dev, what, "Wu", Wu, ldw, D, 2)) return rc;
      if (int rc = check_matrix(dev, what, "dX", dX, lddx, D, 2)) return rc;
    }
    if (dWg)
      if (int rc = check_operand(dev, what, "X", X, ldx, D, 2)) return rc;
  }
  if (dWg) {
    if (int rc = check_matrix(dev, what, "dWg", dWg, lddw, D, 2)) return rc;
    if (int rc = check_matrix(dev, what, "dWu", dWu, lddw, D, 2)) return rc;
  }
  if (T == 0) dX = nullptr;   // no rows
  if (!dX && !dWg) return MI355_OK;
  MI355_REQUIRE(dev, workspace && ((uintptr_t)workspace & 255u) == 0, "%s: the workspace is null or not aligned to 256 bytes", what);
  const size_t need = mi355_glu_backward_bytes(dev, T, F, D);
  MI355_REQUIRE(dev, workspace_bytes >= need, "%s: a workspace of %zu bytes, %zu are needed", what, workspace_bytes, need);
  MI355_SET_DEVICE(dev);
  return mi355_launch_glu_backward(dev, type, act, dH, lddh, X, ldx, Wg, Wu, ldw, G, U, ldg, dX, lddx, dWg, dWu, lddw, T, F, D, (uint8_t *)workspace);
}

extern "C" int mi355_gemm_i8_scaled_workspace(mi355_dev *dev, uint32_t M, uint32_t N, uint32_t K, size_t *bytes) {
  MI355_HANDLE(dev);
  MI355_REQUIRE(dev, bytes, "gemm_i8_scaled_workspace: null out pointer");
  *bytes = 0;
  if (int rc = check_sizes(dev, "gemm_i8_scaled_workspace", M, N, K, 1)) return rc;
  if (M > 0) *bytes = mi355_ffn_workspace(dev, kEpiScaled, M, N, K);
  return MI355_OK;
}

// 128 * 128 * K stays below 2^31: no sum leaves int32.
constexpr uint32_t kMaxI8Depth = 130944;

extern "C" int mi355_gemm_i8_scaled(mi355_dev *dev, const int8_t *A, uint64_t lda, const int8_t *B, uint64_t ldb, const float *scale_a,
                                    const float *scale_b, const float *bias, int type, void *C, uint64_t ldc, uint32_t M, uint32_t N, uint32_t K,
                                    void *workspace, size_t workspace_bytes) {
  MI355_HANDLE(dev);
  const char *what = "gemm_i8_scaled";
  MI355_REQUIRE(dev, type == MI355_TYPE_BF16 || type == MI355_TYPE_F16 || type == MI355_TYPE_F32, "%s: unknown type %d", what, type);
  if (int rc = check_sizes(dev, what, M, N, K, 1)) return rc;
  MI355_REQUIRE(dev, K <= kMaxI8Depth, "%s: K is %u, sums of more than %u products may leave int32", what, K, kMaxI8Depth);
  if (M == 0) return MI355_OK;
  if (int rc = check_operand(dev, what, "A", A, lda, K, 1)) return rc;
  if (int rc = check_operand(dev, what, "B", B, ldb, K, 1)) return rc;
  if (int rc = check_vector(dev, what, "scale_a", scale_a)) return rc;
  if (int rc = check_vector(dev, what, "scale_b", scale_b)) return rc;
  MI355_REQUIRE(dev, (uintptr_t)bias % 4u == 0, "%s: the bias is not aligned to its elements", what);
  if (int rc = check_matrix(dev, what, "C", C, ldc, N, type == MI355_TYPE_F32 ? 4 : 2)) return rc;
  MI355_REQUIRE(dev, ((uintptr_t)workspace & 15u) == 0, "%s: the workspace must be 16-byte aligned", what);
  MI355_SET_DEVICE(dev);
  FfnProduct p{};
  p.a = (const uint8_t *)A; p.b = (const uint8_t *)B;
  p.lda = lda; p.ldb = ldb;
  p.m = M; p.n = N; p.k_bytes = K;
  p.out.c = C; p.out.ldc = ldc; p.out.sa = scale_a; p.out.sb = scale_b; p.out.bias = bias; p.out.type = type;
  return mi355_ffn_product(dev, kQuadI8, kEpiScaled, what, p, workspace, workspace_bytes);
}

extern "C" int mi355_glu_i8(mi355_dev *dev, int act, const int8_t *A, uint64_t lda, const int8_t *Bg, const int8_t *Bu, uint64_t ldb,
                            const float *scale_a, const float *scale_g, const float *scale_u, int type, void *H, uint64_t ldh,
                            uint32_t M, uint32_t F, uint32_t K) {
  MI355_HANDLE(dev);
  const char *what = "glu_i8";
  MI355_REQUIRE(dev, type == MI355_TYPE_BF16 || type == MI355_TYPE_F16 || type == MI355_TYPE_F32, "%s: unknown type %d", what, type);
  MI355_REQUIRE(dev, act >= MI355_GLU_SILU && act <= MI355_GLU_RELU, "%s: unknown activation %d", what, act);
  if (int rc = check_sizes(dev, what, M, F, K, 1)) return rc;
  MI355_REQUIRE(dev, K <= kMaxI8Depth, "%s: K is %u, sums of more than %u products may leave int32", what, K, kMaxI8Depth);
  if (M == 0) return MI355_OK;
  if (int rc = check_operand(dev, what, "A", A, lda, K, 1)) return rc;
  if (int rc = check_operand(dev, what, "Bg", Bg, ldb, K, 1)) return rc;
  if (int rc = check_operand(dev, what, "Bu", Bu, ldb, K, 1)) return rc;
  if (int rc = check_vector(dev, what, "scale_a", scale_a)) return rc;
  if (int rc = check_vector(dev, what, "scale_g", scale_g)) return rc;
  if (int rc = check_vector(dev, what, "scale_u", scale_u)) return rc;
  if (int rc = check_matrix(dev, what, "H", H, ldh, F, type == MI355_TYPE_F32 ? 4 : 2)) return rc;
  MI355_SET_DEVICE(dev);
  FfnProduct p{};
  p.a = (const uint8_t *)A; p.b = (const uint8_t *)Bg; p.b2 = (const uint8_t *)Bu;
  p.lda = lda; p.ldb = ldb;
  p.m = M; p.n = F; p.k_bytes = K;
  p.out.c = H; p.out.ldc = ldh; p.out.sa = scale_a; p.out.sb = scale_g; p.out.sb2 = scale_u; p.out.type = type; p.out.act = act;
  return mi355_ffn_product(dev, kQuadI8, kEpiGatedScaled, what, p, nullptr, 0);
}
