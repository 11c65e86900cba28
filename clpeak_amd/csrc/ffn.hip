// The entry points of the feed-forward products: their checks, and which kernel a product runs on.
#include "ffn.h"

namespace {

constexpr uint32_t kMaxCount = 1u << 30;          // rows / columns of a matrix: indices and launches stay within 32 bits
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
  MI355_REQUIRE(dev, rows <= kMaxCount && cols <= kMaxCount, "%s: %u rows and %u columns: at most 2^30 of each are taken", what, rows, cols);
  MI355_REQUIRE(dev, (uint64_t)k * elem % 128u == 0 && (uint64_t)k * elem <= kMaxRow, "%s: sums over %u elements: a multiple of %u and at most 64 MiB are wanted", what, k, 128u / elem);
  return MI355_OK;
}

}  // namespace

// Which kernel.  Up to 64 rows the weights' bytes are the time: ffn_rows.hip.  Above, the two tilings by their measured
// time per step of K (0.85 us for a 256x256 tile of sums, 0.40 us for a 128x128 one, and some 5 us around the walk) and
// the rounds of tiles that the CUs have to make; slices of K where those leave CUs idle, at the price of a second launch
// and of the sums' way through memory.
namespace {

struct Choice {
  enum { kRows, kQuad, kSmall } kernel;
  uint32_t slices;
};
Choice choose(const mi355_dev *dev, int epi, uint32_t m, uint32_t n, uint32_t k_bytes, bool can_slice) {
  if (dev->gemm_tiling == MI355_GEMM_TILING_256) return {Choice::kQuad, 1};
  const bool pinned = dev->gemm_tiling == MI355_GEMM_TILING_128;
  if (m <= 64u && !pinned) return {Choice::kRows, 1};
  const uint64_t cus = dev->props.num_cus > 0 ? (uint64_t)dev->props.num_cus : 1u, steps = k_bytes / 128u;
  const uint64_t sums_n = epi_is_gated(epi) ? 2ull * n : n;
  const uint64_t big = ((m + 255ull) / 256u) * ((sums_n + 255u) / 256u), small = ((m + 127ull) / 128u) * ((sums_n + 127u) / 128u);
  auto rounds = [&](uint64_t tiles) { return (double)((tiles + cus - 1u) / cus); };
  const double big_us = rounds(big) * (double)steps * 0.85 + 6.0;
  double best = rounds(small) * (double)steps * 0.40 + 5.0;
  Choice c{Choice::kSmall, 1};
  if (can_slice && !epi_is_gated(epi)) {
    for (uint32_t s = 2; s <= 16u && s * 4u <= steps; s++) {
      const double us = rounds(small * s) * (double)((steps + s - 1u) / s) * 0.40 + 5.0 + 4.0 + (double)m * n * (s * 8.0 + 2.0) / 4e6;
      if (us < best) { best = us; c.slices = s; }
    }
  }
  if (big_us < best && !pinned) return {Choice::kQuad, 1};
  return c;
}

}  // namespace

size_t mi355_ffn_workspace(const mi355_dev *dev, int epi, uint32_t m, uint32_t n, uint32_t k_bytes) {
  const Choice c = choose(dev, epi, m, n, k_bytes, true);
  return c.slices > 1 ? (size_t)(c.slices * (uint64_t)m * mi355_ffn_slice_row(n) * 4u) : 0;
}

// The caller has checked everything.
int mi355_ffn_product(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p, void *workspace, size_t workspace_bytes) {
  Choice c = choose(dev, epi, p.m, p.n, p.k_bytes, true);
  if (c.slices > 1 && (!workspace || workspace_bytes < mi355_ffn_workspace(dev, epi, p.m, p.n, p.k_bytes))) c = choose(dev, epi, p.m, p.n, p.k_bytes, false);
  if (c.kernel == Choice::kRows) return mi355_launch_ffn_rows(dev, op, epi, what, p);
  if (c.kernel == Choice::kQuad) return mi355_launch_ffn_quad(dev, op, epi, what, p);
  return mi355_launch_ffn_small(dev, op, epi, what, p, c.slices, workspace);
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
  *bytes = mi355_glu_backward_bytes(T, F, D);
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
  const size_t need = mi355_glu_backward_bytes(T, F, D);
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
