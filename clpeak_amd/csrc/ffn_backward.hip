// The gradients of the gated projection.  dG and dU are one elementwise pass, the rest are products whose sums run over the
// rows of their operands: dX over F, the rows of the weights, dW over T, the rows of X and of dG, dU.
//
// Products of many tiles read such operands as they are (ffn_across.hip).  The others run on the kernels that want the
// sum's index innermost, together in one launch (or dX of few rows in one of its own), for which the pass that makes dG
// and dU writes them both ways and X and the weights are turned once into the workspace.  Which of these goes by the
// expected times: turning costs the products of a training batch (8192x8192x4096) 106 of 1585 us; one launch for all
// three products instead of one each takes a call of 1024x1024x1024 from 41.9 to 28.2 us, of 200x700x512 from 24.4 to 16.8,
// of 1009x2752x1024 from 55.0 to 51.4 (in graphs).  Either way the workspace's copies are padded with zeros
// to the kernels' 64 values of the sum, which is what lets T and F be anything.
//
// The pass that makes dG and dU rounds them to the operands' 16 bits, half a step each: what the matrix instructions take.
// Beside the rounding of the results it is the only one, and where there are many values their errors, independent and
// alike in size, add up to the root of two times a single one's.  Where there are few, two or three large ones can make
// that far more; there each is carried as two 16-bit values, its rounding and the rounding of what that leaves, as two
// rows: dW sums over both (X stands twice), dX is the sum of two rows of its product.  That is so for up to 2^15 values (of
// products of three normal values as many as some hundred alike), where it is the launch that adds the rows that takes
// time: 1x100x512 bf16 8.3 -> 10.2 us, 300x100x512 10.9 -> 14.5, 1x8192x4096 77.8 -> 79.5.
// The pass is bound by memory, 3 T F values read and 2 T F written (131 us at 8192x8192).
#include "ffn.h"
#include "ffn_across.h"
#include <algorithm>

namespace {

constexpr int kTileEdge = 64, kThreads = 256, kVec = 8;

__host__ __device__ constexpr uint64_t round_up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

constexpr uint64_t kFewValues = 1u << 15;

// The workspace: dG | dU by rows [Tp][2 Fk]; by columns 2 x [Fp][Tp] where dW wants that; the weights turned [D][2 Fk], or
// their last rows 2 x [64][D]; X turned [D][Tp], or its last rows [64][D] (where it stands twice, all of it [Tp][D]); and
// what the products use of it where they are cut along their sums.
struct Plan {
  bool twice;                                  // a value is two rows
  uint32_t rows_of;                            // T or 2 T
  uint64_t fk, fp, tp;                         // F padded to a row of a product, F padded to whole tiles, the rows padded to a row
  enum { kNone, kAcross, kOnRows, kGrouped } dx_on, dw_on;
  bool dx_across, dw_across;
  AcrossChoice dx, dw;
  FfnGroup group;                              // what goes together (dX first): sizes
  FfnGroupChoice grouped;
  uint64_t rows, cols, w, x, sums, bytes;      // offsets
};
Plan plan_of(const mi355_dev *dev, uint32_t T, uint32_t F, uint32_t D) {
  Plan p;
  p.fk = round_up(F, 64);
  p.fp = round_up(F, 256);
  p.twice = (uint64_t)T * F <= kFewValues;
  const uint32_t R = p.rows_of = p.twice ? 2u * T : T;
  p.tp = T ? round_up(R, 64) : 64;
  // across, or turned at the price of the copies' way through memory (4.5 bytes a picosecond)
  const uint32_t dx_k = (uint32_t)(4 * p.fk), dw_k = (uint32_t)(2 * p.tp);
  p.dx = mi355_choose_ffn_across(dev, T ? R : 1, 1, D, dx_k / 128u);
  if (p.twice) p.dx.main_rows = 0;
  p.dw = mi355_choose_ffn_across(dev, F, 2, D, dw_k / 128u);
  const double turn_dx = 8.0 * F * D / 4.5e6, turn_dw = (4.0 * R * F + 4.0 * R * D) / 4.5e6;
  const bool pinned = dev->gemm_tiling != MI355_GEMM_TILING_AUTO, pinned_256 = dev->gemm_tiling == MI355_GEMM_TILING_256;
  double least = 1e30;
  for (int on = 0; on < 6; on++) {
    const auto dx_on = !T ? Plan::kNone : on % 3 == 0 ? Plan::kAcross : on % 3 == 1 ? Plan::kOnRows : Plan::kGrouped;
    const auto dw_on = on / 3 ? Plan::kGrouped : Plan::kAcross;
    if (pinned && ((dx_on != Plan::kNone && (dx_on == Plan::kAcross) != pinned_256) || dx_on == Plan::kOnRows || (dw_on == Plan::kAcross) != pinned_256)) continue;
    FfnGroup g{};
    auto add = [&](uint32_t m, uint32_t k_bytes, bool pairs) {
      FfnGroup::One &o = g.of[g.count++];
      o.m = m; o.n = D; o.k_bytes = k_bytes; o.pairs = pairs;
    };
    double us = 1.5 * ((dx_on == Plan::kAcross || dx_on == Plan::kOnRows) + (dw_on == Plan::kAcross));   // (from a launch to the next)
    if (dx_on == Plan::kAcross) us += p.dx.us;
    else if (dx_on != Plan::kNone) us += turn_dx;
    if (dx_on == Plan::kOnRows) us += mi355_ffn_rows_us(dev, kEpiPlain, R, D, dx_k) + (p.twice ? 4.0 : 0.0);
    if (dx_on == Plan::kGrouped) add(R, dx_k, p.twice);
    if (dw_on == Plan::kAcross) us += p.dw.us;
    else us += turn_dw, add(F, dw_k, false), add(F, dw_k, false);
    FfnGroupChoice c{};
    if (g.count) c = mi355_choose_ffn_group(dev, g);
    us += c.us;
    if (us >= least) continue;
    least = us;
    p.dx_on = dx_on; p.dw_on = dw_on;
    p.group = g; p.grouped = c;
  }
  p.dx_across = p.dx_on == Plan::kAcross;
  p.dw_across = p.dw_on == Plan::kAcross;
  p.rows = 0;
  p.cols = round_up(p.rows + p.tp * 2 * p.fk * 2, 256);
  p.w = round_up(p.cols + (p.dw_across ? 0 : 2 * p.fp * p.tp * 2), 256);
  p.x = round_up(p.w + (p.dx_across ? 2 * 64 * (uint64_t)D * 2 : (uint64_t)D * 2 * p.fk * 2), 256);
  p.sums = round_up(p.x + (p.dw_across && !p.twice ? 64 * (uint64_t)D * 2 : (uint64_t)D * p.tp * 2), 256);
  auto sums = [&](uint32_t slices, uint64_t rows, bool pairs) { return slices > 1 || pairs ? slices * rows * D * 4 : 0; };
  uint64_t dx = 0, dw = 0;
  if (p.dx_across) dx = std::max(sums(p.dx.slices, p.dx.main_rows ? p.dx.main_rows : R, p.twice), p.dx.main_rows ? sums(p.dx.rest_slices, R - p.dx.main_rows, false) : 0);
  else if (p.dx_on == Plan::kOnRows) dx = sums(1, R, p.twice);
  if (p.dw_across) dw = sums(p.dw.slices, 2 * (uint64_t)F, false);
  const uint64_t group = p.group.count ? mi355_ffn_group_workspace(p.group, p.grouped) : 0;
  p.bytes = round_up(p.sums + std::max(std::max(dx, dw), group), 256);
  return p;
}

// A 64x64 tile of 16-bit values in LDS, written by rows and read by columns.
struct Tile {
  uint16_t at[kTileEdge][kTileEdge + 2];
};

struct Vec8 {
  uint16_t v[kVec];
};
// 8 values of a row from an address that is element-aligned only; past the end of the row: 0.
__device__ __forceinline__ Vec8 load8(const uint16_t *row, uint32_t at, uint32_t n) {
  Vec8 x;
  if (at + kVec <= n) {
    __builtin_memcpy(&x, row + at, sizeof(x));
  } else {
#pragma unroll
    for (int e = 0; e < kVec; e++) x.v[e] = at + e < n ? row[at + e] : 0;
  }
  return x;
}
template <int TYPE>
__device__ __forceinline__ float widen(uint16_t h) {
  if constexpr (TYPE == MI355_TYPE_F16) return (float)__builtin_bit_cast(_Float16, h);
  else return __builtin_bit_cast(float, (uint32_t)h << 16);
}
template <int TYPE>
__device__ __forceinline__ uint16_t narrow(float x) {
  return (uint16_t)(TYPE == MI355_TYPE_F16 ? mi355_pack_f16x2(x, 0.0f) : mi355_pack_bf16x2(x, 0.0f));
}

// What the rounding of x leaves of it, exactly; of what rounds to an infinity nothing.
template <int TYPE>
__device__ __forceinline__ float left_of(float x) {
  const float near = widen<TYPE>(narrow<TYPE>(x));
  return __builtin_isinf(near) ? 0.0f : x - near;
}

// Column c of the tile (8 of its values from row r on) to 16 bytes of dst.
__device__ __forceinline__ void store_column(const Tile &t, uint32_t c, uint32_t r, uint16_t *dst) {
  Vec8 x;
#pragma unroll
  for (int e = 0; e < kVec; e++) x.v[e] = t.at[r + e][c];
  *reinterpret_cast<uint4 *>(dst) = __builtin_bit_cast(uint4, x);
}

// What precedes the products, all of it one launch: the workgroups are tiles of 64x64 values, first those of dG and dU, then
// those of the matrices to be turned or whose last rows are to be copied.
struct Layout {
  const uint16_t *src;          // R rows of C values (C a multiple of 64), ld apart
  uint16_t *dst;                // turned: C rows of R values; otherwise R rows of C; zeros behind R, up to a multiple of 64
  uint64_t ld, ld_dst;
  uint32_t R, again, tiles_c, tiles;   // (from row `again` on: the first ones once more), C / 64, tiles in all
  bool turned;
};
struct Gate {
  const uint16_t *dH, *G, *U;
  uint64_t lddh, ldg;
  uint16_t *rows, *cols;
  uint32_t T, R, F, fk, tp;   // (R: T, or 2 T where the second T rows are what the rounding of the first ones left)
  uint64_t fp;
  int act;
  uint32_t tiles_f, tiles;
  bool by_rows, by_columns;
};

// dG and dU of a tile: by rows (dG at column f, dU at column fk + f of a row of 2 fk; zeros from F to fk and in the rows
// from R to tp) and by columns (row f of [fp][tp], dU fp rows on; zeros from R to tp).
template <int TYPE>
__device__ __forceinline__ void gate_tile(const Gate &p, uint32_t tile, Tile &tg, Tile &tu) {
  const uint32_t f0 = tile % p.tiles_f * kTileEdge, t0 = tile / p.tiles_f * kTileEdge;
  const uint32_t c = threadIdx.x % 8u * kVec, r0 = threadIdx.x / 8u;
#pragma unroll
  for (uint32_t r = r0; r < kTileEdge; r += kThreads / 8) {
    const uint32_t row = t0 + r, f = f0 + c;
    Vec8 dg{}, du{};
    if (row < p.R) {
      const bool left = row >= p.T;
      const uint32_t t = left ? row - p.T : row;
      const Vec8 h = load8(p.dH + (uint64_t)t * p.lddh, f, p.F), g = load8(p.G + (uint64_t)t * p.ldg, f, p.F), u = load8(p.U + (uint64_t)t * p.ldg, f, p.F);
#pragma unroll
      for (int e = 0; e < kVec; e++) {
        float a, da;
        ffn_act_grad(p.act, widen<TYPE>(g.v[e]), a, da);
        const float d = widen<TYPE>(h.v[e]);
        const float x = d * da * widen<TYPE>(u.v[e]), y = d * a;   // (past F: 0; da is at most 1.13: nothing overflows before the result does)
        dg.v[e] = narrow<TYPE>(left ? left_of<TYPE>(x) : x);
        du.v[e] = narrow<TYPE>(left ? left_of<TYPE>(y) : y);
      }
    }
    if (p.by_rows) {
      uint16_t *to = p.rows + (uint64_t)row * 2u * p.fk + f;
      *reinterpret_cast<uint4 *>(to) = __builtin_bit_cast(uint4, dg);
      *reinterpret_cast<uint4 *>(to + p.fk) = __builtin_bit_cast(uint4, du);
    }
    if (!p.by_columns) continue;
#pragma unroll
    for (int e = 0; e < kVec; e++) {
      tg.at[r][c + e] = dg.v[e];
      tu.at[r][c + e] = du.v[e];
    }
  }
  if (!p.by_columns) return;
  __syncthreads();
#pragma unroll
  for (uint32_t r = r0; r < kTileEdge; r += kThreads / 8) {   // r: a column of the tile, c: 8 of its rows
    if (f0 + r < p.F) {
      uint16_t *to = p.cols + (uint64_t)(f0 + r) * p.tp + t0 + c;
      store_column(tg, r, c, to);
      store_column(tu, r, c, to + p.fp * p.tp);
    }
  }
}

__device__ __forceinline__ void layout_tile(const Layout &p, uint32_t number, Tile &tile) {
  const uint32_t c0 = number % p.tiles_c * kTileEdge, r0 = number / p.tiles_c * kTileEdge;
  const uint32_t c = threadIdx.x % 8u * kVec;
#pragma unroll
  for (uint32_t r = threadIdx.x / 8u; r < kTileEdge; r += kThreads / 8) {
    Vec8 x{};
    const uint32_t row = r0 + r < p.again ? r0 + r : r0 + r - p.again;
    if (r0 + r < p.R) x = __builtin_bit_cast(Vec8, *reinterpret_cast<const uint4 *>(p.src + (uint64_t)row * p.ld + c0 + c));
    if (!p.turned) {
      *reinterpret_cast<uint4 *>(p.dst + (uint64_t)(r0 + r) * p.ld_dst + c0 + c) = __builtin_bit_cast(uint4, x);
      continue;
    }
#pragma unroll
    for (int e = 0; e < kVec; e++) tile.at[r][c + e] = x.v[e];
  }
  if (!p.turned) return;
  __syncthreads();
#pragma unroll
  for (uint32_t r = threadIdx.x / 8u; r < kTileEdge; r += kThreads / 8) store_column(tile, r, c, p.dst + (uint64_t)(c0 + r) * p.ld_dst + r0 + c);
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads) glu_backward_prepare_kernel(Gate gate, Layout l0, Layout l1, Layout l2) {
  __shared__ Tile a, b;
  uint32_t i = blockIdx.x;
  if (i < gate.tiles) return gate_tile<TYPE>(gate, i, a, b);
  i -= gate.tiles;
  if (i < l0.tiles) return layout_tile(l0, i, a);
  i -= l0.tiles;
  if (i < l1.tiles) return layout_tile(l1, i, a);
  layout_tile(l2, i - l1.tiles, a);
}

Layout turned(const void *src, uint64_t ld, uint8_t *dst, uint64_t ld_dst, uint32_t R, uint32_t again, uint64_t rp, uint32_t C) {
  Layout t;
  t.again = again;
  t.src = (const uint16_t *)src; t.dst = (uint16_t *)dst;
  t.ld = ld; t.ld_dst = ld_dst;
  t.R = R; t.tiles_c = C / 64u; t.tiles = (uint32_t)((uint64_t)t.tiles_c * (rp / 64u));
  t.turned = true;
  return t;
}
// The rows of [R][C] behind the last whole 64 (R = 0: none, 64 rows of zeros; no such rows: nothing to do).
Layout last_rows(const void *src, uint64_t ld, uint8_t *dst, uint32_t R, uint32_t C) {
  Layout t{};
  if (R > 0 && R % 64u == 0u) return t;
  t.src = (const uint16_t *)src + (uint64_t)(R / 64u * 64u) * ld; t.dst = (uint16_t *)dst;
  t.ld = ld; t.ld_dst = C;
  t.R = t.again = R % 64u; t.tiles_c = t.tiles = C / 64u;
  return t;
}
// All rows twice, as they are.
Layout all_twice(const void *src, uint64_t ld, uint8_t *dst, uint32_t T, uint64_t rp, uint32_t C) {
  Layout t = turned(src, ld, dst, C, 2u * T, T, rp, C);
  t.turned = false;
  return t;
}
// The same rows as stretches of B: the whole 64s where they are, then the copy.
void add_stretches(FfnAcross &q, const void *src, uint64_t ld, const uint8_t *copy, uint32_t R, uint32_t C) {
  if (R >= 64u) q.b[q.stretches++] = {(const uint8_t *)src, (uint32_t)(ld * 2u), R / 64u};
  if (R == 0 || R % 64u) q.b[q.stretches++] = {copy, C * 2u, 1};
}

}  // namespace

int mi355_glu_backward_limits(mi355_dev *dev, const char *what, uint32_t T, uint32_t F) {
  // T and 2 F are depths of products here: their rows are held to 64 MiB too
  MI355_REQUIRE(dev, T <= (32u << 20) && F <= (16u << 20) - 64u, "%s: T = %u, F = %u: at most 2^25 and 2^24 - 64 are taken", what, T, F);
  return MI355_OK;
}

size_t mi355_glu_backward_bytes(const mi355_dev *dev, uint32_t T, uint32_t F, uint32_t D) { return (size_t)plan_of(dev, T, F, D).bytes; }

int mi355_launch_glu_backward(mi355_dev *dev, int type, int act, const void *dH, uint64_t lddh, const void *X, uint64_t ldx, const void *Wg,
                              const void *Wu, uint64_t ldw, const void *G, const void *U, uint64_t ldg, void *dX, uint64_t lddx, void *dWg,
                              void *dWu, uint64_t lddw, uint32_t T, uint32_t F, uint32_t D, uint8_t *ws) {
  const Plan p = plan_of(dev, T, F, D);
  const int op = type == MI355_TYPE_BF16 ? kQuadBf16 : kQuadF16;
  const uint64_t tiles = p.fk / 64u * (p.tp / 64u) + (uint64_t)(D / 64u) * (2u * (p.fk / 64u) + p.tp / 64u);
  MI355_REQUIRE(dev, tiles <= 0xffffffull, "glu_backward: T = %u, F = %u, D = %u are more than one launch takes", T, F, D);
  uint8_t *const wu_copy = ws + p.w + (p.dx_across ? 64 * (uint64_t)D * 2 : p.fk * 2);
  Gate gate;
  gate.dH = (const uint16_t *)dH; gate.G = (const uint16_t *)G; gate.U = (const uint16_t *)U;
  gate.lddh = lddh; gate.ldg = ldg;
  gate.rows = (uint16_t *)(ws + p.rows); gate.cols = (uint16_t *)(ws + p.cols);
  gate.T = T; gate.R = p.rows_of; gate.F = F; gate.fk = (uint32_t)p.fk; gate.fp = p.fp; gate.tp = (uint32_t)p.tp; gate.act = act;
  gate.tiles_f = (uint32_t)(p.fk / 64u); gate.tiles = (uint32_t)(p.fk / 64u * (p.tp / 64u));
  gate.by_rows = dX || (dWg && p.dw_across); gate.by_columns = dWg && !p.dw_across;
  Layout wg{}, wu{}, x{};
  if (dX && p.dx_across) {
    wg = last_rows(Wg, ldw, ws + p.w, F, D);
    wu = last_rows(Wu, ldw, wu_copy, F, D);
  } else if (dX) {
    wg = turned(Wg, ldw, ws + p.w, 2 * p.fk, F, F, p.fk, D);
    wu = turned(Wu, ldw, wu_copy, 2 * p.fk, F, F, p.fk, D);
  }
  if (dWg && p.dw_across) x = p.twice && T ? all_twice(X, ldx, ws + p.x, T, p.tp, D) : last_rows(X, ldx, ws + p.x, T, D);
  else if (dWg) x = turned(X, ldx, ws + p.x, p.tp, p.rows_of, T, p.tp, D);
  const uint32_t grid = gate.tiles + wg.tiles + wu.tiles + x.tiles;
  if (type == MI355_TYPE_BF16) glu_backward_prepare_kernel<MI355_TYPE_BF16><<<grid, kThreads, 0, dev->stream>>>(gate, wg, wu, x);
  else glu_backward_prepare_kernel<MI355_TYPE_F16><<<grid, kThreads, 0, dev->stream>>>(gate, wg, wu, x);
  MI355_LAUNCH_CHECK(dev, "glu_backward (prepare)");
  FfnAcross c{};
  c.a = ws + p.rows; c.lda = 4 * p.fk;
  c.n = D;
  c.out.type = type;
  FfnGroup g{};           // the members of the planned group that are wanted
  FfnGroupChoice choice = p.grouped;
  g.type = type;
  uint32_t planned = 0;
  auto add = [&](bool wanted, const uint8_t *a, uint64_t lda, const uint8_t *b, uint64_t ldb, void *out, uint64_t ldc) {
    const FfnGroup::One &size = p.group.of[planned];
    if (wanted) {
      choice.slices[g.count] = p.grouped.slices[planned];
      FfnGroup::One &o = g.of[g.count++];
      o = size;
      o.a = a; o.lda = lda; o.b = b; o.ldb = ldb; o.c = out; o.ldc = ldc;
    }
    planned++;
  };
  if (p.dx_on == Plan::kGrouped) add(dX, ws + p.rows, 4 * p.fk, ws + p.w, 4 * p.fk, dX, lddx);
  if (p.dw_on == Plan::kGrouped) {
    add(dWg, ws + p.cols, 2 * p.tp, ws + p.x, 2 * p.tp, dWg, lddw);
    add(dWu, ws + p.cols + p.fp * p.tp * 2, 2 * p.tp, ws + p.x, 2 * p.tp, dWu, lddw);
  }
  if (dX && p.dx_across) {
    c.m = p.dx.main_rows ? p.dx.main_rows : p.rows_of; c.pairs = p.twice; c.steps = (uint32_t)(2 * p.fk / 64u); c.parts = 1; c.stretches = 0;
    add_stretches(c, Wg, ldw, ws + p.w, F, D);
    add_stretches(c, Wu, ldw, wu_copy, F, D);
    c.out.c = dX; c.out.ldc = lddx;
    if (int rc = mi355_launch_ffn_across(dev, op, false, "glu_backward (dX)", c, p.dx.slices, ws + p.sums)) return rc;
    if (p.dx.main_rows) {
      c.a += p.dx.main_rows * c.lda;
      c.m = T - p.dx.main_rows;
      c.out.c = (uint16_t *)dX + p.dx.main_rows * lddx;
      if (int rc = mi355_launch_ffn_across(dev, op, false, "glu_backward (dX)", c, p.dx.rest_slices, ws + p.sums)) return rc;
    }
  } else if (dX && p.dx_on == Plan::kOnRows) {
    FfnProduct q{};
    q.a = ws + p.rows; q.lda = 4 * p.fk;
    q.b = ws + p.w; q.ldb = 4 * p.fk;
    q.m = p.rows_of; q.n = D; q.k_bytes = (uint32_t)(4 * p.fk);
    q.out.c = dX; q.out.ldc = lddx; q.out.type = type;
    if (int rc = mi355_launch_ffn_rows(dev, op, kEpiPlain, "glu_backward (dX)", p.twice ? mi355_ffn_slices_of(q, ws + p.sums) : q)) return rc;
    FfnJoin join = mi355_ffn_join_of(q, 1, true, ws + p.sums);
    if (p.twice)
      if (int rc = mi355_launch_ffn_join(dev, op, kEpiPlain, "glu_backward (dX)", &join, 1)) return rc;
  }
  if (dWg && p.dw_across) {
    c.a = ws + p.rows;
    c.m = F; c.pairs = false; c.steps = (uint32_t)(p.tp / 64u); c.parts = 2; c.part = (uint32_t)p.fk; c.stretches = 0;
    if (p.twice && T) c.b[c.stretches++] = {ws + p.x, D * 2u, (uint32_t)(p.tp / 64u)};
    else add_stretches(c, X, ldx, ws + p.x, T, D);
    c.out.c = dWg; c.c2 = dWu; c.out.ldc = lddw;
    if (int rc = mi355_launch_ffn_across(dev, op, true, "glu_backward (dW)", c, p.dw.slices, ws + p.sums)) return rc;
  }
  return g.count ? mi355_ffn_group(dev, op, "glu_backward", g, choice, ws + p.sums) : MI355_OK;
}
