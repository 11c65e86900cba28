// The gradients of the gated projection.  dG and dU are one elementwise pass, the rest are products whose sums run over the
// rows of their operands: dX over F, the rows of the weights, dW over T, the rows of X and of dG, dU.
//
// Products of many tiles read such operands as they are (ffn_across.hip).  The others run on the kernels that want the
// sum's index innermost, together in one launch (or dX of few rows in one of its own), for which the pass that makes dG
// and dU writes them both ways and X and the weights are turned once into the workspace.  Which of these goes by the
// expected times: turning costs the products of a training batch (8192x8192x4096) 106 of 1585 us; one launch for all
// three products instead of one each takes a call of 1024x1024x1024 from 41.9 to 28.2 us, of 200x700x512 from 24.4 to 16.8,
// of 1009x2752x1024 from 55.0 to 51.4 (in graphs; fp16's pass for the largest value is not in these).  Either way the
// workspace's copies are padded with zeros to the kernels' 64 values of the sum, which is what lets T and F be anything.
//
// The pass that makes dG and dU rounds them to the operands' 16 bits, half a step each: what the matrix instructions take.
// Beside the rounding of the results it is the only one, and where there are many values their errors, independent and
// alike in size, add up to the root of two times a single one's.  Where there are few, two or three large ones can make
// that far more; there each is carried as two 16-bit values, its rounding and the rounding of what that leaves, as two
// rows: dW sums over both (X stands twice), dX is the sum of two rows of its product.  That is so for up to 2^15 values (of
// products of three normal values as many as some hundred alike), where it is the launch that adds the rows that takes
// time: 1x100x512 bf16 8.3 -> 10.2 us, 300x100x512 10.9 -> 14.5, 1x8192x4096 77.8 -> 79.5.
// The pass is bound by memory, 3 T F values read and 2 T F written (126 us at 8192x8192).
//
// fp16 has five bits of exponent: dG and dU of a loss that is a mean over many tokens lie below its normal values, those of
// one that is scaled up may lie above its largest, where the results, sums with other factors, are in range.  They are
// therefore rounded after a power of two that brings the largest of them, finite ones, to 2^14 .. 2^15, and the products' sums
// are multiplied by its inverse: values down to 2^-28 of the largest keep all their bits, smaller ones are off by at
// most 2^-39 of it.  (One factor for both: dX sums over F and dW over T, so none for each row or column would do.)  Finding
// the largest is a pass of its own in front, 3 T F values read (90 us at 8192x8192, 4.5 TB/s and nearly as much arithmetic; 8
// at 1009x2752).  bf16 has the range of fp32 and needs none of this.
#include "ffn.h"
#include "ffn_across.h"
#include <algorithm>

namespace {

constexpr int kTileEdge = 64, kThreads = 256, kVec = 8, kLargestThreads = 512;   // (the latter: a row of a tile for every 8)

__host__ __device__ constexpr uint64_t round_up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

constexpr uint64_t kFewValues = 1u << 15;
constexpr uint32_t kLargest = 1024;   // workgroups that look for the largest value, at most

// The workspace: dG | dU by rows [Tp][2 Fk]; by columns 2 x [Fp][Tp] where dW wants that; the weights turned [D][2 Fk], or
// their last rows 2 x [64][D]; X turned [D][Tp], or its last rows [64][D] (where it stands twice, all of it [Tp][D]); and
// what the products use of it where they are cut along their sums; of fp16 the workgroups' largest values and the factor
// that undoes the scaling.
struct Plan {
  bool twice;                                  // a value is two rows
  uint32_t rows_of;                            // T or 2 T
  uint64_t fk, fp, tp;                         // F padded to a row of a product, F padded to whole tiles, the rows padded to a row
  enum { kNone, kAcross, kOnRows, kGrouped } dx_on, dw_on;
  bool dx_across, dw_across;
  AcrossChoice dx, dw;
  FfnGroup group;                              // what goes together (dX first): sizes
  FfnGroupChoice grouped;
  uint64_t rows, cols, w, x, sums, largest, bytes;   // offsets
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
  p.largest = round_up(p.sums + std::max(std::max(dx, dw), group), 256);
  p.bytes = p.largest + round_up((kLargest + 1) * 4, 256);
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
  uint32_t *largest;          // fp16: the bits of the largest finite values that workgroups have found, `found` of them,
  uint32_t found;             // and behind kLargest the factor that undoes the scaling
};

// 8 neighbours of a row, and dG and dU of them (past F: 0).
template <int TYPE>
struct GateIn {
  Vec8 h, g, u;
  __device__ __forceinline__ void load(const Gate &p, uint32_t t, uint32_t f) {
    h = load8(p.dH + (uint64_t)t * p.lddh, f, p.F);
    g = load8(p.G + (uint64_t)t * p.ldg, f, p.F);
    u = load8(p.U + (uint64_t)t * p.ldg, f, p.F);
  }
  __device__ __forceinline__ void values(int act, float (&x)[kVec], float (&y)[kVec]) const {
    // one branch on the activation for the 8 values
    auto with = [&](int act) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < kVec; e++) {
        float a, da;
        ffn_act_grad(act, widen<TYPE>(g.v[e]), a, da);
        const float d = widen<TYPE>(h.v[e]), v = widen<TYPE>(u.v[e]);
        // half of act' (which is at most 1.13) first times the larger of the other two, then the smaller: neither product
        // overflows, or falls below the normal values, unless the result does
        const bool d_first = fabsf(d) > fabsf(v);
        x[e] = 2.0f * (0.5f * da * (d_first ? d : v) * (d_first ? v : d));
        y[e] = d * a;
      }
    };
    if (act == MI355_GLU_SILU) with(MI355_GLU_SILU);
    else if (act == MI355_GLU_GELU_TANH) with(MI355_GLU_GELU_TANH);
    else if (act == MI355_GLU_GELU) with(MI355_GLU_GELU);
    else with(MI355_GLU_RELU);
  }
};

// The largest of a workgroup's values; every thread's once all have arrived.
template <int WAVES>
__device__ __forceinline__ uint32_t workgroup_max(uint32_t v, uint32_t (&of_wave)[WAVES]) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  if (threadIdx.x % 64u == 0u) of_wave[threadIdx.x / 64u] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; i++) v = max(v, of_wave[i]);
  return v;
}

// The largest finite magnitude of dG and dU, as bits (whole numbers order them), one for each workgroup.
__global__ void __launch_bounds__(kLargestThreads) glu_backward_largest_kernel(Gate p, uint32_t tiles) {
  __shared__ uint32_t of_wave[kLargestThreads / 64];
  float top = 0.0f;
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const uint32_t f = tile % p.tiles_f * kTileEdge + threadIdx.x % 8u * kVec, t0 = tile / p.tiles_f * kTileEdge + threadIdx.x / 8u;
    GateIn<MI355_TYPE_F16> in;
    in.load(p, min(t0, p.T - 1u), f);   // (the last row again changes nothing)
    float x[kVec], y[kVec];
    in.values(p.act, x, y);
    float here = 0.0f;   // (the larger of a number and a NaN is the number)
#pragma unroll
    for (int e = 0; e < kVec; e++) here = fmaxf(here, fmaxf(fabsf(x[e]), fabsf(y[e])));
    if (__builtin_expect(__builtin_isinf(here), 0)) {
      here = 0.0f;
#pragma unroll
      for (int e = 0; e < kVec; e++) {
        here = fmaxf(here, __builtin_isinf(x[e]) ? 0.0f : fabsf(x[e]));
        here = fmaxf(here, __builtin_isinf(y[e]) ? 0.0f : fabsf(y[e]));
      }
    }
    top = fmaxf(top, here);
  }
  const uint32_t all = workgroup_max(__builtin_bit_cast(uint32_t, top), of_wave);
  if (threadIdx.x == 0) p.largest[blockIdx.x] = all;
}
// The power of two that brings that value to 2^14 .. 2^15 (one below 2^-112: times 2^126), from its exponent; the inverse goes
// to memory for the launches that follow.
__device__ __forceinline__ float scale_for_f16(const Gate &p, uint32_t (&of_wave)[kThreads / 64]) {
  uint32_t top = 0;
  for (uint32_t i = threadIdx.x; i < p.found; i += kThreads) top = max(top, p.largest[i]);
  const uint32_t exponent = max(workgroup_max(top, of_wave) >> 23, 15u);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.largest[kLargest] = (exponent - 14u) << 23;
  return __builtin_bit_cast(float, (268u - exponent) << 23);
}

// dG and dU of a tile: by rows (dG at column f, dU at column fk + f of a row of 2 fk; zeros from F to fk and in the rows
// from R to tp) and by columns (row f of [fp][tp], dU fp rows on; zeros from R to tp).
template <int TYPE>
__device__ __forceinline__ void gate_tile(const Gate &p, uint32_t tile, float scale, Tile &tg, Tile &tu) {
  const uint32_t f0 = tile % p.tiles_f * kTileEdge, t0 = tile / p.tiles_f * kTileEdge;
  const uint32_t c = threadIdx.x % 8u * kVec, r0 = threadIdx.x / 8u;
#pragma unroll
  for (uint32_t r = r0; r < kTileEdge; r += kThreads / 8) {
    const uint32_t row = t0 + r, f = f0 + c;
    Vec8 dg{}, du{};
    if (row < p.R) {
      const bool left = row >= p.T;
      const uint32_t t = left ? row - p.T : row;
      float x[kVec], y[kVec];
      GateIn<TYPE> in;
      in.load(p, t, f);
      in.values(p.act, x, y);
#pragma unroll
      for (int e = 0; e < kVec; e++) {
        if constexpr (TYPE == MI355_TYPE_F16) { x[e] *= scale; y[e] *= scale; }
        dg.v[e] = narrow<TYPE>(left ? left_of<TYPE>(x[e]) : x[e]);
        du.v[e] = narrow<TYPE>(left ? left_of<TYPE>(y[e]) : y[e]);
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
  if (i < gate.tiles) {
    float scale = 1.0f;
    if constexpr (TYPE == MI355_TYPE_F16) {
      __shared__ uint32_t of_wave[kThreads / 64];
      scale = scale_for_f16(gate, of_wave);
    }
    return gate_tile<TYPE>(gate, i, scale, a, b);
  }
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
  gate.largest = (uint32_t *)(ws + p.largest); gate.found = 0;
  const float *const undo = type == MI355_TYPE_F16 ? (const float *)gate.largest + kLargest : nullptr;
  if (type == MI355_TYPE_F16 && T) {
    const uint32_t tiles_t = (T + 63u) / 64u, all = gate.tiles_f * tiles_t;
    gate.found = std::min(all, kLargest);
    glu_backward_largest_kernel<<<gate.found, kLargestThreads, 0, dev->stream>>>(gate, all);
    MI355_LAUNCH_CHECK(dev, "glu_backward (largest)");
  }
  const uint32_t grid = gate.tiles + wg.tiles + wu.tiles + x.tiles;
  if (type == MI355_TYPE_BF16) glu_backward_prepare_kernel<MI355_TYPE_BF16><<<grid, kThreads, 0, dev->stream>>>(gate, wg, wu, x);
  else glu_backward_prepare_kernel<MI355_TYPE_F16><<<grid, kThreads, 0, dev->stream>>>(gate, wg, wu, x);
  MI355_LAUNCH_CHECK(dev, "glu_backward (prepare)");
  FfnAcross c{};
  c.a = ws + p.rows; c.lda = 4 * p.fk;
  c.n = D;
  c.out.type = type; c.out.sa = undo;
  FfnGroup g{};           // the members of the planned group that are wanted
  FfnGroupChoice choice = p.grouped;
  g.type = type; g.sa = undo;
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
    q.out.c = dX; q.out.ldc = lddx; q.out.type = type; q.out.sa = undo;
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
