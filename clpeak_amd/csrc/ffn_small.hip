// The feed-forward products on the schedule of gemm_small.hip: a workgroup of four waves and one 128x128 tile of sums, for
// products that have too few 256x256 ones, or one of 256x128 (MI = 8, a wave 128x64), for those that have less than one of
// 256x256 for each CU and more than one of 128x128: of the same sums a tall tile reads a quarter less.  Operands may end
// inside a tile (ffn_quad.hip says how), and for the gated projection the tile's rows of B are 32 of the gate's weights,
// the same 32 of the other projection's, and again 32 and 32: a wave fetches one matrix's and owns 32 channels of both.
//
// Where even these tiles are few and K is long, K is cut into slices, a workgroup for each tile and slice; the sums of a
// slice go to the workspace as they are and a second launch (ffn_join.hip) adds the slices and finishes.  The plain
// products of 16-bit operands come in groups of up to three, whose workgroups are one launch.
//
// Measured: 512x8192x4096 int8 22.1 us (on 64x64 tiles 42.6, on 256x256 40.8); the gated projection 333x2731x1024 bf16 10.4 us
// (20.2, 25.8), 512x8192x4096 bf16 on tall tiles 56.3 us (on 128x128 75.5, on 256x256 81.4), 1000x8192x8192 int8 60.4 us (66.0,
// 73.3).  Few tiles: bound by the walk along K, 0.3 us a step (tall 0.55 to 0.85), and 5 us for its start and the sums'
// way out.
#include "ffn.h"
#include "gemm_small_step.h"

namespace {

template <int OP, int EPI, int I, int JP>
__device__ __forceinline__ void finish_tiles(const FfnProduct &p, uint32_t row0, uint32_t col0, uint32_t lane, const FfnColumns<EPI> &c) {
  const uint32_t row = row0 + 16u * I;
  float sa = 0.0f;
  if constexpr (EPI == kEpiScaled || EPI == kEpiGatedScaled) sa = p.out.sa[min(row, p.m - 1u)];
  const i32x4v s[2] = {small_take_tile<I * 4 + JP>(), small_take_tile<I * 4 + JP + 1>()};
  if constexpr (epi_is_gated(EPI)) {
    const i32x4v s2[2] = {small_take_tile<I * 4 + 2>(), small_take_tile<I * 4 + 3>()};
    ffn_finish_pair<OP, EPI>(p.out, row, col0, lane, p.m, p.n, sa, c, s, s2);
  } else {
    ffn_finish_pair<OP, EPI>(p.out, row, col0 + 16u * JP, lane, p.m, p.n, sa, c, s, s);
  }
}
template <int OP, int EPI, int JP, int... I>
__device__ __forceinline__ void finish_columns(std::integer_sequence<int, I...>, const FfnProduct &p, uint32_t row0, uint32_t col0, uint32_t lane) {
  FfnColumns<EPI> c;
  c.load(p.out, col0 + 16u * JP, lane, p.n);
  (finish_tiles<OP, EPI, I, JP>(p, row0, col0, lane, c), ...);
}
template <int MI, class Walk, int... Q>
__device__ __forceinline__ void load_slab(std::integer_sequence<int, Q...>, const Walk &w) { (small_load<Q, MI>(w), ...); }
template <int MI, int... R>
__device__ __forceinline__ void read_slab(std::integer_sequence<int, R...>, SmallFragsOf<MI> &f, const SmallEdgeWalk<MI> &w) { (small_read<R, MI>(f, w), ...); }

template <int OP, int EPI, int MI>
__global__ void __launch_bounds__(kSmallThreads) ffn_small_kernel(FfnLaunch<EPI> args) {
  const FfnWork work = args.work();
  const FfnProduct &p = work.p;
  constexpr bool kGated = epi_is_gated(EPI);
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const uint32_t tid = threadIdx.x, lane = tid % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const uint32_t wm = wave / 2, wn = wave % 2;
  TileGrid grid;
  grid.tiles_m = work.tiles_m; grid.tiles_n = work.tiles_n; grid.total = grid.stride = work.tiles_m * work.tiles_n;
  grid.first = work.tile; grid.mine = 1;
  uint32_t tm, tn;
  ffn_tile_at(grid, 0, tm, tn);
  uint32_t steps = p.k_bytes / kRowBytes, k0 = 0;
  if constexpr (EPI == kEpiPlain || EPI == kEpiPartial) {   // (at most 2^19 steps and 16 slices)
    const uint32_t all = steps;
    k0 = all * work.slice / work.slices;
    steps = all * (work.slice + 1u) / work.slices - k0;
  }
  const uint32_t lda = (uint32_t)p.lda, ldb = (uint32_t)p.ldb;
  using Ring = SmallRing<MI>;
  auto after = [](uint32_t slot_off) { return slot_off + Ring::kSlot == Ring::kBytes ? 0u : slot_off + Ring::kSlot; };

  // global -> LDS: wave w fills rows [8 MI w, 8 MI (w + 1)) of the A slab and [32w, 32w+32) of the B slab, 8 rows per
  // instruction; lane i is position i%8 of row i/8, which holds logical chunk (i%8) ^ (i/8)
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  const uint32_t dst_wave = __builtin_amdgcn_readfirstlane(lds_base + wave * 8u * MI * (uint32_t)kRowBytes);
  const uint32_t dst_wave_b = __builtin_amdgcn_readfirstlane(lds_base + wave * 32u * (uint32_t)kRowBytes);
  std::conditional_t<MI == 4, SmallEdgeWalk<4>, SmallTallWalk> w;
  const uint32_t a_row = min(tm * Ring::kRows + wave * 8u * MI, p.m - 1u);
  const uint32_t b_row = min(kGated ? tn * 64u + wave / 2u * 32u : tn * 128u + wave * 32u, p.n - 1u);
  const uint8_t *b = kGated && (wave & 1u) ? p.b2 : p.b;
#pragma unroll
  for (uint32_t q = 0; q < MI; q++) {
    const uint32_t chunk = ((lane % 8u) ^ (lane / 8u)) * 16u;
    w.voff[q] = min(lane / 8u + 8u * q, p.m - 1u - a_row) * lda + chunk;
    if (q < 4u) w.voff_b[q] = min(lane / 8u + 8u * q, p.n - 1u - b_row) * ldb + chunk;
  }
  // the walk over K starts at a place of the XCD's own (ffn_rows.hip says why) and wraps around
  const uint32_t k_rot = work.tile % 8u * (steps / 8u);
  w.ga = (uint64_t)(uintptr_t)(p.a + (uint64_t)a_row * lda + (uint64_t)(k0 + k_rot) * kRowBytes);
  w.gb = (uint64_t)(uintptr_t)(b + (uint64_t)b_row * ldb + (uint64_t)(k0 + k_rot) * kRowBytes);
  uint32_t fetch_left = steps - k_rot, fill = 0, look = 0;   // slot offsets: the one to fill, the one to read
  auto fetched = [&]() {                             // on to the next slab; past the last one: the first again
    w.ga += kRowBytes;
    w.gb += kRowBytes;
    if (--fetch_left == 0u) { w.ga -= (uint64_t)steps * kRowBytes; w.gb -= (uint64_t)steps * kRowBytes; fetch_left = steps; }
    fill = after(fill);
  };
  const uint32_t swz0 = ((lane / 16u) ^ (lane & 7u)) << 4;
  const uint32_t lane_a = lds_base + (wm * 16u * MI + lane % 16u) * kRowBytes + swz0;
  const uint32_t lane_b = lds_base + Ring::kSlabA + (wn * 64u + lane % 16u) * kRowBytes + swz0;
  auto place = [&]() {
    w.a0 = lane_a + look; w.a1 = w.a0 ^ 64u;
    w.b0 = lane_b + look; w.b1 = w.b0 ^ 64u;
    w.dst = dst_wave + fill;
    if constexpr (MI == 8) w.dst_b = dst_wave_b + fill;
  };

  small_claim_accumulators<MI>();
  small_zero_accumulators(std::make_integer_sequence<int, 4 * Ring::kTiles>{});

  // the first slabs into the slots; the fragments of slab 0
  for (uint32_t d = 0; d < Ring::kAhead; d++) {
    place();
    load_slab<MI>(std::make_integer_sequence<int, Ring::kLoads>{}, w);
    fetched();
  }
  asm volatile("s_waitcnt vmcnt(%0)\n s_barrier" :: "n"(Ring::kLoads * (Ring::kAhead - 1)) : "memory");
  SmallFragsOf<MI> f0, f1;
  place();
  read_slab<MI>(std::make_integer_sequence<int, Ring::kReads>{}, f0, w);
  small_arrived(f0);

  constexpr auto kSlots = std::make_integer_sequence<int, 8 * MI>{};
  uint32_t s = 0;
  for (; s + 2 < steps; s += 2) {
    look = after(look); place();
    small_step<OP, false>(kSlots, f0, f1, w);
    fetched();
    look = after(look); place();
    small_step<OP, false>(kSlots, f1, f0, w);
    fetched();
  }
  if (s + 2 == steps) {
    look = after(look); place();
    small_step<OP, false>(kSlots, f0, f1, w);
    small_step<OP, true>(kSlots, f1, f0, w);
  } else {
    small_step<OP, true>(kSlots, f0, f1, w);
  }
  // the wait states between the last matrix instruction and the first read of its result; the fetches that ran
  // ahead of the last step still write LDS
  asm volatile("s_nop 15\n s_nop 15\n s_waitcnt vmcnt(0)" ::: "memory");
  const uint32_t row0 = tm * Ring::kRows + wm * 16u * MI + lane % 16u, col0 = tn * (kGated ? 64u : 128u) + wn * (kGated ? 32u : 64u);
  constexpr auto kDown = std::make_integer_sequence<int, MI>{};
  finish_columns<OP, EPI, 0>(kDown, p, row0, col0, lane);
  if constexpr (!kGated) finish_columns<OP, EPI, 2>(kDown, p, row0, col0, lane);
}

template <int OP, int EPI, int MI>
int launch_tiles(mi355_dev *dev, const char *what, const FfnProduct &p, uint32_t slices) {
  using Ring = SmallRing<MI>;
  if (int rc = allow_full_lds<MI == 4 ? kLdsFfnSmall : kLdsFfnTall, ffn_kind(OP, EPI)>(dev, &ffn_small_kernel<OP, EPI, MI>)) return rc;
  const uint32_t cols = epi_is_gated(EPI) ? 64 : 128;
  const uint64_t tiles_m = (p.m + Ring::kRows - 1ull) / Ring::kRows, tiles_n = (p.n + cols - 1ull) / cols;
  MI355_REQUIRE(dev, tiles_m * tiles_n <= 0xffffffull, "%s: %u x %u outputs are more than one launch takes", what, p.m, p.n);
  const FfnLaunch<EPI> args{p, (uint32_t)tiles_m, (uint32_t)tiles_n};
  ffn_small_kernel<OP, EPI, MI><<<dim3((uint32_t)(tiles_m * tiles_n), slices), kSmallThreads, Ring::kBytes, dev->stream>>>(args);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}
template <int OP, int EPI, int MI>
int launch(mi355_dev *dev, const char *what, const FfnProduct &p, uint32_t slices, void *workspace) {
  if constexpr (EPI == kEpiScaled)
    if (slices > 1) {
      if (int rc = launch_tiles<OP, kEpiPartial, MI>(dev, what, mi355_ffn_slices_of(p, workspace), slices)) return rc;
      FfnJoin join = mi355_ffn_join_of(p, slices, false, workspace);
      return mi355_launch_ffn_join(dev, OP, EPI, what, &join, 1);
    }
  return launch_tiles<OP, EPI, MI>(dev, what, p, 1);
}
template <int MI>
int launch_kind(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p, uint32_t slices, void *workspace) {
  if (op == kQuadI8) return epi == kEpiScaled ? launch<kQuadI8, kEpiScaled, MI>(dev, what, p, slices, workspace) : launch<kQuadI8, kEpiGatedScaled, MI>(dev, what, p, 1, nullptr);
  if (epi != kEpiGated) return mi355_fail(dev, MI355_ERR_ARG, "%s: such products go in groups", what);
  return op == kQuadBf16 ? launch<kQuadBf16, kEpiGated, MI>(dev, what, p, 1, nullptr) : launch<kQuadF16, kEpiGated, MI>(dev, what, p, 1, nullptr);
}
template <int OP, int MI>
int launch_group(mi355_dev *dev, const char *what, const FfnGroup &g) {
  using Ring = SmallRing<MI>;
  if (int rc = allow_full_lds<MI == 4 ? kLdsFfnSmall : kLdsFfnTall, ffn_kind(OP, kEpiPlain)>(dev, &ffn_small_kernel<OP, kEpiPlain, MI>)) return rc;
  FfnLaunch<kEpiPlain> args{g};
  uint32_t blocks = 0;
  if (int rc = mi355_ffn_lay_out_group(dev, what, args.g, Ring::kRows, kSmallTile, blocks)) return rc;
  ffn_small_kernel<OP, kEpiPlain, MI><<<blocks, kSmallThreads, Ring::kBytes, dev->stream>>>(args);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}

}  // namespace

int mi355_launch_ffn_small(mi355_dev *dev, int op, int epi, const char *what, bool tall, const FfnProduct &p, uint32_t slices, void *workspace) {
  return tall ? launch_kind<8>(dev, op, epi, what, p, slices, workspace) : launch_kind<4>(dev, op, epi, what, p, slices, workspace);
}
int mi355_launch_ffn_small_group(mi355_dev *dev, int op, const char *what, bool tall, const FfnGroup &g) {
  if (op == kQuadBf16) return tall ? launch_group<kQuadBf16, 8>(dev, what, g) : launch_group<kQuadBf16, 4>(dev, what, g);
  return tall ? launch_group<kQuadF16, 8>(dev, what, g) : launch_group<kQuadF16, 4>(dev, what, g);
}
