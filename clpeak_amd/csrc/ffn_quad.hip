// The feed-forward products on the schedule of gemm_quad.hip: a workgroup of four waves owns a 256x256 tile of sums,
// persistent, one per CU.  Three things differ.
//
// Operands that end inside a tile.  A lane's row past the last one is read as the last one (the offsets of the wave's 8
// loads are worked out anew for every tile, between two steps), and what such rows give is not stored.
//
// Two products in one.  For the gated projection the tile's 256 rows of B are 64 of the gate's weights, the same 64 of
// the other projection's, and again 64 and 64: each wave fetches the 64 rows of a slab that are one matrix's, so that
// waves 0 and 2 fetch the gate's and 1 and 3 the other's, and a wave's 128 columns of sums are 64 channels of both.
// Gate and value of a channel meet in one lane, and only their product goes to memory.
//
// What becomes of the sums (Finish) runs once per tile, on the vector unit, while the loads of the next tile are
// in flight.
//
// Measured: 8192x8192x4096 bf16 with both sums kept 720 to 760 us by card (1.45 to 1.53 PFLOP/s), 4096x8190x8192 int8 204 us
// (2.7 PFLOP/s of whole numbers), gated 6000x16384x4096 int8 563 to 603 us (2.67 to 2.86); 2048x8192x4096 int8 51.9 us, on
// 128x128 tiles 77.4.  The matrix pipe is busy for 71 to 77 % of that: its clock under load, and 4 to 9 us a round in which
// the CUs' stores leave together, bound it.
#include "ffn.h"
#include "gemm_quad_step.h"
#include "ffn_quad_finish.h"

namespace {

template <int OP, int EPI, int TYPE>
__global__ void __launch_bounds__(kQuadThreads) ffn_quad_kernel(FfnProduct p, uint32_t tiles_m, uint32_t tiles_n) {
  constexpr bool kGated = epi_is_gated(EPI);
  constexpr uint32_t kCols = kGated ? 128 : 256;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const uint32_t tid = threadIdx.x, lane = tid % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const uint32_t wm = wave / 2, wn = wave % 2;
  const TileGrid grid = tiles_of_workgroup(tiles_m, tiles_n);
  const bool many_rounds = grid.total >= Finish<OP, EPI, TYPE>::kManyRounds * grid.stride && Finish<OP, EPI, TYPE>::on_64_bytes(p.out);
  const uint32_t k_bytes = p.k_bytes, steps = k_bytes / kRowBytes;
  const uint32_t lda = (uint32_t)p.lda, ldb = (uint32_t)p.ldb;
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;

  QuadEdgeWalk w;
  const uint32_t chunk = ((lane % 8u) ^ (lane / 8u)) * 16u;
  w.dst_wave = __builtin_amdgcn_readfirstlane(lds_base + wave * 64u * (uint32_t)kRowBytes);
  const uint32_t swz0 = ((lane / 16u) ^ (lane & 7u)) << 4;
  w.lane_a = lds_base + (wm * 128u + lane % 16u) * kRowBytes + swz0;
  w.b_base = lds_base + kSlotB0 + (wn * 128u + lane % 16u) * kRowBytes + swz0;
  w.b_base_hi = w.b_base ^ 64u;

  // the fetch stream, as in gemm_quad.hip: slabs numbered through all tiles of the workgroup, wrapping around behind the
  // last; the walk over K starts at a place of the XCD's own
  uint32_t f_round = 0, f_left = steps, w_left = steps;
  const uint32_t k_rot = (grid.first % 8u) * (steps / 8u);
  auto rows_of = [&](uint32_t rnd) {
    uint32_t tm, tn;
    ffn_tile_at(grid, rnd, tm, tn);
    const uint8_t *b = kGated && (wave & 1u) ? p.b2 : p.b;
    const uint32_t a_row = min(tm * 256u + wave * 64u, p.m - 1u);
    const uint32_t b_row = min(kGated ? tn * 128u + wave / 2u * 64u : tn * 256u + wave * 64u, p.n - 1u);
    w.ga = (uint64_t)(uintptr_t)(p.a + (uint64_t)a_row * lda) + k_rot * kRowBytes;
    w.gb = (uint64_t)(uintptr_t)(b + (uint64_t)b_row * ldb) + k_rot * kRowBytes;
    const uint32_t a_last = p.m - 1u - a_row, b_last = p.n - 1u - b_row;
#pragma unroll
    for (uint32_t q = 0; q < 8; q++) {
      w.voff[q] = min(lane / 8u + 8u * q, a_last) * lda + chunk;
      w.voff_b[q] = min(lane / 8u + 8u * q, b_last) * ldb + chunk;
    }
    w_left = steps - k_rot;
  };
  auto next_fetch_tile = [&]() {
    f_round = f_round + 1u == grid.mine ? 0u : f_round + 1u;
    rows_of(f_round);
    f_left = steps;
  };
  auto fetch = [&](uint32_t slot_a, uint32_t slot_b) {
#pragma unroll
    for (uint32_t q = 0; q < 8; q++) MI355_LOAD_LDS(w.voff_b[q], w.gb, w.dst_wave + kSlotB0 + slot_b * kSlabBytes + q * 1024u);
#pragma unroll
    for (uint32_t q = 0; q < 8; q++) MI355_LOAD_LDS(w.voff[q], w.ga, w.dst_wave + kSlotA0 + slot_a * kSlabBytes + q * 1024u);
    w.ga += kRowBytes;
    w.gb += kRowBytes;
    if (--w_left == 0u) { w.ga -= k_bytes; w.gb -= k_bytes; w_left = steps; }
    if (--f_left == 0u) next_fetch_tile();
  };
  QuadFrags f;
  rows_of(0);
  fetch(0, 0);
  fetch(1, 1);
  asm volatile("s_waitcnt vmcnt(16)\n s_barrier" ::: "memory");   // slab 0 has landed

  quad_claim_accumulators();
  quad_zero_accumulators(std::make_integer_sequence<int, 256>{});
  w.off_cur = 0; w.off_nxt = kSlabBytes; w.off_dst = 2u * kSlabBytes;
  w.dst_a = w.dst_wave + w.off_dst;
  w.a_cur = w.lane_a; w.a_cur_hi = w.a_cur ^ 64u;
  w.a_nxt = w.lane_a + w.off_nxt; w.a_nxt_hi = w.a_nxt ^ 64u;
  w.first = 0;
  {   // what a step expects on entry: the B fragments of its slab in register set 0, rows 0,1 of its A fragments, and
      // its barrier Y behind it
#pragma unroll
    for (int j = 0; j < 8; j++) { Q_DS_READ(f.b_lo[0][j], w.b_base, j * 2048); Q_DS_READ(f.b_hi[0][j], w.b_base_hi, j * 2048); }
#pragma unroll
    for (int r = 0; r < kAhead; r++) { Q_DS_READ(f.a_lo[r], w.a_cur, r * 2048); Q_DS_READ(f.a_hi[r], w.a_cur_hi, r * 2048); }
    asm volatile("s_waitcnt lgkmcnt(0)\n s_barrier"
                 : Q_TIE8(f.b_lo[0]), Q_TIE8(f.b_hi[0]), "+v"(f.a_lo[0]), "+v"(f.a_hi[0]), "+v"(f.a_lo[1]), "+v"(f.a_hi[1]),
                   "+v"(f.a_lo[2]), "+v"(f.a_hi[2]) :: "memory");
  }

  // One countdown to the next event: the fetch stream wraps around or moves on to its next tile, or the tile being
  // multiplied is complete.
  uint32_t round = 0, left = steps;
  auto next_span = [&]() {
    uint32_t m = left < f_left ? left : f_left;
    return m < w_left ? m : w_left;
  };
  uint32_t span = next_span(), ev = span;
  auto event = [&]() -> bool {   // true after the last tile
    left -= span;
    f_left -= span;
    w_left -= span;
    if (w_left == 0u) { w.ga -= k_bytes; w.gb -= k_bytes; w_left = steps; }
    if (f_left == 0u) next_fetch_tile();   // (the step has already moved ga / gb on by a slab: overwritten here)
    bool done = false;
    if (left == 0u) {
      uint32_t tm, tn;
      ffn_tile_at(grid, round, tm, tn);
      Finish<OP, EPI, TYPE>{p, tm * 256u + wm * 128u + lane % 16u, tn * kCols + wn * (kCols / 2u), lane, many_rounds}.run();
      left = steps;
      w.first = 1;
      done = ++round == grid.mine;
    }
    span = next_span();
    ev = span;
    return done;
  };
  constexpr auto slots = std::make_integer_sequence<int, 64>{};
  for (;;) {
    quad_step<OP, 0>(slots, f, w);
    if (__builtin_expect(--ev == 0u, 0) && event()) break;
    quad_step<OP, 1>(slots, f, w);
    if (__builtin_expect(--ev == 0u, 0) && event()) break;
  }
  MI355_DRAIN_RING();
}

template <int OP, int EPI, int TYPE>
int launch(mi355_dev *dev, const char *what, const FfnProduct &p) {
  constexpr bool kGated = epi_is_gated(EPI);
  if (int rc = allow_full_lds<kLdsFfnQuad, (OP != kQuadI8 ? OP - kQuadBf16 : 2 + 3 * kGated + TYPE)>(dev, &ffn_quad_kernel<OP, EPI, TYPE>)) return rc;
  const uint32_t cols = kGated ? 128 : 256;
  const uint64_t tiles_m = (p.m + 255ull) / 256u, tiles_n = (p.n + cols - 1ull) / cols;
  MI355_REQUIRE(dev, tiles_m * tiles_n <= 0x3fffffffull, "%s: %u x %u outputs are more than one launch takes", what, p.m, p.n);
  ffn_quad_kernel<OP, EPI, TYPE><<<gemm_workgroups(dev, (uint32_t)(tiles_m * tiles_n)), kQuadThreads, kRingBytes, dev->stream>>>(p, (uint32_t)tiles_m, (uint32_t)tiles_n);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}
template <int EPI>
int launch_i8(mi355_dev *dev, const char *what, const FfnProduct &p) {
  if (p.out.type == MI355_TYPE_BF16) return launch<kQuadI8, EPI, MI355_TYPE_BF16>(dev, what, p);
  if (p.out.type == MI355_TYPE_F16) return launch<kQuadI8, EPI, MI355_TYPE_F16>(dev, what, p);
  return launch<kQuadI8, EPI, MI355_TYPE_F32>(dev, what, p);
}

}  // namespace

int mi355_launch_ffn_quad(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p) {
  if (op == kQuadI8) return epi == kEpiScaled ? launch_i8<kEpiScaled>(dev, what, p) : launch_i8<kEpiGatedScaled>(dev, what, p);
  if (epi != kEpiGated) return mi355_fail(dev, MI355_ERR_ARG, "%s: no such product on 256x256 tiles", what);   // (plain ones: ffn_across.hip)
  return op == kQuadBf16 ? launch<kQuadBf16, kEpiGated, MI355_TYPE_BF16>(dev, what, p) : launch<kQuadF16, kEpiGated, MI355_TYPE_F16>(dev, what, p);
}
