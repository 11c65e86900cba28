// Products whose sum runs over the rows of an operand, as the gradients' do: dX = dG Wg + dU Wu sums over the rows of the
// weights, dW = dG^T X over the rows of both.  In memory such an operand has the sum's index outside ("across"): the 8
// values of a lane's fragment are a row apart.  CDNA4 reads them out of LDS that way round (ds_read_b64_tr_b16: 16 lanes
// read a block of 4 rows by 16 columns, 8 bytes each, and lane c gets column c, 4 values of the sum's index), so nothing
// has to be turned in memory first.
//
// Otherwise this is the schedule of gemm_quad.hip with ffn_quad.hip's edges: 256x256 tiles of sums, four waves, steps of
// 64 values of the sum, three A slots and two B slots of 32 KiB, the accumulators in the accumulation registers.  What
// differs:
//   * An across slab is 64 rows of 256 columns, 512 bytes a row.  32-byte chunk c (16 columns) of row r lies at position
//     c ^ f(r), f = r & 3 plus 4 for odd eights of rows: the four rows that 16 lanes read at once, and the two groups of
//     16 lanes next to each other, then come from different banks.  Fragment number i of a wave is chunk 8 w + i, so its
//     address is that of fragment 0 with bits 5..7 xored with i.
//   * B (always across) is up to four stretches of rows, one behind the other along the sum: dX has Wg's rows and Wu's, and
//     where their number is no multiple of 64 the last ones come from a copy padded with zeros.  The fetch stream stops
//     between two steps to go on to the next stretch, as it does for the next tile.
//   * The LDS reads are the compiler's (there is no way to name half of a register tuple in inline assembly), which
//     therefore places the waits for their results; matrix instructions, loads and barriers are as in gemm_quad.hip.
//
// Measured, for 8192x8192x4096 bf16: dX 696 us, both dW in one launch 708 us (1.55 PFLOP/s each), the matrix pipe busy for
// 85 % and 80 % of it, no bank conflicts.  Bound by the clock under load.
#include "ffn_across.h"
#include "ffn_quad_finish.h"

namespace {

typedef short v4i16 __attribute__((ext_vector_type(4)));

struct AcrossFrags {
  i32x4v b_lo[2][8], b_hi[2][8];   // two register sets of B fragments (current step / next step)
  i32x4v a_lo[4], a_hi[4];         // four rotating A fragment slots: row i lives in slot i mod 4
};
struct AcrossWalk {
  uint32_t a_cur, a_nxt;           // LDS address of this lane's A fragment 0 in the slots of slabs s, s+1
  uint32_t lane_a;                 // ... within a slot
  uint32_t b_base;                 // the same for B, in B slot 0
  uint32_t off_cur, off_nxt, off_dst;
  uint32_t dst_a, dst_wave;
  uint64_t ga, gb, step_a, step_b; // addresses of the next slab to fetch and the bytes from a slab to the next (uniform)
  uint32_t voff[8], voff_b[8];
  uint32_t first;
};

__device__ __forceinline__ i32x4v read16(uint32_t at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) i32x4v *>((uintptr_t)at);
}
// 8 values of one column, rows apart: two blocks of 4 rows, 2 KiB on.
__device__ __forceinline__ i32x4v read_across(uint32_t at) {
  typedef __attribute__((address_space(3))) v4i16 *block;
  const v4i16 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((block)(uintptr_t)at), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((block)(uintptr_t)(at + 2048u));
  return __builtin_bit_cast(i32x4v, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// An address that is the same in all lanes, in scalar registers: where the loads' inline assembly wants it, whatever the
// compiler has made of the arithmetic.
__device__ __forceinline__ uint64_t in_scalars(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

template <bool ACROSS_A>
__device__ __forceinline__ void read_a(AcrossFrags &f, uint32_t base, int row) {
  if constexpr (ACROSS_A) {
    const uint32_t at = base ^ (uint32_t)(row * 32);
    f.a_lo[row % 4] = read_across(at);
    f.a_hi[row % 4] = read_across(at + 16384u);
  } else {
    f.a_lo[row % 4] = read16(base + row * 2048u);
    f.a_hi[row % 4] = read16((base ^ 64u) + row * 2048u);
  }
}
template <int SLOT>
__device__ __forceinline__ void read_b(AcrossFrags &f, const AcrossWalk &w, int j, int half) {
  const uint32_t at = (w.b_base ^ (uint32_t)(j * 32)) + SLOT * kSlabBytes + half * 16384u;
  if (half == 0) f.b_lo[SLOT][j] = read_across(at);
  else f.b_hi[SLOT][j] = read_across(at);
}

// Slot P of a step of parity PAR; gemm_quad_step.h says what rides on which slot.
template <int OP, bool ACROSS_A, int PAR, int P>
__device__ __forceinline__ void across_slot(AcrossFrags &f, AcrossWalk &w) {
  constexpr int i = P / 8, j = P % 8, sl = i % 4, T = P;
  if constexpr (j == 0) {
    Q_PIN();
    if constexpr (i + kAhead <= 7) read_a<ACROSS_A>(f, w.a_cur, i + kAhead);
    else read_a<ACROSS_A>(f, w.a_nxt, i + kAhead - 8);
    Q_PIN();
  }
  constexpr int q = P / kLoadEvery;
  constexpr bool with_load = P % kLoadEvery == 0 && q < 16;
  if constexpr (with_load && q < 8)
    q_mfma_load<OP, T, kSlotB0 + PAR * kSlabBytes + q * 1024>(f.b_lo[PAR][j], f.a_lo[sl], w.dst_wave, w.voff_b[q], w.gb);
  else if constexpr (with_load)
    q_mfma_load<OP, T, (q - 8) * 1024>(f.b_lo[PAR][j], f.a_lo[sl], w.dst_a, w.voff[q - 8], w.ga);
  else
    q_mfma<OP, T>(f.b_lo[PAR][j], f.a_lo[sl]);
  q_mfma<OP, T>(f.b_hi[PAR][j], f.a_hi[sl]);
  if constexpr (P == kSlotX) {
    asm volatile("s_cmp_lg_u32 %0, 0\n s_cbranch_scc1 1f\n s_waitcnt vmcnt(%1)\n1:\n s_barrier" :: "s"(w.first), "n"(kKeepAtX) : "memory", "scc");
  }
  if constexpr (P > kSlotX && P <= kSlotX + 16) {
    Q_PIN();
    read_b<(PAR ^ 1)>(f, w, (P - kSlotX - 1) / 2, (P - kSlotX - 1) % 2);
    Q_PIN();
  }
  if constexpr (P == 7 * kLoadEvery + 1) { Q_PIN(); w.gb += w.step_b; Q_PIN(); }
  if constexpr (P == kSlotX + 1) { Q_PIN(); w.first = 0; Q_PIN(); }
  if constexpr (P == 15 * kLoadEvery + 1) { Q_PIN(); w.ga += w.step_a; Q_PIN(); }
  if constexpr (P == 15 * kLoadEvery + 2) {
    Q_PIN();
    const uint32_t t = w.off_cur;
    w.off_cur = w.off_nxt; w.off_nxt = w.off_dst; w.off_dst = t;
    w.dst_a = (uint32_t)__builtin_amdgcn_readfirstlane((int)(w.dst_wave + w.off_dst));
    Q_PIN();
  }
  if constexpr (P == 57) {
    Q_PIN();
    w.a_cur = w.a_nxt;
    w.a_nxt = w.lane_a + w.off_nxt;
    Q_PIN();
  }
  // every read of this step has arrived; barrier Y of the next step: the slots that its loads overwrite have been read
  if constexpr (P == 60) asm volatile("s_waitcnt lgkmcnt(0)\n s_barrier" ::: "memory");
}
template <int OP, bool ACROSS_A, int PAR, int... Ps>
__device__ __forceinline__ void across_step(std::integer_sequence<int, Ps...>, AcrossFrags &f, AcrossWalk &w) {
  (across_slot<OP, ACROSS_A, PAR, Ps>(f, w), ...);
}

// ACROSS_A: A is [k][columns], in parts of p.part columns each (a product for each, B shared); otherwise [rows][k].
// Slice blockIdx.y of gridDim.y of the sum (kEpiPartial: the sums go to p.out.c, p.c2 as matrix number blockIdx.y there).
template <int OP, bool ACROSS_A, int EPI, int TYPE>
__global__ void __launch_bounds__(kQuadThreads) ffn_across_kernel(FfnAcross p, uint32_t tiles_m, uint32_t tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const uint32_t tid = threadIdx.x, lane = tid % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const uint32_t wm = wave / 2, wn = wave % 2;
  const TileGrid grid = tiles_of_workgroup(tiles_m, tiles_n);
  const uint32_t k0 = EPI == kEpiPartial ? (uint32_t)((uint64_t)p.steps * blockIdx.y / gridDim.y) : 0u;
  const uint32_t steps = EPI == kEpiPartial ? (uint32_t)((uint64_t)p.steps * (blockIdx.y + 1u) / gridDim.y) - k0 : p.steps;
  const uint32_t lda = (uint32_t)p.lda;
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  const uint32_t tiles_part = ACROSS_A ? tiles_m / p.parts : tiles_m;

  AcrossWalk w;
  w.dst_wave = __builtin_amdgcn_readfirstlane(lds_base + wave * 64u * (uint32_t)kRowBytes);
  // LDS -> fragments.  Across: row 8 (lane / 16) + lane % 16 / 4 of the slab, chunk 8 wm (wn) of it, 8 bytes at lane % 4
  const uint32_t row = 8u * (lane / 16u) + lane % 16u / 4u, f_row = (row & 3u) | (row >> 3 & 1u) << 2;
  const uint32_t across = row * 512u + f_row * 32u + lane % 4u * 8u;
  w.lane_a = ACROSS_A ? lds_base + across + wm * 256u : lds_base + (wm * 128u + lane % 16u) * kRowBytes + (((lane / 16u) ^ (lane & 7u)) << 4);
  w.b_base = lds_base + kSlotB0 + across + wn * 256u;

  // global -> LDS.  Load q of a wave fills 1 KiB: 8 rows of 128 bytes, or across 2 rows of 512, rows 16 wave + 2 q and one
  // more; lane i is 16-byte position i % 32 of row i / 32, half of chunk position i % 32 / 2
  const uint32_t chunk = ((lane % 8u) ^ (lane / 8u)) * 16u;
  auto across_column = [&](uint32_t q) {   // this lane's first column, of the 256
    const uint32_t r = 2u * q + lane / 32u, f = (r & 3u) | (r >> 3 & 1u) << 2;
    return ((lane % 32u / 2u) ^ f) * 16u + (lane & 1u) * 8u;
  };

  // The fetch stream: slabs numbered through all tiles of the workgroup, wrapping around behind the last; the walk over the
  // sum starts at a place of the XCD's own.
  uint32_t f_round = 0, f_left = steps, stretch_left = 0;
  const uint32_t k_rot = (grid.first % 8u) * (steps / 8u);
  w.step_a = ACROSS_A ? 64ull * lda : (uint64_t)kRowBytes;
  auto place = [&](uint32_t rnd, uint32_t pos) __attribute__((always_inline)) {   // the stream stands on slab `pos` of the tile of round `rnd`
    uint32_t tm, tn;
    ffn_tile_at(grid, rnd, tm, tn);
    const uint32_t slab = k0 + pos;
    if constexpr (ACROSS_A) {
      const uint32_t part = tm / tiles_part, col0 = (tm - part * tiles_part) * 256u;
      w.ga = in_scalars((uint64_t)(uintptr_t)(p.a + (uint64_t)part * p.part * 2u + ((uint64_t)slab * 64u + wave * 16u) * lda));
#pragma unroll
      for (uint32_t q = 0; q < 8; q++) w.voff[q] = (2u * q + lane / 32u) * lda + 2u * min(col0 + across_column(q), p.part - 8u);
    } else {
      const uint32_t a_row = min(tm * 256u + wave * 64u, p.m - 1u);
      w.ga = in_scalars((uint64_t)(uintptr_t)(p.a + (uint64_t)a_row * lda + (uint64_t)slab * kRowBytes));
#pragma unroll
      for (uint32_t q = 0; q < 8; q++) w.voff[q] = min(lane / 8u + 8u * q, p.m - 1u - a_row) * lda + chunk;
    }
    uint32_t at = slab, slabs = p.b[0].slabs, ldb = p.b[0].ld;
    const uint8_t *rows = p.b[0].rows;
#pragma unroll
    for (uint32_t s = 1; s < 4; s++) {   // (no index that varies: the addresses have to stay in scalar registers)
      const bool on = s < p.stretches && at >= slabs;
      at = on ? at - slabs : at;
      rows = on ? p.b[s].rows : rows;
      ldb = on ? p.b[s].ld : ldb;
      slabs = on ? p.b[s].slabs : slabs;
    }
    stretch_left = min(slabs - at, steps - pos);   // (a slice may end inside a stretch)
    w.gb = in_scalars((uint64_t)(uintptr_t)(rows + ((uint64_t)at * 64u + wave * 16u) * ldb));
    w.step_b = 64ull * ldb;
#pragma unroll
    for (uint32_t q = 0; q < 8; q++) w.voff_b[q] = (2u * q + lane / 32u) * ldb + 2u * min(tn * 256u + across_column(q), p.n - 8u);
  };
  auto follow = [&]() __attribute__((always_inline)) {   // behind the end of a stretch or of a tile
    if (f_left == 0u) {
      f_round = f_round + 1u == grid.mine ? 0u : f_round + 1u;
      f_left = steps;
      place(f_round, k_rot);
    } else if (stretch_left == 0u) {
      const uint32_t pos = k_rot + steps - f_left;
      place(f_round, pos >= steps ? pos - steps : pos);
    }
  };
  auto fetch = [&](uint32_t slot_a, uint32_t slot_b) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t q = 0; q < 8; q++) MI355_LOAD_LDS(w.voff_b[q], w.gb, w.dst_wave + kSlotB0 + slot_b * kSlabBytes + q * 1024u);
#pragma unroll
    for (uint32_t q = 0; q < 8; q++) MI355_LOAD_LDS(w.voff[q], w.ga, w.dst_wave + kSlotA0 + slot_a * kSlabBytes + q * 1024u);
    w.ga += w.step_a;
    w.gb += w.step_b;
    f_left--;
    stretch_left--;
    follow();
  };
  AcrossFrags f;
  place(0, k_rot);
  fetch(0, 0);
  fetch(1, 1);
  asm volatile("s_waitcnt vmcnt(16)\n s_barrier" ::: "memory");   // slab 0 has landed

  quad_claim_accumulators();
  quad_zero_accumulators(std::make_integer_sequence<int, 256>{});
  w.off_cur = 0; w.off_nxt = kSlabBytes; w.off_dst = 2u * kSlabBytes;
  w.dst_a = w.dst_wave + w.off_dst;
  w.a_cur = w.lane_a;
  w.a_nxt = w.lane_a + w.off_nxt;
  w.first = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) { read_b<0>(f, w, j, 0); read_b<0>(f, w, j, 1); }
#pragma unroll
  for (int r = 0; r < kAhead; r++) read_a<ACROSS_A>(f, w.a_cur, r);
  asm volatile("s_waitcnt lgkmcnt(0)\n s_barrier" ::: "memory");

  // One countdown to the next event: the fetch stream goes on to another stretch or tile, or the tile being multiplied is
  // complete.
  uint32_t round = 0, left = steps;
  auto next_span = [&]() {
    const uint32_t m = left < f_left ? left : f_left;
    return m < stretch_left ? m : stretch_left;
  };
  uint32_t span = next_span(), ev = span;
  auto event = [&]() __attribute__((always_inline)) -> bool {   // true after the last tile
    left -= span;
    f_left -= span;
    stretch_left -= span;
    follow();   // (the step has already moved ga / gb on by a slab: overwritten there)
    bool done = false;
    if (left == 0u) {
      uint32_t tm, tn;
      ffn_tile_at(grid, round, tm, tn);
      FfnProduct o{};
      o.m = p.m; o.n = p.n;
      o.out = p.out;
      uint32_t row_tile = tm;
      if constexpr (ACROSS_A) {
        const uint32_t part = tm / tiles_part;
        row_tile = tm - part * tiles_part;
        if (part) o.out.c = p.c2;
      }
      if constexpr (EPI == kEpiPartial) o.out.c = static_cast<float *>(o.out.c) + (uint64_t)blockIdx.y * p.m * p.out.ldc;
      Finish<OP, EPI, TYPE>{o, row_tile * 256u + wm * 128u + lane % 16u, tn * 256u + wn * 128u, lane, false}.run();
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
    across_step<OP, ACROSS_A, 0>(slots, f, w);
    if (__builtin_expect(--ev == 0u, 0) && event()) break;
    across_step<OP, ACROSS_A, 1>(slots, f, w);
    if (__builtin_expect(--ev == 0u, 0) && event()) break;
  }
  MI355_DRAIN_RING();
}

template <int OP, bool ACROSS_A, int EPI, int TYPE>
int launch(mi355_dev *dev, const char *what, const FfnAcross &p, uint32_t slices) {
  if (int rc = allow_full_lds<kLdsFfnAcross, (OP == kQuadF16) * 4 + ACROSS_A * 2 + (EPI == kEpiPartial)>(dev, &ffn_across_kernel<OP, ACROSS_A, EPI, TYPE>)) return rc;
  const uint64_t tiles_m = (uint64_t)p.parts * ((p.m + 255u) / 256u), tiles_n = (p.n + 255u) / 256u;
  MI355_REQUIRE(dev, tiles_m * tiles_n <= 0x3fffffffull, "%s: %u x %u outputs are more than one launch takes", what, p.m, p.n);
  const dim3 grid(slices > 1 ? (uint32_t)(tiles_m * tiles_n) : gemm_workgroups(dev, (uint32_t)(tiles_m * tiles_n)), slices);
  ffn_across_kernel<OP, ACROSS_A, EPI, TYPE><<<grid, kQuadThreads, kRingBytes, dev->stream>>>(p, (uint32_t)tiles_m, (uint32_t)tiles_n);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}
template <int OP, bool ACROSS_A, int TYPE>
int launch_slices(mi355_dev *dev, const char *what, const FfnAcross &p, uint32_t slices, uint8_t *workspace) {
  if (slices <= 1 && !p.pairs) return launch<OP, ACROSS_A, kEpiPlain, TYPE>(dev, what, p, 1);
  const uint64_t part = slices * (uint64_t)p.m * p.n * 4u;
  FfnAcross q = p;
  q.out.c = workspace;
  q.c2 = workspace + part;
  q.out.ldc = p.n;
  if (int rc = launch<OP, ACROSS_A, kEpiPartial, MI355_TYPE_F32>(dev, what, q, slices)) return rc;
  FfnJoin join[2];
  for (uint32_t i = 0; i < p.parts; i++) {
    FfnProduct o{};
    o.m = p.m; o.n = p.n;
    o.out = p.out;
    if (i) o.out.c = p.c2;
    join[i] = mi355_ffn_join_of(o, slices, p.pairs, workspace + i * part);
  }
  return mi355_launch_ffn_join(dev, OP, kEpiPlain, what, join, p.parts);
}

}  // namespace

int mi355_launch_ffn_across(mi355_dev *dev, int op, bool across_a, const char *what, const FfnAcross &p, uint32_t slices, uint8_t *workspace) {
  if (op == kQuadBf16) return across_a ? launch_slices<kQuadBf16, true, MI355_TYPE_BF16>(dev, what, p, slices, workspace) : launch_slices<kQuadBf16, false, MI355_TYPE_BF16>(dev, what, p, slices, workspace);
  return across_a ? launch_slices<kQuadF16, true, MI355_TYPE_F16>(dev, what, p, slices, workspace) : launch_slices<kQuadF16, false, MI355_TYPE_F16>(dev, what, p, slices, workspace);
}
