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
#include "ffn.h"
#include "gemm_quad_step.h"

namespace {

// Where a lane's share of a pair of neighbouring tiles goes: 16-bit outputs 8 columns, after the two tiles have traded
// halves (ffn_store_pair in ffn.h), 4-byte ones 4 columns of each.  `at` moves down the wave's rows, 16 at a time.
template <int TYPE>
struct PairOut {
  static constexpr uint32_t kElem = TYPE == MI355_TYPE_F32 ? 4 : 2;
  uint8_t *at;
  uint64_t step;       // bytes between rows 16 apart
  __device__ __forceinline__ static uint32_t first_column(uint32_t lane) {
    const uint32_t g = lane / 16u;
    return TYPE == MI355_TYPE_F32 ? 4u * g : 16u * (g & 1u) + 8u * (g >> 1);
  }
  __device__ __forceinline__ void set(void *base, uint64_t ld, uint32_t row0, uint32_t col0, uint32_t lane) {
    at = static_cast<uint8_t *>(base) + ((uint64_t)row0 * ld + col0 + first_column(lane)) * kElem;
    step = 16u * ld * kElem;
  }
  // `whole`: the row exists and so do all of the lane's columns; `some`: the row exists and only the columns below `rem` do
  // (rem counts from the lane's first column).
  __device__ __forceinline__ void store(const float (&x)[2][4], bool whole, bool edge, bool some, int32_t rem) {
    if constexpr (TYPE == MI355_TYPE_F32) {
      if (whole) {
        __builtin_memcpy(__builtin_assume_aligned(at, 4), x[0], 16);
        __builtin_memcpy(__builtin_assume_aligned(at + 64, 4), x[1], 16);
      }
      if (__builtin_expect(edge, 0)) {
        if (some) {
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (16 * (e / 4) + e % 4 < rem) reinterpret_cast<float *>(at)[16 * (e / 4) + e % 4] = x[e / 4][e % 4];
        }
      }
    } else {
      uint32_t p[2][2];
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          p[t][h] = TYPE == MI355_TYPE_F16 ? mi355_pack_f16x2(x[t][2 * h], x[t][2 * h + 1]) : mi355_pack_bf16x2(x[t][2 * h], x[t][2 * h + 1]);
      const auto q01 = __builtin_amdgcn_permlane16_swap(p[0][0], p[1][0], false, false);
      const auto q23 = __builtin_amdgcn_permlane16_swap(p[0][1], p[1][1], false, false);
      const uint32_t w[4] = {q01[0], q23[0], q01[1], q23[1]};
      if (whole) __builtin_memcpy(__builtin_assume_aligned(at, 2), w, 16);
      if (__builtin_expect(edge, 0)) {
        if (some) {   // (a loop, so that this rare case stays short code)
          uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
          uint16_t *to = reinterpret_cast<uint16_t *>(at);
#pragma unroll 1
          for (int32_t c = 0; c < rem; c++) {
            *to++ = (uint16_t)lo;
            lo = lo >> 16 | hi << 48;
            hi >>= 16;
          }
        }
      }
    }
    at += step;
  }
};

// The scales (and biases) of the columns that a lane has sums of, in a pair of tiles: four neighbours in each.
template <int EPI>
struct PairScales {
  float sb[2][4], more[2][4];   // more: of the other product, or the bias
  __device__ __forceinline__ static void load4(float (&x)[4], const float *from, uint32_t col, uint32_t n) {
    if (col + 4u <= n) {
      __builtin_memcpy(x, __builtin_assume_aligned(from + col, 4), 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = from[min(col + e, n - 1u)];
    }
  }
  __device__ __forceinline__ void load(const FfnOut &o, uint32_t col0, uint32_t lane, uint32_t n) {
    if constexpr (EPI == kEpiScaled || EPI == kEpiGatedScaled) {
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const uint32_t col = col0 + 16u * t + 4u * (lane / 16u);
        load4(sb[t], o.sb, col, n);
        if constexpr (EPI == kEpiGatedScaled) load4(more[t], o.sb2, col, n);
        else if (o.bias) load4(more[t], o.bias, col, n);
      }
    }
  }
};

template <int OP, int EPI, int TYPE>
struct Finish {
  const FfnProduct &p;
  uint32_t row0, col0, lane;   // the lane's first row, the wave's first column
  float sa[8];
  PairOut<TYPE> c, g, u;

  template <int I, int JP>
  __device__ __forceinline__ void tiles(const PairScales<EPI> &k, int32_t rem, bool edge) {
    const i32x4v s[2] = {quad_take_tile<I * 8 + JP>(), quad_take_tile<I * 8 + JP + 1>()};
    float x[2][4], y[2][4];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int32_t v = s[t][e];   // (through a scalar: __builtin_bit_cast of a vector's element reads element 0)
        if constexpr (EPI == kEpiScaled) x[t][e] = p.out.bias ? ffn_scaled_plus(v, sa[I], k.sb[t][e], k.more[t][e]) : ffn_scaled(v, sa[I], k.sb[t][e]);
        else if constexpr (EPI == kEpiGatedScaled) x[t][e] = ffn_scaled(v, sa[I], k.sb[t][e]);
        else x[t][e] = __builtin_bit_cast(float, v);
      }
    const bool row = 16u * I < p.m - row0 && row0 < p.m;
    const bool whole = row && rem >= (TYPE == MI355_TYPE_F32 ? 20 : 8);
    if constexpr (epi_is_gated(EPI)) {
      const i32x4v s2[2] = {quad_take_tile<I * 8 + JP + 4>(), quad_take_tile<I * 8 + JP + 5>()};
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int32_t v = s2[t][e];
          if constexpr (EPI == kEpiGatedScaled) y[t][e] = ffn_scaled(v, sa[I], k.more[t][e]);
          else y[t][e] = __builtin_bit_cast(float, v);
        }
      if constexpr (EPI == kEpiGated)
        if (p.out.g) {
          g.store(x, whole, edge, row && !whole, rem);
          u.store(y, whole, edge, row && !whole, rem);
        }
      // one branch on the activation for the 8 values
      auto gate = [&](int act) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e / 4][e % 4] = ffn_act(act, x[e / 4][e % 4]) * y[e / 4][e % 4];
      };
      if (p.out.act == MI355_GLU_SILU) gate(MI355_GLU_SILU);
      else if (p.out.act == MI355_GLU_GELU_TANH) gate(MI355_GLU_GELU_TANH);
      else if (p.out.act == MI355_GLU_GELU) gate(MI355_GLU_GELU);
      else gate(MI355_GLU_RELU);
    }
    c.store(x, whole, edge, row && !whole, rem);
    __builtin_amdgcn_sched_barrier(0);   // few tiles at a time: the fragment registers stay live, few are free
  }
  template <int JP, int... Is>
  __device__ __forceinline__ void columns(std::integer_sequence<int, Is...>, const PairScales<EPI> &k) {
    const uint32_t col = col0 + 16u * JP;
    const int32_t rem = (int32_t)(p.n - col) - (int32_t)PairOut<TYPE>::first_column(lane);
    const bool edge = col + 32u > p.n;
    c.set(p.out.c, p.out.ldc, row0, col, lane);
    if constexpr (EPI == kEpiGated)
      if (p.out.g) {
        g.set(p.out.g, p.out.ldg, row0, col, lane);
        u.set(p.out.u, p.out.ldg, row0, col, lane);
      }
    (tiles<Is, JP>(k, rem, edge), ...);
  }
  // The scales of the first columns are on their way before the wave waits for the last matrix instructions and for the
  // loads of its next slabs, those of every further pair of tiles while the pair before is finished.
  __device__ __forceinline__ void run() {
    PairScales<EPI> k0, k1;
    k0.load(p.out, col0, lane, p.n);
    if constexpr (OP == kQuadI8) {
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) sa[i] = p.out.sa[min(row0 + 16u * i, p.m - 1u)];
    }
    // the wait states the compiler cannot know about, then every load of this wave (the next barrier X then needs no
    // wait of its own, and the stores issued here do not enter its count)
    asm volatile("s_nop 15\n s_nop 15\n s_waitcnt vmcnt(0)" ::: "memory");
    constexpr auto rows = std::make_integer_sequence<int, 8>{};
    k1.load(p.out, col0 + 32u, lane, p.n);
    columns<0>(rows, k0);
    if constexpr (epi_is_gated(EPI)) {
      columns<2>(rows, k1);
    } else {
      k0.load(p.out, col0 + 64u, lane, p.n);
      columns<2>(rows, k1);
      k1.load(p.out, col0 + 96u, lane, p.n);
      columns<4>(rows, k0);
      columns<6>(rows, k1);
    }
    asm volatile("s_nop 7");   // accumulation registers written by the vector unit, read next by the matrix unit
  }
};

template <int OP, int EPI, int TYPE>
__global__ void __launch_bounds__(kQuadThreads) ffn_quad_kernel(FfnProduct p, uint32_t tiles_m, uint32_t tiles_n) {
  constexpr bool kGated = epi_is_gated(EPI);
  constexpr uint32_t kCols = kGated ? 128 : 256;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const uint32_t tid = threadIdx.x, lane = tid % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const uint32_t wm = wave / 2, wn = wave % 2;
  const TileGrid grid = tiles_of_workgroup(tiles_m, tiles_n);
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
    tile_at(grid, rnd, tm, tn);
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
      tile_at(grid, round, tm, tn);
      Finish<OP, EPI, TYPE>{p, tm * 256u + wm * 128u + lane % 16u, tn * kCols + wn * (kCols / 2u), lane}.run();
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
  if (int rc = allow_full_lds(dev, &ffn_quad_kernel<OP, EPI, TYPE>, kLdsFfnQuad0 + ffn_kind(OP, EPI, TYPE))) return rc;
  const uint32_t cols = epi_is_gated(EPI) ? 128 : 256;
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
  if (op == kQuadBf16) return epi == kEpiPlain ? launch<kQuadBf16, kEpiPlain, MI355_TYPE_BF16>(dev, what, p) : launch<kQuadBf16, kEpiGated, MI355_TYPE_BF16>(dev, what, p);
  return epi == kEpiPlain ? launch<kQuadF16, kEpiPlain, MI355_TYPE_F16>(dev, what, p) : launch<kQuadF16, kEpiGated, MI355_TYPE_F16>(dev, what, p);
}
