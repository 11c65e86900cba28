// The 8- and 16-bit GEMM kinds on 128x128 tiles, for products whose 256x256 tiling would leave most of the part idle.
//
// gemm_quad.hip gives every workgroup a 256x256 tile of C and the whole LDS of a CU; a product of fewer than 256 such
// tiles (2048^3 has 64) then runs on a fraction of the CUs.  This kernel is the small sibling: one workgroup of four
// waves per 128x128 tile (a wave owns 64x64 = 4x4 tiles of 16x16, in 64 accumulation registers), K walked in steps of
// one 128-byte row segment, a slab of 128 rows x 128 B = 16 KiB per operand and step, global memory straight into
// LDS with the row swizzle of the other GEMM kernels (the 16-byte chunk c of row r lies at position c ^ (r & 7) of the
// row: fragment reads without bank conflicts).
//
// A step is 32 matrix instructions per wave (16 for fp8), 512 cycles of the matrix pipe, a fifth of a microsecond: far
// less than a load takes to arrive.  So the LDS of the CU is a ring of five 32 KiB slots (A and B slab of a step side
// by side), the loads of a slab go out three steps before its fragments are read, and those are read a step before
// they are multiplied, into the other of two fragment sets, in the shadow of the matrix instructions of the step
// before.  Step s: wait until this wave's loads of slab s+1 have landed (loads complete in order: all but the newest
// 16), barrier (now everybody's have, and everybody holds the fragments of slab s in registers, so the slot of slab
// s-1 is free); the matrix instructions on the fragments of slab s, with the 16 reads of slab s+1 behind those of the
// first half and the 8 loads of slab s+4 riding on every fourth; wait for the reads.  The last step reads and loads
// nothing.  Past the last
// slab the loads wrap around to the start of the rows (fetches nobody reads, so that every step but the last is the
// same code); they are waited for before the wave ends.
//
// What bounds it: the issue slots of the wave.  With one wave per SIMD every instruction of a step is issued by the
// wave whose matrix instructions it sits between, about one per four cycles: beside the 32 matrix instructions a step
// has 16 reads, 8 loads with their M0 writes and some scalar bookkeeping, and a direct-to-LDS load holds the issue
// port longer than other instructions.  Measured on constant operands, per step: 0.29-0.30 us (0.21 us is the 512
// cycles of the matrix instructions at 2.4 GHz); with the loads taken out 0.24, with the reads taken out 0.29.  The
// same on 4 and on 128 CUs and for operands of 0.5 MiB (L2) and of 128 MiB (HBM): not a matter of where the data comes
// from, and four slabs in flight instead of three change nothing.  On the whole part under random operands a step
// takes 0.40 us (the clock is lower there, and waves wait more).  (An earlier form of the loads - M0 written, a wait state and the address
// arithmetic in front of every load, all eight behind matrix instructions of the first half - took 0.34 us.)
//
// The sums run over K in order, one step after the other: results differ from the 256x256 kernel's only in rounding
// (that kernel starts its walk over K at a different place on every XCD); the int8 kind is exact either way.
#include "internal.h"
#include "mfma_common.h"
#include "gemm_ring.h"
#include "gemm_quad.h"
#include "gemm_small_step.h"

namespace {

// Tile T = 4i + j of the wave to C: a lane holds 4 consecutive N elements of a row (the product is issued transposed).
template <int OP, int T>
__device__ __forceinline__ void small_store_tile(void *__restrict__ C, uint32_t N, uint32_t row0, uint32_t col0, float scale) {
  const i32x4v t = small_take_tile<T>();
  const size_t at = (size_t)(row0 + (T / 4) * 16u) * N + col0 + (T % 4) * 16u;
  if constexpr (OP == kQuadI8) {
    *reinterpret_cast<i32x4v *>(static_cast<int32_t *>(C) + at) = t;
  } else {
    float x[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int bits = t[r];   // (through a scalar copy: __builtin_bit_cast applied to an element of a vector reads element 0)
      x[r] = __builtin_bit_cast(float, bits);
      if constexpr (small_is_fp8(OP)) x[r] *= scale;
    }
    uint2 packed;
    packed.x = OP == kQuadF16 ? mi355_pack_f16x2(x[0], x[1]) : mi355_pack_bf16x2(x[0], x[1]);
    packed.y = OP == kQuadF16 ? mi355_pack_f16x2(x[2], x[3]) : mi355_pack_bf16x2(x[2], x[3]);
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(C) + at) = packed;
  }
}
template <int OP, int... Ts>
__device__ __forceinline__ void small_store(std::integer_sequence<int, Ts...>, void *__restrict__ C, uint32_t N, uint32_t row0, uint32_t col0, float scale) {
  (small_store_tile<OP, Ts>(C, N, row0, col0, scale), ...);
}

template <int OP>
__global__ void __launch_bounds__(kSmallThreads)
gemm_small_kernel(const uint8_t *__restrict__ A, const uint8_t *__restrict__ B, void *__restrict__ C, uint32_t N, uint32_t k_bytes,
                  float scale, uint32_t tiles_m, uint32_t tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const uint32_t tid = threadIdx.x, lane = tid % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const uint32_t wm = wave / 2, wn = wave % 2;
  TileGrid grid;
  grid.tiles_m = tiles_m; grid.tiles_n = tiles_n; grid.total = tiles_m * tiles_n;
  grid.first = blockIdx.x; grid.stride = gridDim.x; grid.mine = 1;
  uint32_t tm, tn;
  tile_at(grid, 0, tm, tn);
  const uint32_t steps = k_bytes / kRowBytes;
  constexpr uint32_t kRing = kSmallSlots * kSmallSlot;
  auto after = [](uint32_t slot_off) { return slot_off + kSmallSlot == kRing ? 0u : slot_off + kSmallSlot; };

  // global -> LDS: wave w fills rows [32w, 32w+32) of the A slab and of the B slab, 8 rows per instruction; lane i is
  // position i%8 of row i/8, which holds logical chunk (i%8) ^ (i/8)
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  const uint32_t dst_wave = __builtin_amdgcn_readfirstlane(lds_base + wave * 32u * (uint32_t)kRowBytes);
  SmallWalk w;
#pragma unroll
  for (uint32_t q = 0; q < 4; q++) w.voff[q] = (lane / 8u + 8u * q) * k_bytes + ((lane % 8u) ^ (lane / 8u)) * 16u;
  w.ga = (uint64_t)(uintptr_t)(A + ((size_t)tm * kSmallTile + wave * 32u) * k_bytes);
  w.gb = (uint64_t)(uintptr_t)(B + ((size_t)tn * kSmallTile + wave * 32u) * k_bytes);
  uint32_t fetch_left = steps, fill = 0, look = 0;   // slot offsets: the one to fill, the one to read
  auto fetched = [&]() {                             // on to the next slab; past the last one: the first again
    w.ga += kRowBytes;
    w.gb += kRowBytes;
    if (--fetch_left == 0u) { w.ga -= k_bytes; w.gb -= k_bytes; fetch_left = steps; }
    fill = after(fill);
  };
  // LDS -> fragments: row lane%16 of the wave's part, chunk lane/16 (+4 for the second K half: bit 6 of the address),
  // swizzled with row & 7 = lane & 7
  const uint32_t swz0 = ((lane / 16u) ^ (lane & 7u)) << 4;
  const uint32_t lane_a = lds_base + (wm * 64u + lane % 16u) * kRowBytes + swz0;
  const uint32_t lane_b = lds_base + kSmallSlab + (wn * 64u + lane % 16u) * kRowBytes + swz0;
  auto place = [&]() {
    w.a0 = lane_a + look; w.a1 = w.a0 ^ 64u;
    w.b0 = lane_b + look; w.b1 = w.b0 ^ 64u;
    w.dst = dst_wave + fill;
  };

  small_claim_accumulators();
  small_zero_accumulators(std::make_integer_sequence<int, 64>{});

  // slabs 0..3 into slots 0..3; the fragments of slab 0
  for (uint32_t d = 0; d < kSmallAhead; d++) {
    place();
    small_load<0>(w); small_load<1>(w); small_load<2>(w); small_load<3>(w);
    small_load<4>(w); small_load<5>(w); small_load<6>(w); small_load<7>(w);
    fetched();
  }
  asm volatile("s_waitcnt vmcnt(%0)\n s_barrier" :: "n"(8 * (kSmallAhead - 1)) : "memory");
  SmallFrags f0, f1;
  place();
  small_read<0>(f0, w); small_read<1>(f0, w); small_read<2>(f0, w); small_read<3>(f0, w);
  small_read<4>(f0, w); small_read<5>(f0, w); small_read<6>(f0, w); small_read<7>(f0, w);
  small_read<8>(f0, w); small_read<9>(f0, w); small_read<10>(f0, w); small_read<11>(f0, w);
  small_read<12>(f0, w); small_read<13>(f0, w); small_read<14>(f0, w); small_read<15>(f0, w);
  small_arrived(f0);

  // Step s multiplies the fragments of slab s, reads those of slab s+1 and fills the slot of slab s-1, which every
  // wave had in registers before it came to the barrier of step s-1, with slab s+4 (past the last slab: with the
  // first ones again, fetches nobody reads).  Two steps per turn, so that the two fragment sets swap by name.
  constexpr auto kSlots = std::make_integer_sequence<int, small_is_fp8(OP) ? 16 : 32>{};
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
  small_store<OP>(std::make_integer_sequence<int, 16>{}, C, N, tm * kSmallTile + wm * 64u + lane % 16u, tn * kSmallTile + wn * 64u + 4u * (lane / 16u), scale);
}

template <int OP>
int launch_small(mi355_dev *dev, const char *what, const void *A, const void *B, void *C, uint32_t M, uint32_t N, uint32_t k_bytes, float scale) {
  if (int rc = allow_full_lds<kLdsSmall, OP>(dev, &gemm_small_kernel<OP>)) return rc;
  const uint32_t tiles_m = M / kSmallTile, tiles_n = N / kSmallTile;
  gemm_small_kernel<OP><<<tiles_m * tiles_n, kSmallThreads, kRingBytes, dev->stream>>>((const uint8_t *)A, (const uint8_t *)B, C, N, k_bytes, scale,
                                                                                         tiles_m, tiles_n);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}

}  // namespace

// Shapes have been checked by the caller (M and N multiples of 128; K a multiple of 128 bytes; 16-byte aligned buffers;
// a row of K at most 64 MiB).
int mi355_launch_gemm_small(mi355_dev *dev, int op, const char *what, const void *A, const void *B, void *C, uint32_t M, uint32_t N,
                            uint32_t k_bytes, float scale) {
  switch (op) {
    case kQuadE4m3: return launch_small<kQuadE4m3>(dev, what, A, B, C, M, N, k_bytes, scale);
    case kQuadE5m2: return launch_small<kQuadE5m2>(dev, what, A, B, C, M, N, k_bytes, scale);
    case kQuadBf16: return launch_small<kQuadBf16>(dev, what, A, B, C, M, N, k_bytes, scale);
    case kQuadF16: return launch_small<kQuadF16>(dev, what, A, B, C, M, N, k_bytes, scale);
    case kQuadI8: return launch_small<kQuadI8>(dev, what, A, B, C, M, N, k_bytes, scale);
  }
  return mi355_fail(dev, MI355_ERR_ARG, "gemm: unknown operand kind %d", op);
}
