// Products of some dozens of rows: too many to read every operand straight into registers (ffn_rows.hip: there each group of
// 16 rows of A is read again by every workgroup, at the rate of the vector cache), too few to keep the matrix pipe busy.
// The time is still that of reading the weights, so the kernel is built to keep as much of them in flight as LDS holds:
// a workgroup of four waves owns a 64x64 tile of sums (gated: 32 channels of both matrices) and the whole LDS of a CU, ten
// slots of 16 KiB (64 rows of A and 64 of B, 128 bytes of K), nine of them being filled while the tenth is read.  That is
// 72 KiB of weights on their way to each CU, 18 MiB to the part.
//
// Measured: 48x4096x16384 int8, 64 tiles in 4 slices, 67 MB of weights in 15.5 us (4.3 TB/s), with the join
// 18.1 us; not cut 28.0 us.  128x4096x4096 int8 10.5 us, on 128x128 tiles 17.4 us.  Bound by the weights' way from memory.
//
// A step: wait for this wave's four loads of the slab (they complete in order, eight younger slabs may be in flight) and
// for its own reads of the slab before; barrier; four loads into the slot that everybody has read; eight fragment reads,
// eight matrix instructions.  Slab rows are swizzled as in the other kernels (chunk c of row r at position c ^ (r & 7)).
#include "ffn.h"
#include "gemm_ring.h"

namespace {

constexpr uint32_t kMidTile = 64, kMidThreads = 256;
constexpr uint32_t kMidSlab = kMidTile * kRowBytes, kMidSlot = 2 * kMidSlab, kMidSlots = 10, kMidAhead = 9;
static_assert(kMidSlots * kMidSlot == kRingBytes && kMidAhead + 1 == kMidSlots, "the ring is the whole LDS of a CU");

template <int OP, int EPI>
__global__ void __launch_bounds__(kMidThreads) ffn_mid_kernel(FfnLaunch<EPI> args) {
  const FfnWork work = args.work();
  const FfnProduct &p = work.p;
  constexpr bool kGated = epi_is_gated(EPI);
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t wm = wave / 2, wn = wave % 2;
  const uint32_t tm = work.tile / work.tiles_n, tn = work.tile - tm * work.tiles_n;
  uint32_t steps = p.k_bytes / kRowBytes, k0 = 0;
  if constexpr (EPI == kEpiPlain || EPI == kEpiPartial) {   // (at most 2^19 steps and 16 slices)
    const uint32_t all = steps;
    k0 = all * work.slice / work.slices;
    steps = all * (work.slice + 1u) / work.slices - k0;
  }
  const uint32_t lda = (uint32_t)p.lda, ldb = (uint32_t)p.ldb;

  // global -> LDS: wave w fills rows [16w, 16w+16) of the A slab and of the B slab, 8 rows per instruction (rows past the
  // last one: the last one); lane i is position i%8 of row i/8, which holds logical chunk (i%8) ^ (i/8)
  const uint32_t lds_base = (uint32_t)(uintptr_t)lds;
  const uint32_t dst_wave = __builtin_amdgcn_readfirstlane(lds_base + wave * 16u * (uint32_t)kRowBytes);
  const uint32_t a_row = min(tm * kMidTile + wave * 16u, p.m - 1u);
  const uint32_t b_row = min(kGated ? tn * 32u + wave / 2u * 16u : tn * kMidTile + wave * 16u, p.n - 1u);
  const uint32_t chunk = ((lane % 8u) ^ (lane / 8u)) * 16u;
  uint32_t va[2], vb[2];
#pragma unroll
  for (uint32_t q = 0; q < 2; q++) {
    va[q] = min(lane / 8u + 8u * q, p.m - 1u - a_row) * lda + chunk;
    vb[q] = min(lane / 8u + 8u * q, p.n - 1u - b_row) * ldb + chunk;
  }
  // the walk over K starts at a place of the workgroup's own (ffn_rows.hip says why) and wraps around; past its end it
  // runs on, fetches that nobody reads, so that every step is the same code
  const uint8_t *a0 = p.a + (uint64_t)a_row * lda + (uint64_t)k0 * kRowBytes;
  const uint8_t *b0 = (kGated && (wave & 1u) ? p.b2 : p.b) + (uint64_t)b_row * ldb + (uint64_t)k0 * kRowBytes;
  uint32_t at = (tn / 8u * 8u + tn % 8u * (steps / 8u)) % steps, fill = 0;
  auto fetch = [&]() {
    const uint64_t ga = (uint64_t)(uintptr_t)(a0 + (uint64_t)at * kRowBytes), gb = (uint64_t)(uintptr_t)(b0 + (uint64_t)at * kRowBytes);
    MI355_LOAD_LDS(vb[0], gb, dst_wave + fill + kMidSlab);
    MI355_LOAD_LDS(vb[1], gb, dst_wave + fill + kMidSlab + 1024u);
    MI355_LOAD_LDS(va[0], ga, dst_wave + fill);
    MI355_LOAD_LDS(va[1], ga, dst_wave + fill + 1024u);
    at = at + 1u == steps ? 0u : at + 1u;
    fill = fill + kMidSlot == kRingBytes ? 0u : fill + kMidSlot;
  };
  // LDS -> fragments: row lane%16 of the wave's part, chunk lane/16 (+4 for the second K half: bit 6 of the address)
  const uint32_t swz = ((lane / 16u) ^ (lane & 7u)) << 4;
  const uint32_t lane_a = (wm * 32u + lane % 16u) * kRowBytes + swz, lane_b = kMidSlab + (wn * 32u + lane % 16u) * kRowBytes + swz;

  i32x4v acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; i++) acc[i / 2][i % 2] = (i32x4v){0, 0, 0, 0};
  for (uint32_t d = 0; d < kMidAhead; d++) fetch();
  uint32_t look = 0;
  for (uint32_t s = 0; s < steps; s++) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n s_barrier" :: "n"(4 * (kMidAhead - 1)) : "memory");
    fetch();
    i32x4v a[2][2], b[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        a[i][h] = *reinterpret_cast<const i32x4v *>(lds + look + ((lane_a + i * 16 * kRowBytes) ^ (h * 64u)));
        b[i][h] = *reinterpret_cast<const i32x4v *>(lds + look + ((lane_b + i * 16 * kRowBytes) ^ (h * 64u)));
      }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = ffn_mfma<OP>(b[j][h], a[i][h], acc[i][j]);
    look = look + kMidSlot == kRingBytes ? 0u : look + kMidSlot;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the fetches that ran ahead still write LDS

  const FfnOut &o = p.out;
  const uint32_t row0 = tm * kMidTile + wm * 32u + lane % 16u;
  if constexpr (kGated) {   // (no two neighbouring tiles: 16 channels of both matrices)
#pragma unroll
    for (uint32_t i = 0; i < 2; i++)
      if (row0 + 16u * i < p.m) ffn_finish4<OP, EPI>(o, row0 + 16u * i, tn * 32u + wn * 16u + 4u * (lane / 16u), p.n, acc[i][0], acc[i][1]);
  } else {
    const uint32_t col0 = tn * kMidTile + wn * 32u;
    FfnColumns<EPI> c;
    c.load(o, col0, lane, p.n);
#pragma unroll
    for (uint32_t i = 0; i < 2; i++) {
      float sa = 0.0f;
      if constexpr (EPI == kEpiScaled) sa = o.sa[min(row0 + 16u * i, p.m - 1u)];
      ffn_finish_pair<OP, EPI>(o, row0 + 16u * i, col0, lane, p.m, p.n, sa, c, acc[i], acc[i]);
    }
  }
}

template <int OP, int EPI>
int launch_tiles(mi355_dev *dev, const char *what, const FfnProduct &p, uint32_t slices) {
  if (int rc = allow_full_lds<kLdsFfnMid, ffn_kind(OP, EPI)>(dev, &ffn_mid_kernel<OP, EPI>)) return rc;
  const uint32_t cols = epi_is_gated(EPI) ? 32 : 64;
  const uint64_t tiles_m = (p.m + 63ull) / 64u, tiles_n = (p.n + cols - 1ull) / cols;
  MI355_REQUIRE(dev, tiles_m * tiles_n <= 0xffffffull, "%s: %u x %u outputs are more than one launch takes", what, p.m, p.n);
  const FfnLaunch<EPI> args{p, (uint32_t)tiles_m, (uint32_t)tiles_n};
  ffn_mid_kernel<OP, EPI><<<dim3((uint32_t)(tiles_m * tiles_n), slices), kMidThreads, kRingBytes, dev->stream>>>(args);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}
template <int OP, int EPI>
int launch(mi355_dev *dev, const char *what, const FfnProduct &p, uint32_t slices, void *workspace) {
  if constexpr (EPI == kEpiScaled)
    if (slices > 1) {
      if (int rc = launch_tiles<OP, kEpiPartial>(dev, what, mi355_ffn_slices_of(p, workspace), slices)) return rc;
      FfnJoin join = mi355_ffn_join_of(p, slices, false, workspace);
      return mi355_launch_ffn_join(dev, OP, EPI, what, &join, 1);
    }
  return launch_tiles<OP, EPI>(dev, what, p, 1);
}
template <int OP>
int launch_group(mi355_dev *dev, const char *what, const FfnGroup &g) {
  if (int rc = allow_full_lds<kLdsFfnMid, ffn_kind(OP, kEpiPlain)>(dev, &ffn_mid_kernel<OP, kEpiPlain>)) return rc;
  FfnLaunch<kEpiPlain> args{g};
  uint32_t blocks = 0;
  if (int rc = mi355_ffn_lay_out_group(dev, what, args.g, kMidTile, kMidTile, blocks)) return rc;
  ffn_mid_kernel<OP, kEpiPlain><<<blocks, kMidThreads, kRingBytes, dev->stream>>>(args);
  MI355_LAUNCH_CHECK(dev, what);
  return MI355_OK;
}

}  // namespace

int mi355_launch_ffn_mid(mi355_dev *dev, int op, int epi, const char *what, const FfnProduct &p, uint32_t slices, void *workspace) {
  if (op == kQuadI8) return epi == kEpiScaled ? launch<kQuadI8, kEpiScaled>(dev, what, p, slices, workspace) : launch<kQuadI8, kEpiGatedScaled>(dev, what, p, 1, nullptr);
  if (epi != kEpiGated) return mi355_fail(dev, MI355_ERR_ARG, "%s: such products go in groups", what);
  return op == kQuadBf16 ? launch<kQuadBf16, kEpiGated>(dev, what, p, 1, nullptr) : launch<kQuadF16, kEpiGated>(dev, what, p, 1, nullptr);
}
int mi355_launch_ffn_mid_group(mi355_dev *dev, int op, const char *what, const FfnGroup &g) {
  return op == kQuadBf16 ? launch_group<kQuadBf16>(dev, what, g) : launch_group<kQuadF16>(dev, what, g);
}
