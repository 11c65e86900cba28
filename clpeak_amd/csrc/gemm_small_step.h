// The step of the GEMM kernel on 128x128 tiles: what gemm_small.hip describes, shared by its kernel and by the
// feed-forward products (ffn_small.hip), whose operands may end inside a tile and whose tiles may be twice as tall: MI is the
// number of 16-row tiles of a wave (4, or 8 for 256x128 sums, a wave 128x64), of columns it has 4.
#pragma once
#include "mfma_common.h"
#include "gemm_ring.h"
#include "gemm_quad.h"
#include <utility>

namespace {

constexpr int kSmallTile = 128, kSmallThreads = 256;
constexpr uint32_t kSmallSlab = kSmallTile * kRowBytes;   // 16 KiB per operand and step
constexpr uint32_t kSmallSlot = 2u * kSmallSlab;          // A slab, then B slab
constexpr uint32_t kSmallSlots = 5, kSmallAhead = 4;      // ring depth; how many steps ahead of its use a slab is fetched
static_assert(kSmallSlots * kSmallSlot == kRingBytes && kSmallAhead + 1 == kSmallSlots, "the ring is the whole LDS of a CU");
// The same for either height.  The tall ring holds three steps: a slab is fetched three steps ahead, into the slot whose
// fragments every wave has in registers.
template <int MI>
struct SmallRing {
  static constexpr uint32_t kRows = 32 * MI, kSlabA = kRows * kRowBytes, kSlot = kSlabA + kSmallSlab;
  static constexpr uint32_t kSlots = MI == 4 ? kSmallSlots : 3, kAhead = MI == 4 ? kSmallAhead : 3, kBytes = kSlots * kSlot;
  static constexpr int kLoads = MI + 4, kReads = 2 * (MI + 4), kTiles = MI * 4;
  static_assert(kBytes <= kRingBytes && kAhead <= kSlots, "");
};

constexpr bool small_is_fp8(int op) { return op == kQuadE4m3 || op == kQuadE5m2; }

#define S_DS_READ(dst, addr, off) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(dst) : "v"(addr), "n"(off))
#define S_TIE4(x) "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3])

// The fragments of one step: rows [16i, 16i+16) of the wave's rows of A (a_*[i]) and of B (b_*[i]), K halves lo / hi.
template <int MI>
struct SmallFragsOf {
  i32x4v a_lo[MI], a_hi[MI], b_lo[4], b_hi[4];
};
using SmallFrags = SmallFragsOf<4>;

// What a step needs to know beside its fragments.
template <int MI>
struct SmallWalkOf {
  uint32_t a0, a1, b0, b1;   // LDS addresses of this lane's first A / B fragment in the slab to read, K halves lo / hi
  uint32_t dst;              // LDS destination of the wave's first rows in the slot to fill
  uint32_t voff[MI];         // this lane's byte offset from ga / gb in each of the wave's groups of 8 rows
  uint64_t ga, gb;           // the wave's A / B rows in the slab to fetch
};
using SmallWalk = SmallWalkOf<4>;
// Where an operand may end inside a tile its rows past the end are read as its last one, so that the lanes' offsets differ
// between A (voff) and B.
template <int MI>
struct SmallEdgeWalk : SmallWalkOf<MI> {
  uint32_t voff_b[4];
};
__device__ __forceinline__ uint32_t small_voff_b(const SmallWalk &w, int q) { return w.voff[q]; }
template <int MI>
__device__ __forceinline__ uint32_t small_voff_b(const SmallEdgeWalk<MI> &w, int q) { return w.voff_b[q]; }
// A wave's first rows of B, but for the slab in front of them; in a tall tile they are not as far on as its rows of A.
struct SmallTallWalk : SmallEdgeWalk<8> {
  uint32_t dst_b;
};
__device__ __forceinline__ uint32_t small_dst_b(const SmallWalk &w) { return w.dst; }
__device__ __forceinline__ uint32_t small_dst_b(const SmallTallWalk &w) { return w.dst_b; }

// The accumulators are the accumulation registers a[0:63] (tall: a[0:127]), named in the instruction text: tile (i, j) of
// the wave's MI x 4 tiles is a[4T : 4T+3], T = 4i + j.  The compiler is told once that they are taken and never sees them as values:
// what it holds as a value it may copy where paths of the program join, and it does not know that a register written
// by a matrix instruction of this file's text must not be read for some cycles.
template <int MI = 4>
__device__ __forceinline__ void small_claim_accumulators() {
#define S_A10(n) "a" #n "0", "a" #n "1", "a" #n "2", "a" #n "3", "a" #n "4", "a" #n "5", "a" #n "6", "a" #n "7", "a" #n "8", "a" #n "9"
  asm volatile("" ::: "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", S_A10(1), S_A10(2), S_A10(3), S_A10(4), S_A10(5), "a60", "a61",
               "a62", "a63");
  if constexpr (MI == 8)
    asm volatile("" ::: "a64", "a65", "a66", "a67", "a68", "a69", S_A10(7), S_A10(8), S_A10(9), S_A10(10), S_A10(11), "a120", "a121", "a122", "a123",
                 "a124", "a125", "a126", "a127");
#undef S_A10
}
template <int R>
__device__ __forceinline__ void small_zero_register() { asm volatile("v_accvgpr_write_b32 a[%0], 0" :: "n"(R)); }
template <int... Rs>
__device__ __forceinline__ void small_zero_accumulators(std::integer_sequence<int, Rs...>) {
  (small_zero_register<Rs>(), ...);
  asm volatile("s_nop 7");   // written by the vector unit, read next by the matrix unit
}
// Tile T out of the accumulation registers, as raw bits.
template <int T>
__device__ __forceinline__ i32x4v small_take_tile() {
  int v0, v1, v2, v3;
  asm volatile("v_accvgpr_read_b32 %0, a[%4]\n v_accvgpr_read_b32 %1, a[%5]\n v_accvgpr_read_b32 %2, a[%6]\n v_accvgpr_read_b32 %3, a[%7]"
               : "=&v"(v0), "=&v"(v1), "=&v"(v2), "=&v"(v3) : "n"(4 * T), "n"(4 * T + 1), "n"(4 * T + 2), "n"(4 * T + 3));
  return (i32x4v){v0, v1, v2, v3};
}

// Matrix instruction number S of a step.  The 16-bit and int8 kinds take 8 MI, an instruction per K half: row i of the
// wave's tiles is instructions 8i .. 8i+7, its four first halves and then its four second halves, so that an
// instruction never waits for the one just before it.  fp8 takes 16, one K = 128 instruction on both halves (the A
// fragment is the second source of the transposed product: format field blgp for an e5m2 A).
// Q >= 0: load number Q of the slab to fetch rides along (8 rows of A for Q < MI, of B otherwise, into the slot being
// filled): M0, which holds the LDS destination, is written in front of the matrix instruction, which is the wait state
// M0 needs before a load reads it, and the load is issued behind it; three instructions in all.
template <int OP, int S, int Q = -1, int MI, class Walk>
__device__ __forceinline__ void small_mfma(const SmallFragsOf<MI> &f, const Walk &w) {
#define S_MFMA(insn, fmt, T, b, a)                                                                                              \
  if constexpr (Q < 0) asm volatile(insn " a[%2:%3], %0, %1, a[%2:%3]" fmt :: "v"(b), "v"(a), "n"(4 * (T)), "n"(4 * (T) + 3));    \
  else asm volatile("s_add_u32 m0, %4, %5\n " insn " a[%2:%3], %0, %1, a[%2:%3]" fmt "\n global_load_lds_dwordx4 %6, %7"         \
                    :: "v"(b), "v"(a), "n"(4 * (T)), "n"(4 * (T) + 3), "s"(Q < MI ? w.dst : small_dst_b(w)), "n"(Q < MI ? Q * 1024 : (int)SmallRing<MI>::kSlabA + (Q - MI) * 1024), \
                       "v"(Q < MI ? w.voff[Q < 0 ? 0 : Q % MI] : small_voff_b(w, Q < MI ? 0 : Q - MI)), "s"(Q < MI ? w.ga : w.gb) : "memory", "m0", "scc")
  if constexpr (small_is_fp8(OP)) {
    constexpr int i = S / 4, j = S % 4;
    const i32x8v a8 = __builtin_shufflevector(f.a_lo[i], f.a_hi[i], 0, 1, 2, 3, 4, 5, 6, 7);
    const i32x8v b8 = __builtin_shufflevector(f.b_lo[j], f.b_hi[j], 0, 1, 2, 3, 4, 5, 6, 7);
    if constexpr (OP == kQuadE5m2) { S_MFMA("v_mfma_f32_16x16x128_f8f6f4", " blgp:1", 4 * i + j, b8, a8); }
    else { S_MFMA("v_mfma_f32_16x16x128_f8f6f4", "", 4 * i + j, b8, a8); }
  } else {
    constexpr int i = S / 8, hi = (S % 8) / 4, j = S % 4;
    const i32x4v &a = hi ? f.a_hi[i] : f.a_lo[i], &b = hi ? f.b_hi[j] : f.b_lo[j];
    if constexpr (OP == kQuadBf16) { S_MFMA("v_mfma_f32_16x16x32_bf16", "", 4 * i + j, b, a); }
    else if constexpr (OP == kQuadF16) { S_MFMA("v_mfma_f32_16x16x32_f16", "", 4 * i + j, b, a); }
    else { S_MFMA("v_mfma_i32_16x16x64_i8", "", 4 * i + j, b, a); }
  }
#undef S_MFMA
}

// Fragment read number R of 2 (MI + 4): the B fragments (rows 16j.. of the wave's part of the B slab), then the A fragments.
template <int R, int MI>
__device__ __forceinline__ void small_read(SmallFragsOf<MI> &f, const SmallWalkOf<MI> &w) {
  constexpr int i = (R < 8 ? R : R - 8) / 2, off = i * 16 * kRowBytes;
  if constexpr (R < 8) {
    if constexpr (R % 2 == 0) S_DS_READ(f.b_lo[i], w.b0, off); else S_DS_READ(f.b_hi[i], w.b1, off);
  } else {
    if constexpr (R % 2 == 0) S_DS_READ(f.a_lo[i], w.a0, off); else S_DS_READ(f.a_hi[i], w.a1, off);
  }
}

// Load number Q of MI + 4 of a slab on its own (filling the ring before the first step).
template <int Q, int MI = 4, class Walk>
__device__ __forceinline__ void small_load(const Walk &w) {
  if constexpr (Q < MI) MI355_LOAD_LDS(w.voff[Q], w.ga, w.dst + Q * 1024u);
  else MI355_LOAD_LDS(small_voff_b(w, Q - MI), w.gb, small_dst_b(w) + SmallRing<MI>::kSlabA + (Q - MI) * 1024u);
}

// The reads of a fragment set have arrived.  The registers ride along so that nothing that uses them can be placed
// before the wait (an asm statement takes 30 operands at most: two statements).  Between issuing reads and this wait
// there must be no branch: where paths join, the compiler may copy registers, and it does not know that these are
// still being written.
__device__ __forceinline__ void small_arrived(SmallFrags &f) {
  asm volatile("s_waitcnt lgkmcnt(0)" : S_TIE4(f.a_lo), S_TIE4(f.a_hi)
               : "v"(f.b_lo[0]), "v"(f.b_lo[1]), "v"(f.b_lo[2]), "v"(f.b_lo[3]), "v"(f.b_hi[0]), "v"(f.b_hi[1]), "v"(f.b_hi[2]), "v"(f.b_hi[3]));
  asm volatile("" : S_TIE4(f.b_lo), S_TIE4(f.b_hi));
}
__device__ __forceinline__ void small_arrived(SmallFragsOf<8> &f) {
  asm volatile("s_waitcnt lgkmcnt(0)" : S_TIE4(f.a_lo), "+v"(f.a_lo[4]), "+v"(f.a_lo[5]), "+v"(f.a_lo[6]), "+v"(f.a_lo[7])
               : "v"(f.a_hi[0]), "v"(f.a_hi[1]), "v"(f.a_hi[2]), "v"(f.a_hi[3]), "v"(f.a_hi[4]), "v"(f.a_hi[5]), "v"(f.a_hi[6]), "v"(f.a_hi[7]));
  asm volatile("" : S_TIE4(f.a_hi), "+v"(f.a_hi[4]), "+v"(f.a_hi[5]), "+v"(f.a_hi[6]), "+v"(f.a_hi[7]));
  asm volatile("" : S_TIE4(f.b_lo), S_TIE4(f.b_hi));
}

// One step: the matrix instructions on `cur`, and in their shadow the 16 (24) reads of the next step's fragments into
// `nxt` and the 8 (12) loads of the slab four (three) steps on.  A lone wave issues an instruction every four cycles or so, whatever
// it is, so a 16-cycle matrix instruction has room for three others beside it: the loads ride one on every fourth
// matrix instruction (every second for fp8, every fifth where there are 64) over the whole step, the reads one behind each
// of the first 16 (24; fp8: two behind each of the first 8), so that they have arrived when the rest is through.
// LAST: the step behind which nothing follows reads and loads nothing.
template <int OP, bool LAST, int S, int MI, class Walk>
__device__ __forceinline__ void small_slot(const SmallFragsOf<MI> &cur, SmallFragsOf<MI> &nxt, const Walk &w) {
  constexpr int kEvery = small_is_fp8(OP) ? 2 : MI == 4 ? 4 : 5;
  if constexpr (LAST || S % kEvery != 0 || S / kEvery >= SmallRing<MI>::kLoads) small_mfma<OP, S>(cur, w);
  else small_mfma<OP, S, S / kEvery>(cur, w);
  if constexpr (LAST) return;
  if constexpr (small_is_fp8(OP)) {
    if constexpr (S < 8) { small_read<2 * S>(nxt, w); small_read<2 * S + 1>(nxt, w); }
  } else {
    if constexpr (S < SmallRing<MI>::kReads) small_read<S>(nxt, w);
  }
}

template <int OP, bool LAST, int MI, class Walk, int... S>
__device__ __forceinline__ void small_step(std::integer_sequence<int, S...>, SmallFragsOf<MI> &cur, SmallFragsOf<MI> &nxt, const Walk &w) {
  // This wave's loads of the slab to read have landed (loads complete in order, 8 per slab; the two slabs behind it
  // may be in flight; tall: 12, and one); after the barrier everybody's have, and every wave has `cur` in registers, so
  // that the slot `cur` came from can be filled by the loads of the next step (tall: of this one).
  if constexpr (!LAST) asm volatile("s_waitcnt vmcnt(%0)\n s_barrier" :: "n"(SmallRing<MI>::kLoads * (SmallRing<MI>::kAhead - 2)) : "memory");
  (small_slot<OP, LAST, S>(cur, nxt, w), ...);
  if constexpr (!LAST) small_arrived(nxt);
}

}  // namespace
