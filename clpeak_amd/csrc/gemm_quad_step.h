// The step of the four-wave GEMM kernel on 256x256 tiles: what gemm_quad.hip describes, shared by its kernel and by the
// feed-forward products (ffn_quad.hip), whose operands may end inside a tile.
#pragma once
#include "mfma_common.h"
#include "gemm_ring.h"
#include "gemm_quad.h"
#include <utility>

namespace {

constexpr int kQuadThreads = 256;
constexpr uint32_t kSlotA0 = 0, kSlotB0 = 3u * kSlabBytes;   // three A slots, then two B slots

struct QuadFrags {
  i32x4v b_lo[2][8], b_hi[2][8];   // two register sets of B fragments (current step / next step)
  i32x4v a_lo[4], a_hi[4];         // four rotating A fragment slots: row i lives in slot i mod 4
  i32x4v sa[2], sb[2];             // block-scaled kind: the scale bytes of the current / next step (see quad_mx_scales)
};

struct QuadWalk {
  uint32_t a_cur, a_cur_hi;  // LDS address of this lane's A fragment of row 0, first / second K half, in the slot of slab s
  uint32_t a_nxt, a_nxt_hi;  // ... in the slot of slab s+1
  uint32_t lane_a;           // ... within an A slot
  uint32_t b_base, b_base_hi;   // the same for the B fragment, in B slot 0 (B slot 1 is reached through the offset field)
  uint32_t off_cur, off_nxt, off_dst;   // byte offsets of the A slots of slabs s, s+1 and s+2 (uniform)
  uint32_t dst_a;            // LDS destination of this wave's A rows of slab s+2 (uniform)
  uint32_t dst_wave;         // this wave's rows within a slot (uniform)
  uint64_t ga, gb;           // global addresses of this wave's first A / B row of slab s+2 (uniform)
  uint32_t voff[8];          // this lane's byte offset from ga / gb for each of the wave's 8 loads of a slab
  uint32_t first;            // the step is the first of a tile (uniform)
  uint64_t sa_next, sb_next; // block-scaled kind: addresses of the next step's 1 KiB of A / B scale bytes (uniform)
  uint32_t s_off;            // ... and this lane's offset there
};

// Where an operand may end inside a tile its rows past the end are read as its last one, so that the lanes' offsets differ
// between A (voff) and B.
struct QuadEdgeWalk : QuadWalk {
  uint32_t voff_b[8];
};
__device__ __forceinline__ uint32_t quad_voff_b(const QuadWalk &w, int q) { return w.voff[q]; }
__device__ __forceinline__ uint32_t quad_voff_b(const QuadEdgeWalk &w, int q) { return w.voff_b[q]; }

#define Q_DS_READ(dst, addr, off) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(dst) : "v"(addr), "n"(off))
#define Q_WAIT_LGKM(n) asm volatile("s_waitcnt lgkmcnt(%0)" :: "n"(n) : "memory")

// The accumulators are the accumulation registers a[0:255], named in the instruction text: tile (i, j) of the wave is
// a[4T : 4T+3], T = 8i + j.  The compiler is told once that they are taken (quad_claim_accumulators) and never sees them
// as values: with 256 of 256 in use as operands of its own it finds no allocation without spills.
//
// One matrix instruction of a pair kind, optionally with one direct-to-LDS load riding along: M0 is set before the
// matrix instruction (which is the wait state M0 needs before a load reads it) and the load is issued behind it.
#define Q_INSN_BF16 "v_mfma_f32_16x16x32_bf16"
#define Q_INSN_F16 "v_mfma_f32_16x16x32_f16"
#define Q_INSN_I8 "v_mfma_i32_16x16x64_i8"
#define Q_INSN_F8 "v_mfma_f32_16x16x128_f8f6f4"
template <int OP, int T>
__device__ __forceinline__ void q_mfma(const i32x4v &b, const i32x4v &a) {
#define Q_PLAIN(insn) asm volatile(insn " a[%2:%3], %0, %1, a[%2:%3]" :: "v"(b), "v"(a), "n"(4 * T), "n"(4 * T + 3))
  if constexpr (OP == kQuadBf16) Q_PLAIN(Q_INSN_BF16);
  else if constexpr (OP == kQuadF16) Q_PLAIN(Q_INSN_F16);
  else Q_PLAIN(Q_INSN_I8);
#undef Q_PLAIN
}
template <int OP, int T, int IMM>
__device__ __forceinline__ void q_mfma_load(const i32x4v &b, const i32x4v &a, uint32_t dst, uint32_t voff, uint64_t base) {
#define Q_WITH_LOAD(insn)                                                                                              \
  asm volatile("s_add_u32 m0, %4, %5\n " insn " a[%2:%3], %0, %1, a[%2:%3]\n global_load_lds_dwordx4 %6, %7"           \
               :: "v"(b), "v"(a), "n"(4 * T), "n"(4 * T + 3), "s"(dst), "n"(IMM), "v"(voff), "s"(base) : "memory", "m0", "scc")
  if constexpr (OP == kQuadBf16) Q_WITH_LOAD(Q_INSN_BF16);
  else if constexpr (OP == kQuadF16) Q_WITH_LOAD(Q_INSN_F16);
  else Q_WITH_LOAD(Q_INSN_I8);
#undef Q_WITH_LOAD
}
// fp8: one K=128 instruction on the 32-byte operands (e5m2 A: format field blgp, the A fragment being the second
// source of the transposed product).
template <int OP, int T>
__device__ __forceinline__ void q_mfma8(const i32x8v &b, const i32x8v &a) {
  if constexpr (OP == kQuadE5m2) asm volatile(Q_INSN_F8 " a[%2:%3], %0, %1, a[%2:%3] blgp:1" :: "v"(b), "v"(a), "n"(4 * T), "n"(4 * T + 3));
  else asm volatile(Q_INSN_F8 " a[%2:%3], %0, %1, a[%2:%3]" :: "v"(b), "v"(a), "n"(4 * T), "n"(4 * T + 3));
}
template <int OP, int T, int IMM>
__device__ __forceinline__ void q_mfma8_load(const i32x8v &b, const i32x8v &a, uint32_t dst, uint32_t voff, uint64_t base) {
#define Q_WITH_LOAD8(fmt)                                                                                              \
  asm volatile("s_add_u32 m0, %4, %5\n " Q_INSN_F8 " a[%2:%3], %0, %1, a[%2:%3]" fmt "\n global_load_lds_dwordx4 %6, %7" \
               :: "v"(b), "v"(a), "n"(4 * T), "n"(4 * T + 3), "s"(dst), "n"(IMM), "v"(voff), "s"(base) : "memory", "m0", "scc")
  if constexpr (OP == kQuadE5m2) Q_WITH_LOAD8(" blgp:1");
  else Q_WITH_LOAD8("");
#undef Q_WITH_LOAD8
}

// Block-scaled e2m1 (OCP MXFP4): a lane's 16-byte chunk is the 32 codes of one scale block, so a slot is again a pair of
// K=128 instructions on the two K halves, each with the scale bytes of its blocks.  A wave's scale bytes of a step are
// 16 bytes per lane and operand, byte 2i+h belonging to fragment i, K half h: the instruction takes byte
// (op_sel + 2 * op_sel_hi) of the register it is given: op_sel = K half, op_sel_hi = parity of the fragment, register =
// fragment / 2.  They do not pass through LDS: a pre-pass (gemm_mxfp4.hip) has written them in this order, and a step
// loads those of the next step with one instruction per operand, its oldest loads.
#define Q_INSN_MX "v_mfma_scale_f32_16x16x128_f8f6f4"
template <int T, int H, int JB, int IB>
__device__ __forceinline__ void q_mfma_mx(const i32x4v &b, const i32x4v &a, int sb, int sa) {
  asm volatile(Q_INSN_MX " a[%2:%3], %0, %1, a[%2:%3], %4, %5 op_sel:[%6,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
               :: "v"(b), "v"(a), "n"(4 * T), "n"(4 * T + 3), "v"(sb), "v"(sa), "n"(H), "n"(JB), "n"(IB));
}
template <int T, int JB, int IB, int IMM>
__device__ __forceinline__ void q_mfma_mx_load(const i32x4v &b, const i32x4v &a, int sb, int sa, uint32_t dst, uint32_t voff, uint64_t base) {
  asm volatile("s_add_u32 m0, %8, %9\n " Q_INSN_MX " a[%2:%3], %0, %1, a[%2:%3], %4, %5 op_sel:[0,0,0] op_sel_hi:[%6,%7,0] cbsz:4 blgp:4\n"
               " global_load_lds_dwordx4 %10, %11"
               :: "v"(b), "v"(a), "n"(4 * T), "n"(4 * T + 3), "v"(sb), "v"(sa), "n"(JB), "n"(IB), "s"(dst), "n"(IMM), "v"(voff), "s"(base)
               : "memory", "m0", "scc");
}

constexpr bool quad_is_fp8(int op) { return op == kQuadE4m3 || op == kQuadE5m2; }

// Slot P of a step of parity PAR (the B register set in use): row i = P / 8 of the A fragments, B fragment j = P % 8.
// Besides its matrix instructions a slot carries its share of everything else a step does, so that nothing is left
// for the boundary between two steps, where a single wave per SIMD has nothing to hide it behind:
//   slots 0, 3, .. 45   one load each (8 of B rows, then 8 of A rows, of slab s+2): the texture path takes a load's
//                       1 KiB in 16 cycles, the four waves' 64 KiB of a step in half of the step
//   slots 8i            the reads of A row i+2 go out (rows 6, 7: rows 0, 1 of slab s+1), then row i must have arrived
//   slot 40             barrier X
//   slots 41..56        the burst of B(s+1)
//   slots 23, 46, 47    the fetch addresses and the A slots move on; slot 57: the fragment addresses
//   slot 60             every read has arrived; barrier Y of the NEXT step
#define Q_PIN() __builtin_amdgcn_sched_barrier(0)
constexpr int kLoadEvery = 3;   // the wave's 16 loads of a slab ride on slots 0, 3, 6, .. 45 (every 2: 5 % slower; 4: the same)
constexpr int kAhead = 2;       // rows between the read of an A fragment and its use (at most 3: four register slots; 3: the same)
constexpr int kSlotX = 40;      // barrier X follows this slot; the 16 reads of the burst follow it, one per slot (36, 43: the same)
constexpr int quad_burst_reads(int from, int to) {   // reads of the burst issued in slots from..to
  int n = 0;
  for (int p = from; p <= to; p++) n += p > kSlotX && p <= kSlotX + 16;
  return n;
}
// loads of the step's own slab that are issued before barrier X (they are the ones that may still be in flight there)
constexpr int kKeepAtX = kSlotX / kLoadEvery + 1 < 16 ? kSlotX / kLoadEvery + 1 : 16;
static_assert(15 * kLoadEvery + 2 <= 57, "the loads of a step and the bookkeeping behind them end before the addresses move on");
static_assert(kAhead >= 1 && kAhead <= 3 && kSlotX + 16 < 60 && kSlotX >= 46 - 16, "schedule of a step");
template <int OP, int PAR, int P, class Walk>
__device__ __forceinline__ void quad_slot(QuadFrags &f, Walk &w) {
  constexpr int i = P / 8, j = P % 8, sl = i % 4, T = P;
  if constexpr (j == 0) {
    // the reads of the A row kAhead rows on go out (past row 7: of the next slab), then this row's fragment must have
    // arrived: reads return in order, so the count is that of the reads issued behind it (the counter holds 15)
    constexpr int r = i + kAhead;
    if constexpr (r <= 7) {
      Q_DS_READ(f.a_lo[r % 4], w.a_cur, r * 2048);
      Q_DS_READ(f.a_hi[r % 4], w.a_cur_hi, r * 2048);
    } else {
      Q_DS_READ(f.a_lo[r % 4], w.a_nxt, (r - 8) * 2048);
      Q_DS_READ(f.a_hi[r % 4], w.a_nxt_hi, (r - 8) * 2048);
    }
    if constexpr (i >= kAhead) {
      constexpr int behind = 2 * kAhead + quad_burst_reads(8 * (i - kAhead), 8 * i - 1);
      Q_WAIT_LGKM(behind < 15 ? behind : 15);
    }
  }
  constexpr int q = P / kLoadEvery;
  constexpr bool with_load = P % kLoadEvery == 0 && q < 16;
  if constexpr (quad_is_fp8(OP)) {
    const i32x8v b8 = __builtin_shufflevector(f.b_lo[PAR][j], f.b_hi[PAR][j], 0, 1, 2, 3, 4, 5, 6, 7);
    const i32x8v a8 = __builtin_shufflevector(f.a_lo[sl], f.a_hi[sl], 0, 1, 2, 3, 4, 5, 6, 7);
    if constexpr (with_load && q < 8) q_mfma8_load<OP, T, kSlotB0 + PAR * kSlabBytes + q * 1024>(b8, a8, w.dst_wave, quad_voff_b(w, q), w.gb);
    else if constexpr (with_load) q_mfma8_load<OP, T, (q - 8) * 1024>(b8, a8, w.dst_a, w.voff[q - 8], w.ga);
    else q_mfma8<OP, T>(b8, a8);
  } else if constexpr (OP == kQuadMx) {
    const int sb = f.sb[PAR][j / 2], sa = f.sa[PAR][i / 2];
    if constexpr (with_load && q < 8)
      q_mfma_mx_load<T, j % 2, i % 2, kSlotB0 + PAR * kSlabBytes + q * 1024>(f.b_lo[PAR][j], f.a_lo[sl], sb, sa, w.dst_wave, quad_voff_b(w, q), w.gb);
    else if constexpr (with_load)
      q_mfma_mx_load<T, j % 2, i % 2, (q - 8) * 1024>(f.b_lo[PAR][j], f.a_lo[sl], sb, sa, w.dst_a, w.voff[q - 8], w.ga);
    else
      q_mfma_mx<T, 0, j % 2, i % 2>(f.b_lo[PAR][j], f.a_lo[sl], sb, sa);
    q_mfma_mx<T, 1, j % 2, i % 2>(f.b_hi[PAR][j], f.a_hi[sl], sb, sa);
  } else {
    if constexpr (with_load && q < 8)
      q_mfma_load<OP, T, kSlotB0 + PAR * kSlabBytes + q * 1024>(f.b_lo[PAR][j], f.a_lo[sl], w.dst_wave, quad_voff_b(w, q), w.gb);
    else if constexpr (with_load)
      q_mfma_load<OP, T, (q - 8) * 1024>(f.b_lo[PAR][j], f.a_lo[sl], w.dst_a, w.voff[q - 8], w.ga);
    else
      q_mfma<OP, T>(f.b_lo[PAR][j], f.a_lo[sl]);
    q_mfma<OP, T>(f.b_hi[PAR][j], f.a_hi[sl]);
  }
  if constexpr (P == kSlotX) {
    // barrier X: this wave's loads of slab s+1 have landed (the 16 of slab s+2 may be in flight).  In the first step
    // of a tile that wait was done before the stores of the tile before, which must not be counted here.
    asm volatile("s_cmp_lg_u32 %0, 0\n s_cbranch_scc1 1f\n s_waitcnt vmcnt(%1)\n1:\n s_barrier" :: "s"(w.first), "n"(kKeepAtX + (OP == kQuadMx ? 2 : 0)) : "memory", "scc");
  }
  if constexpr (P > kSlotX && P <= kSlotX + 16) {
    // the burst: B fragment r/2, K half r%2 of slab s+1 into the other register set
    constexpr int r = P - kSlotX - 1, jb = r / 2;
    if constexpr (r % 2 == 0) Q_DS_READ(f.b_lo[PAR ^ 1][jb], w.b_base, (PAR ^ 1) * kSlabBytes + jb * 2048);
    else Q_DS_READ(f.b_hi[PAR ^ 1][jb], w.b_base_hi, (PAR ^ 1) * kSlabBytes + jb * 2048);
  }
  if constexpr (P == 7 * kLoadEvery + 1) { Q_PIN(); w.gb += kRowBytes; Q_PIN(); }
  if constexpr (OP == kQuadMx && P == 5) { Q_PIN(); w.sa_next += 1024; w.sb_next += 1024; Q_PIN(); }
  if constexpr (P == kSlotX + 1) { Q_PIN(); w.first = 0; Q_PIN(); }
  if constexpr (P == 15 * kLoadEvery + 1) { Q_PIN(); w.ga += kRowBytes; Q_PIN(); }
  if constexpr (P == 15 * kLoadEvery + 2) {
    Q_PIN();
    const uint32_t t = w.off_cur;
    w.off_cur = w.off_nxt; w.off_nxt = w.off_dst; w.off_dst = t;
    w.dst_a = w.dst_wave + w.off_dst;
    Q_PIN();
  }
  if constexpr (P == 57) {
    Q_PIN();
    w.a_cur = w.a_nxt; w.a_cur_hi = w.a_nxt_hi;
    w.a_nxt = w.lane_a + w.off_nxt; w.a_nxt_hi = w.a_nxt ^ 64u;
    Q_PIN();
  }
  if constexpr (P == 60) {
    // Everything read in this step has arrived; the registers ride along so that nothing that uses them (a copy the
    // compiler might place where control flow joins, the next step) can come before the wait.  Then barrier Y of the
    // next step: every wave has read B(s+1) and all of A(s), whose slots the loads of the next step overwrite.
#define Q_TIE8(x) "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7])
    asm volatile("s_waitcnt lgkmcnt(0)\n s_barrier"
                 : Q_TIE8(f.b_lo[PAR ^ 1]), Q_TIE8(f.b_hi[PAR ^ 1]), "+v"(f.a_lo[0]), "+v"(f.a_hi[0]), "+v"(f.a_lo[1]), "+v"(f.a_hi[1]),
                   "+v"(f.a_lo[2]), "+v"(f.a_hi[2])
                 :: "memory");
  }
}

__device__ __forceinline__ void quad_mx_scales(i32x4v &sa, i32x4v &sb, const QuadWalk &w) {
  asm volatile("global_load_dwordx4 %0, %1, %2" : "=v"(sa) : "v"(w.s_off), "s"(w.sa_next) : "memory");
  asm volatile("global_load_dwordx4 %0, %1, %2" : "=v"(sb) : "v"(w.s_off), "s"(w.sb_next) : "memory");
}

template <int OP, int PAR, class Walk, int... Ps>
__device__ __forceinline__ void quad_step(std::integer_sequence<int, Ps...>, QuadFrags &f, Walk &w) {
  if constexpr (OP == kQuadMx) {
    // this step's scale bytes were requested at the top of the step before, ahead of its 16 loads into LDS (in the first
    // step of a tile they were waited for before the stores of the tile before); then those of the next step go out
    asm volatile("s_cmp_lg_u32 %2, 0\n s_cbranch_scc1 1f\n s_waitcnt vmcnt(16)\n1:" : "+v"(f.sa[PAR]), "+v"(f.sb[PAR]) : "s"(w.first) : "scc");
    quad_mx_scales(f.sa[PAR ^ 1], f.sb[PAR ^ 1], w);
  }
  (quad_slot<OP, PAR, Ps>(f, w), ...);
}

// The accumulation registers belong to the hand-written code from here on.
__device__ __forceinline__ void quad_claim_accumulators() {
#define Q_A8(n) "a" #n "0", "a" #n "1", "a" #n "2", "a" #n "3", "a" #n "4", "a" #n "5", "a" #n "6", "a" #n "7", "a" #n "8", "a" #n "9"
  asm volatile("" ::: "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", Q_A8(1), Q_A8(2), Q_A8(3), Q_A8(4), Q_A8(5), Q_A8(6),
               Q_A8(7), Q_A8(8), Q_A8(9), Q_A8(10), Q_A8(11), Q_A8(12), Q_A8(13), Q_A8(14), Q_A8(15), Q_A8(16), Q_A8(17), Q_A8(18),
               Q_A8(19), Q_A8(20), Q_A8(21), Q_A8(22), Q_A8(23), Q_A8(24), "a250", "a251", "a252", "a253", "a254", "a255");
#undef Q_A8
}

// Tile T of the wave out of the accumulation registers (as raw bits), and zero in its place.
template <int T>
__device__ __forceinline__ i32x4v quad_take_tile() {
  int v0, v1, v2, v3;
  asm volatile("v_accvgpr_read_b32 %0, a[%4]\n v_accvgpr_read_b32 %1, a[%5]\n v_accvgpr_read_b32 %2, a[%6]\n v_accvgpr_read_b32 %3, a[%7]\n"
               " v_accvgpr_write_b32 a[%4], 0\n v_accvgpr_write_b32 a[%5], 0\n v_accvgpr_write_b32 a[%6], 0\n v_accvgpr_write_b32 a[%7], 0"
               : "=&v"(v0), "=&v"(v1), "=&v"(v2), "=&v"(v3) : "n"(4 * T), "n"(4 * T + 1), "n"(4 * T + 2), "n"(4 * T + 3));
  return (i32x4v){v0, v1, v2, v3};
}
template <int R>
__device__ __forceinline__ void quad_zero_register() { asm volatile("v_accvgpr_write_b32 a[%0], 0" :: "n"(R)); }
template <int... Rs>
__device__ __forceinline__ void quad_zero_accumulators(std::integer_sequence<int, Rs...>) {
  (quad_zero_register<Rs>(), ...);
  asm volatile("s_nop 7");
}

}  // namespace
