// What becomes of a wave's 128x128 sums in the kernels on 256x256 tiles (ffn_quad.hip, ffn_across.hip): finished from the
// accumulation registers, stored and cleared.
#pragma once
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
  // streams: past the caches.
  __device__ __forceinline__ void store(const float (&x)[2][4], bool whole, bool edge, bool some, int32_t rem, bool streams) {
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
      if (whole) {
        // (as text: the compiler merges the two arms of a branch that differ only in the cache policy of a store; the wait
        // state keeps a following write to its data registers off, which the compiler sees to for its own stores)
        const i32x4v bits = {(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
        if (streams) asm volatile("global_store_dwordx4 %0, %1, off nt\n s_nop 0" :: "v"(at), "v"(bits) : "memory");
        else __builtin_memcpy(__builtin_assume_aligned(at, 2), w, 16);
      }
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
  static constexpr uint32_t kManyRounds = 4;
  // A store's pieces are 64 bytes of each of 16 rows: whole ones where every row starts on 64 bytes.  Others would reach
  // memory in two parts (7525x8347x64 fp16 with both sums kept: 417 us past the caches, 235 through them).
  __device__ __forceinline__ static bool on_64_bytes(const FfnOut &o) {
    uint64_t bits = (uint64_t)(uintptr_t)o.c | o.ldc * PairOut<TYPE>::kElem;
    if (o.g) bits |= (uint64_t)(uintptr_t)o.g | (uint64_t)(uintptr_t)o.u | o.ldg * PairOut<TYPE>::kElem;
    return (bits & 63u) == 0u;
  }
  const FfnProduct &p;
  uint32_t row0, col0, lane;   // the lane's first row, the wave's first column
  // The outputs of a gated 16-bit product of many rounds go past the caches, where up to three of them would only push out
  // operands that later rounds read again (glu 8192x8192x4096 with G and U, 8 rounds: 743 -> 718 us; 2048 rows, 2 rounds:
  // 177 -> 186 us, the last round's stores being all that is left to wait for; int8, whose operands are half as large:
  // 2 % slower)
  bool many_rounds;
  float sa[8], plain;
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
        if constexpr (OP == kQuadF16 && EPI == kEpiPlain) x[t][e] *= plain;
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
          g.store(x, whole, edge, row && !whole, rem, EPI == kEpiGated && many_rounds);
          u.store(y, whole, edge, row && !whole, rem, EPI == kEpiGated && many_rounds);
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
    c.store(x, whole, edge, row && !whole, rem, EPI == kEpiGated && many_rounds);
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
    if constexpr (OP == kQuadF16 && EPI == kEpiPlain) plain = ffn_plain_factor(p.out);
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

}  // namespace
