// Tile product of the vocabulary losses (vocab_loss.hip): one BM x BN tile of  C[m][n] = sum_k A(m, k) B(n, k)  on the matrix
// cores, 16-bit operands, fp32 accumulation, for operands stored either way round:
//   row operand   [m][k], the contraction contiguous                (h and W of the scores, dS of the hidden gradient)
//   col operand   [k][m], the contraction is the row index          (W of the hidden gradient, dS and h of the weight gradient)
// so that neither W nor dS nor h is ever copied transposed: a col operand is staged as it lies in memory and its fragments come
// out of LDS through the hardware transpose read (ds_read_b64_tr_b16).
//
// PL = 1: one 16-bit plane, 64 contraction steps a stage.  PL = 2: an fp32 operand as two fp16 planes x = hi + lo (22 bits, the
// caller scales the tensor by a power of two so that neither plane leaves fp16's normal range), 32 contraction steps a stage,
// three products hi hi + hi lo + lo hi: what is dropped is 2^-22 of a term.
//
// LDS image of a stage, either way 128 bytes a row (8 chunks of 16 bytes), so that the LDS-DMA (destination lane-linear) can fill
// it with whole 1-KiB pieces and the bank swizzle sits on its SOURCE side:
//   row operand: row = output row; chunk c holds k 8c .. 8c+7 (PL = 2: chunks 0-3 hi, 4-7 lo), stored at c ^ ((row >> 1) & 7):
//                the 16 rows of a ds_read_b128 lane group hit 16 different 16-byte slots of 256 bytes
//   col operand: panels of 64 columns; row = contraction step (PL = 2: rows 0-31 hi, 32-63 lo), chunk c stored at
//                c ^ (((row >> 1) & 1) << 2): the 4 rows x 64 bytes that half a wave's transpose read takes are 256 different bytes
// Both hand lane l of a 32x32x16 fragment its row (or column) l & 31 at contraction steps 8 (l >> 5) .. + 7.
#pragma once
#include <type_traits>

#include "common.h"

namespace vocab {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

// 64 x 16 bytes from base + offset (the base and the destination alike for the wave) to LDS.  Inline assembly, because behind the
// builtin the compiler waits for every transfer in flight before the next read of LDS, the current stage's fragments among them:
// whoever reads the destination waits for vmcnt and passes a barrier first.
__device__ __forceinline__ void dma16(const unsigned short* base, unsigned byte_offset, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(byte_offset), "s"(base) : "memory", "m0");
}

template <bool F16>
__device__ __forceinline__ f32x16_t mma(s16x8_t a, s16x8_t b, f32x16_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// sum of 8 16-bit values + c
template <bool F16>
__device__ __forceinline__ float sum8(s16x8_t v, float c) {
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  typedef short s16x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const s16x2_t x = {v[2 * e], v[2 * e + 1]};
    if constexpr (F16) {
      const f16x2_t one = {(_Float16)1.f, (_Float16)1.f};
      c = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, x), one, c, false);
    } else {
      const bf16x2_t one = {(__bf16)1.f, (__bf16)1.f};
      c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x), one, c, false);
    }
  }
  return c;
}

struct Operand {
  const unsigned short* p;
  int64_t ld;       // elements between rows of the stored matrix
  int64_t plane;    // elements between the hi and the lo plane of a row (PL = 2)
  int64_t rows;     // stored rows that may be read; what lies past them is read as the last one again
  int64_t cols;     // stored columns that may be read (a multiple of 8), likewise
};

template <bool F16_, int PL_, int BM_, int BN_, int WM_, int WN_, bool COLA_, bool COLB_>
struct Tile {
  static constexpr bool F16 = F16_, COLA = COLA_, COLB = COLB_;
  static constexpr int PL = PL_, BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int BK = PL == 1 ? 64 : 32;
  static constexpr int WAVES_N = BN / WN, NW = (BM / WM) * WAVES_N, THREADS = NW * 64;
  static constexpr int TM = WM / 32, TN = WN / 32;
  static constexpr int STAGE = (BM + BN) * 64;           // u16 a stage
  static constexpr int PIECES = (BM + BN) / 8, PPW = PIECES / NW;
  static constexpr int LDS = 2 * STAGE;                  // u16 of the two-stage ring
  static_assert(PIECES % NW == 0 && WM % 32 == 0 && WN % 32 == 0 && BM % 64 == 0 && BN % 64 == 0, "tile shape");

  using Acc = f32x16_t[TM][TN];

  // Accumulates contraction steps [k0, k0 + nk * BK) of the tile at (bm, bn).  Lane l ends with, for output row
  // bm + wr WM + 32 i + (l & 31), the columns bn + wc WN + 32 j + 8 (q >> 2) + 4 (l >> 5) + (q & 3), q < 16: the B operand is the
  // first of the matrix instruction, so a lane holds runs of 4 columns of one row.  Every wave of the workgroup calls it.
  //
  // Two-stage ring, fragments one sub-step (16 contraction steps) ahead in registers: in front of the last sub-step of a stage
  // every fragment of the stage is in registers, so ONE barrier says both that the next stage has landed and that this one's
  // buffer is free; the transfers of the stage after next start right there and have a whole stage of matrix work to land.
  //
  // SUMA and sum (alike for the wave): asum (TM values) also takes the sums of A over the contraction, lane l those of the steps
  // that it holds of row 32 i + (l & 31); lanes l and l ^ 32 together hold all.
  template <bool SUMA = false>
  static __device__ __forceinline__ void run(const Operand& A, const Operand& B, int64_t bm, int64_t bn, int64_t k0, int nk,
                                             unsigned short* smem, Acc& acc, float* asum = nullptr, bool sum = false) {
    if (nk <= 0) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WAVES_N, wc = wave % WAVES_N;

    // ---- the DMA pieces of this wave: 8 image rows x 128 bytes each; byte offsets from the operand's first tile element
    static_assert(BM / 8 % PPW == 0 || PPW % (BM / 8) == 0, "a wave's pieces belong to one operand");
    const bool isA = wave * PPW < BM / 8;
    const Operand& O = isA ? A : B;
    const bool col = isA ? COLA : COLB;
    const int64_t b0 = isA ? bm : bn, r0 = b0 < O.rows ? b0 : O.rows - 1;      // (a row operand's first row)
    const unsigned short* base = O.p + (col ? k0 * O.ld : r0 * O.ld + k0);
    const int64_t step = col ? BK * O.ld : BK;
    const unsigned ld = (unsigned)O.ld;
    unsigned off[PPW];
    [[maybe_unused]] int krow[PPW];
#pragma unroll
    for (int i = 0; i < PPW; ++i) {
      const int q = wave * PPW + i - (isA ? 0 : BM / 8), slot = lane & 7;
      if (!col) {
        const int64_t last = O.rows - 1 - r0;
        int row = q * 8 + (lane >> 3);
        const int c = slot ^ ((row >> 1) & 7);
        if (row > last) row = (int)last;
        off[i] = ((unsigned)row * ld + (PL == 2 ? (c >> 2) * (unsigned)O.plane + (c & 3) * 8 : c * 8)) * 2;
        krow[i] = 0;
      } else {
        const int panel = q >> 3, rr = (q & 7) * 8 + (lane >> 3);
        const int c = slot ^ (((rr >> 1) & 1) << 2);
        int64_t cc = b0 + panel * 64 + c * 8;
        if (cc > O.cols - 8) cc = O.cols - 8;
        krow[i] = PL == 2 ? rr & 31 : rr;
        off[i] = ((unsigned)krow[i] * ld + (PL == 2 ? (rr >> 5) * (unsigned)O.plane : 0) + (unsigned)cc) * 2;
      }
    }
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned short*)smem + wave * PPW * 1024;
    auto issue_piece = [&](int kt, int i, bool tail) {
      const unsigned short* from = base + kt * step;
      unsigned o = off[i];
      if ((COLA || COLB) && tail) {           // contraction rows past the last stored one: that one again
        const int64_t first = k0 + (int64_t)kt * BK, have = O.rows - 1 - first;
        const int keep = have < 0 ? 0 : krow[i] < have ? krow[i] : (int)have;
        if (have < 0) from = O.p + (O.rows - 1) * O.ld;
        o -= (unsigned)(krow[i] - keep) * ld * 2;
      }
      dma16(from, o, lds0 + (kt & 1) * (STAGE * 2) + i * 1024);
    };
    auto is_tail = [&](int kt) { return (COLA || COLB) && col && k0 + (int64_t)(kt + 1) * BK > O.rows; };
    auto issue = [&](int kt) {
      const bool tail = is_tail(kt);
#pragma unroll
      for (int i = 0; i < PPW; ++i) issue_piece(kt, i, tail);
    };

    // ---- fragments
    const int l31 = lane & 31, half = lane >> 5, j = lane & 15, g = lane >> 4;
    auto frag = [&](auto colc, const unsigned short* sec, int w0, int ks, int lo) -> s16x8_t {
      if constexpr (!decltype(colc)::value) {
        const int row = w0 + l31, c = (2 * ks + half + lo * 4) ^ ((l31 >> 1) & 7);
        return *reinterpret_cast<const s16x8_t*>(sec + row * 64 + c * 8);
      } else {
        const int nb = ((w0 & 63) >> 4) + (g & 1), rr = lo * 32 + ks * 16 + 8 * (g >> 1) + (j >> 2);
        const int c = (nb * 2 + ((j & 3) >> 1)) ^ ((j >> 3) << 2);
        const unsigned short* at = sec + (w0 >> 6) * 4096 + rr * 64 + c * 8 + (j & 1) * 4;
        const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)at);
        const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(at + 4 * 64));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    };
    using CA = std::integral_constant<bool, COLA>;
    using CB = std::integral_constant<bool, COLB>;
    constexpr int KS = BK / 16;
    s16x8_t a[2][TM], b[2][TN];                                 // (hi) planes, two sub-steps
    [[maybe_unused]] s16x8_t al[TM], bl[TN];                    // lo planes of the current one
    auto read = [&](s16x8_t (&fa)[TM], s16x8_t (&fb)[TN], int kt, int ks, int lo) {
      const unsigned short* sa = smem + (kt & 1) * STAGE;
      const unsigned short* sb = sa + BM * 64;
#pragma unroll
      for (int n = 0; n < TN; ++n) fb[n] = frag(CB{}, sb, wc * WN + n * 32, ks, lo);
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[i] = frag(CA{}, sa, wr * WM + i * 32, ks, lo);
    };
    auto product = [&](const s16x8_t (&fa)[TM], const s16x8_t (&fb)[TN]) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[i][n] = mma<F16>(fb[n], fa[i], acc[i][n]);
    };
    auto barrier = [&] {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };

    issue(0);
    barrier();
    if (nk > 1) issue(1);
    read(a[0], b[0], 0, 0, 0);
    for (int kt = 0; kt < nk; ++kt) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int set = ks & 1;
        bool next = false, tail = false;
        if constexpr (PL == 2) read(al, bl, kt, ks, 1);
        if (ks + 1 < KS) {
          read(a[set ^ 1], b[set ^ 1], kt, ks + 1, 0);
        } else if (kt + 1 < nk) {
          barrier();
          read(a[set ^ 1], b[set ^ 1], kt + 1, 0, 0);
          next = kt + 2 < nk;
          tail = next && is_tail(kt + 2);
        }
        __builtin_amdgcn_sched_barrier(0);
        product(a[set], b[set]);
        if constexpr (PL == 2) {
          product(a[set], bl);
          product(al, b[set]);
        }
        if (SUMA && sum) {
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            asum[i] = sum8<F16>(a[set][i], asum[i]);
            if constexpr (PL == 2) asum[i] = sum8<F16>(al[i], asum[i]);
          }
        }
        if (next) {
#pragma unroll
          for (int q = 0; q < PPW; ++q) issue_piece(kt + 2, q, tail);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// Workgroup b -> tile (ty, tx) of a tm x tn grid of tiles, false past the last.  Workgroup b runs on XCD b % 8, each with an L2 of
// its own: every XCD gets a contiguous part of a list that walks strips of 8 tile columns row by row, so the workgroups that run
// together on one share their A and B rows through it.
__device__ __forceinline__ bool tile_of(int64_t b, int64_t tm, int64_t tn, int64_t& ty, int64_t& tx) {
  const int64_t T = tm * tn;
  if (b >= T) return false;
  const int64_t xcd = b & 7, i = b >> 3, q = T >> 3, rem = T & 7;
  const int64_t t = (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + i;
  constexpr int64_t W = 8;
  const int64_t nfs = tn / W, full = nfs * tm * W;
  if (t < full) {
    const int64_t strip = t / (tm * W), r = t - strip * tm * W;
    ty = r / W;
    tx = strip * W + r % W;
  } else {
    const int64_t w = tn - nfs * W, r = t - full;
    ty = r / w;
    tx = nfs * W + r % w;
  }
  return true;
}

}  // namespace vocab
