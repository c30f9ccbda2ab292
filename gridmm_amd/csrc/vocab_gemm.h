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
//
// Bound by the way of the operands from L2 to the CU: the 256 x 256 tile asks for 32 bytes a clock at full matrix rate and gets ~21 (9.2 - 10.3
// TB/s over the chip at 1.7 GHz, matrix pipes 58 - 72 % busy, no bank conflicts); ~10 % of a tile's time is its end, which nothing overlaps.
// 8030 x 131072 x 2048 bf16: scores 3.36 ms = 1.28 PFLOP/s, dh and dW, each over two planes of dS, 1.27 - 1.28 (a large library product 1.36 - 1.41;
// boxes and hours differ by 6 %).  128 x 128 tiles
// (two workgroups a CU, 64 bytes a clock) only where the larger ones leave CUs idle.  Measured and not kept: 4 waves of 128 x 128 (278 : 246 us
// a piece), a raised wave priority around the products (the same).
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

// sum of 8 bf16 values + c
__device__ __forceinline__ float sum8(s16x8_t v, float c) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  typedef short s16x2_t __attribute__((ext_vector_type(2)));
  const bf16x2_t one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const s16x2_t x = {v[2 * e], v[2 * e + 1]};
    c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x), one, c, false);
  }
  return c;
}

// sum of 8 fp16 values times weights + c
__device__ __forceinline__ float dot8(s16x8_t v, s16x8_t w, float c) {
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  typedef short s16x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const s16x2_t x = {v[2 * e], v[2 * e + 1]}, y = {w[2 * e], w[2 * e + 1]};
    c = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, x), __builtin_bit_cast(f16x2_t, y), c, false);
  }
  return c;
}

// a pointer that is the same for the wave, in scalar registers
__device__ __forceinline__ const unsigned short* uniform(const unsigned short* p) {
  const uint64_t u = (uint64_t)p;
  return (const unsigned short*)(((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32) |
                                 (unsigned)__builtin_amdgcn_readfirstlane((int)u));
}

__device__ __forceinline__ f32x16_t mma2(float a, float b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

struct Operand {
  const unsigned short* p;
  int64_t ld;       // elements between rows of the stored matrix
  int64_t plane;    // elements between the hi and the lo plane of a row (PL = 2)
  int64_t rows;     // stored rows that may be read; what lies past them is read as the last one again
  int64_t cols;     // stored columns that may be read (a multiple of 8), likewise
};

// A piece of work for a workgroup: one output tile over one range of the contraction.
struct Item {
  int64_t bm, bn, k0;
  int nk;              // stages; 0: the tile is 0
  int extra;           // the caller's
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
  static constexpr int SCRATCH = NW * 2048;              // u16: 4 KB a wave for an epilogue's stores
  static constexpr int WEIGHTS = 2048;                   // of a wave's sums, in its SCRATCH
  static constexpr int PER_CU = BM == 256 ? 1 : 2;       // workgroups that a CU's 160 KB of LDS take
  static_assert(PIECES % NW == 0 && WM % 32 == 0 && WN % 32 == 0 && BM % 64 == 0 && BN % 64 == 0, "tile shape");
  static_assert(BM / 8 % PPW == 0 || PPW % (BM / 8) == 0, "a wave's pieces belong to one operand");

  using Acc = f32x16_t[TM][TN];

  // The workgroup's loop over its items: work(i, item) gives the i-th or false, done(item, acc, sums) takes the finished tile.  Lane l
  // ends with, for output row bm + wr WM + 32 i + (l & 31), the columns bn + wc WN + 32 j + 8 (q >> 2) + 4 (l >> 5) + (q & 3), q < 16:
  // the B operand is the first of the matrix instruction, so a lane holds runs of 4 columns of one row.
  //
  // Two-stage ring that runs on from item to item, fragments one sub-step (16 contraction steps) ahead in registers: in front of the
  // last sub-step of a stage every fragment of the stage is in registers, so ONE barrier says both that the next stage has landed and
  // that this one's buffer is free; the transfers of the stage after next -- of the next tile, near a tile's end -- start right there.
  // While done() works on a tile the next one's first fragments are in registers and its second stage is on the way.
  //
  // twice != 0 (elements): an A of two planes over a B of one, C = (A + A') B with A' that far behind A: an item's range of the
  // contraction once with A and once with A'.
  //
  // SUMA: sums also takes the sums of A over the contraction for the waves that want_sums(item) names, lane l those of the steps that
  // it holds of row 32 i + (l & 31); lanes l and l ^ 32 together hold all.  fp16: each step times its fp16
  // weight, WEIGHTS at a time in the wave's own LDS `room`, and readable that far past the contraction.  (Scalar loads wait for all of
  // the fragments' reads, and those for them: 4096 x 65536 x 2048 fp16 7.1 ms
  // against 6.1.)
  template <bool SUMA = false, class Work, class Want, class Done>
  static __device__ __forceinline__ void run(const Operand& A, const Operand& B, unsigned short* smem, Work work_once, Want want_sums, Done done,
                                             int64_t twice = 0, const unsigned short* weights = nullptr, unsigned short* room = nullptr) {
    auto work = [&](int n, Item& it) {
      const bool is = work_once(n, it);
      if (twice) it.nk *= 2;
      return is;
    };
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WAVES_N, wc = wave % WAVES_N;

    // ---- the transfers: this wave's pieces are 8 image rows x 128 bytes each, byte offsets from the operand's first tile element
    const bool isA = wave * PPW < BM / 8;
    const Operand& O = isA ? A : B;
    const bool col = isA ? COLA : COLB;
    const int64_t step = col ? BK * O.ld : BK;
    const unsigned ld = (unsigned)O.ld;
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned short*)smem + wave * PPW * 1024;
    const unsigned short* base = O.p;
    unsigned off[PPW];
    Item ahead;                          // the item whose stage `akt` is transferred next
    int ai = 0, akt = 0, issued = 0;
    bool have;
    // byte offsets of the pieces; a column operand's contraction rows past `last` of the stage are that one again
    auto aim = [&](int last) {
      const int64_t b0 = isA ? ahead.bm : ahead.bn, r0 = b0 < O.rows ? b0 : O.rows - 1;      // (a row operand's first row)
      base = O.p + (col ? ahead.k0 * O.ld : r0 * O.ld + ahead.k0);
#pragma unroll
      for (int i = 0; i < PPW; ++i) {
        const int q = wave * PPW + i - (isA ? 0 : BM / 8), slot = lane & 7;
        if (!col) {
          int row = q * 8 + (lane >> 3);
          const int c = slot ^ ((row >> 1) & 7);
          if (row > O.rows - 1 - r0) row = (int)(O.rows - 1 - r0);
          off[i] = ((unsigned)row * ld + (PL == 2 ? (c >> 2) * (unsigned)O.plane + (c & 3) * 8 : c * 8)) * 2;
        } else {
          const int panel = q >> 3, rr = (q & 7) * 8 + (lane >> 3);
          const int c = slot ^ (((rr >> 1) & 1) << 2);
          int64_t cc = b0 + panel * 64 + c * 8;
          if (cc > O.cols - 8) cc = O.cols - 8;
          const int kr = min(PL == 2 ? rr & 31 : rr, last);
          off[i] = ((unsigned)kr * ld + (PL == 2 ? (rr >> 5) * (unsigned)O.plane : 0) + (unsigned)cc) * 2;
        }
      }
    };
    auto next_item = [&] {
      do have = work(ai++, ahead); while (have && ahead.nk <= 0);
      akt = 0;
      if (have) aim(BK - 1);
    };
    // The next stage's transfers: point() says where from and to, piece(i) starts one, moved() steps on.  Past the last stage of all they
    // bring that one again, into the buffer that nobody reads any more.
    const unsigned short* from = base;
    unsigned to = 0;
    auto point = [&] {
      to = __builtin_amdgcn_readfirstlane(lds0 + (issued & 1) * (STAGE * 2));
      if (!have) return;
      const bool again = twice && akt >= ahead.nk >> 1;
      const int kt = again ? akt - (ahead.nk >> 1) : akt;
      from = base + kt * step;
      if (COLA || COLB) {
        const int64_t first = ahead.k0 + (int64_t)kt * BK, last = O.rows - 1 - first;
        if (col && (last < BK - 1 || (again && kt == 0))) {       // (the last stages of a range; what follows aims anew)
          if (last < 0) from = O.p + (O.rows - 1) * O.ld;
          aim(last < 0 ? 0 : last < BK - 1 ? (int)last : BK - 1);
        }
      }
      if (again && isA) from += twice;
      from = uniform(from);
    };
    auto piece = [&](int i) { dma16(from, off[i], to + i * 1024); };
    auto moved = [&] {
      ++issued;
      if (have && ++akt == ahead.nk) next_item();
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
    s16x8_t a[2][TM], b[2][TN];                 // (hi) planes, two sub-steps
    s16x8_t al[TM], bl[TN];                     // lo planes of the current one (PL = 2)
    // fragment f of TN + TM, in the order in which the products want them: B 0, A 0, the rest of B, the rest of A
    auto read1 = [&](s16x8_t (&fa)[TM], s16x8_t (&fb)[TN], int f, int stage, int ks, int lo) {
      const unsigned short* sa = smem + (stage & 1) * STAGE;
      const unsigned short* sb = sa + BM * 64;
      const int n = f == 0 ? 0 : f - 1, i = f == 1 ? 0 : f - TN;
      if (f == 0 || (f >= 2 && f <= TN)) fb[n] = frag(CB{}, sb, wc * WN + n * 32, ks, lo);
      else fa[i] = frag(CA{}, sa, wr * WM + i * 32, ks, lo);
    };
    Acc acc;
    auto barrier = [&] {
      // this wave's pieces of the next stage have landed and its reads of the current one are in registers
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };

    next_item();
    if (have) {
      for (int twice = 0; twice < 2; ++twice) {
        point();
#pragma unroll
        for (int i = 0; i < PPW; ++i) piece(i);
        moved();
        if (twice == 0) barrier();
      }
#pragma unroll
      for (int f = 0; f < TM + TN; ++f) read1(a[0], b[0], f, 0, 0, 0);
    }
    Item item;
    int stage = 0;
    for (int n = 0; work(n, item); ++n) {
      float sums[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        sums[i] = 0.f;
#pragma unroll
        for (int c = 0; c < TN; ++c)
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[i][c][q] = 0.f;
      }
      const bool sum = SUMA && want_sums(item);
      // One stage: its products, with the reads of the fragments ahead and the transfers of the stage after next between them, one
      // after each matrix instruction, so that none of them waits for a burst of the others.
      for (int kt = 0; kt < item.nk; ++kt, ++stage) {
        float part[TM];                      // a stage's sums first: fewer roundings of the long ones
#pragma unroll
        for (int i = 0; i < TM; ++i) part[i] = 0.f;
        const int first_k = (twice && kt >= item.nk >> 1 ? kt - (item.nk >> 1) : kt) * BK;
        if (SUMA && F16 && sum && first_k % WEIGHTS == 0) {
#pragma unroll
          for (int i = 0; i < WEIGHTS / 512; ++i)
            *reinterpret_cast<s16x8_t*>(room + i * 512 + lane * 8) = *reinterpret_cast<const s16x8_t*>(weights + item.k0 + first_k + i * 512 + lane * 8);
        }
        constexpr int NP = PL == 2 ? 3 : 1, NM = TM * TN, AT = PL == 2 ? NM - 1 : 0;      // the barrier follows product AT of the last sub-step
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int set = ks & 1;
          const bool last = ks == KS - 1;
          s16x8_t w = {0, 0, 0, 0, 0, 0, 0, 0};
          if (SUMA && F16 && sum) w = *reinterpret_cast<const s16x8_t*>(room + first_k % WEIGHTS + ks * 16 + half * 8);
#pragma unroll
          for (int m = 0; m < NP * NM; ++m) {
            const int p = m / NM, i = m % NM / TN, n2 = m % TN;
            acc[i][n2] = p == 0 ? mma<F16>(b[set][n2], a[set][i], acc[i][n2]) : p == 1 ? mma<F16>(bl[n2], a[set][i], acc[i][n2]) : mma<F16>(b[set][n2], al[i], acc[i][n2]);
            if (PL == 2 && m < TM + TN) read1(al, bl, m, stage, ks, 1);
            if (last && m == AT) {
              barrier();
              point();
            }
            constexpr int ROOM = NP * NM - 1 - AT, RPS = (TM + TN + ROOM - 1) / ROOM;      // products behind the barrier, reads at each
#pragma unroll
            for (int f = 0; f < TM + TN; ++f)
              if (m > AT && f / RPS == m - AT - 1) read1(a[set ^ 1], b[set ^ 1], f, last ? stage + 1 : stage, last ? 0 : ks + 1, 0);
            if (last && m > AT) {
              const int q0 = (m - AT - 1) * PPW / ROOM, q1 = (m - AT) * PPW / ROOM;
#pragma unroll
              for (int q = 0; q < PPW; ++q)
                if (q >= q0 && q < q1) piece(q);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if (SUMA && sum) {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
              if constexpr (F16) part[i] = dot8(a[set][i], w, part[i]);
              else part[i] = sum8(a[set][i], part[i]);
              if constexpr (PL == 2) part[i] = dot8(al[i], w, part[i]);
              if (last) sums[i] += part[i];
            }
          }
          if (last) moved();
        }
      }
      done(item, acc, sums);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // nothing is on its way into LDS that another workgroup may get
  }

  // The same loop over items in fp32, values straight from where they lie, for operands that 16-bit planes do not hold: two contraction
  // steps a matrix instruction, lane l the step k + (l >> 5).  rows(item) gives two functions of (i, k), the values of output row
  // wr WM + 32 i + (l & 31) and of output column wc WN + 32 i + (l & 31) of the tile at contraction step k, 0 where there is none.
  template <bool SUMA = false, class Work, class Want, class Rows, class Done>
  static __device__ __forceinline__ void run_exact(Work work, Want want_sums, Rows rows, Done done) {
    const int half = (threadIdx.x & 63) >> 5;
    Item item;
    for (int n = 0; work(n, item); ++n) {
      Acc acc;
      float sums[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        sums[i] = 0.f;
#pragma unroll
        for (int c = 0; c < TN; ++c)
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[i][c][q] = 0.f;
      }
      const bool sum = SUMA && want_sums(item);
      rows(item, [&](auto fa, auto fb) {
        for (int kt = 0; kt < item.nk; ++kt) {
          float part[TM];                      // a stage's sums first, as above
#pragma unroll
          for (int i = 0; i < TM; ++i) part[i] = 0.f;
#pragma unroll 1
          for (int k0 = 0; k0 < BK; k0 += 8) {
            float a[4][TM], b[4][TN];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int64_t k = item.k0 + (int64_t)kt * BK + k0 + 2 * u + half;
#pragma unroll
              for (int i = 0; i < TM; ++i) a[u][i] = fa(i, k);
#pragma unroll
              for (int c = 0; c < TN; ++c) b[u][c] = fb(c, k);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int i = 0; i < TM; ++i) {
#pragma unroll
                for (int c = 0; c < TN; ++c) acc[i][c] = mma2(b[u][c], a[u][i], acc[i][c]);
                if (sum) part[i] += a[u][i];
              }
          }
#pragma unroll
          for (int i = 0; i < TM; ++i) sums[i] += part[i];
        }
      });
      done(item, acc, sums);
      __syncthreads();                         // (what done() leaves in LDS is read before the next one writes)
    }
  }
};

// The n-th tile (ty, tx) of workgroup b of `blocks`, of a tm x tn grid of tiles, and which of `layers` grids; false past the last.
// Workgroup b runs on XCD b % 8, each with an L2 of its own: every XCD gets a contiguous part of a list that walks strips of 8 tile
// columns row by row, and its workgroups take the list's next tiles in turn, so those that run together share their A and B rows.
__device__ __forceinline__ bool tile_of(unsigned b, unsigned blocks, unsigned n, unsigned tm, unsigned tn, unsigned layers, unsigned& ty,
                                        unsigned& tx, unsigned& layer) {
  const unsigned T = tm * tn * layers, x = b & 7, q = T >> 3, rem = T & 7;
  const unsigned mine = q + (x < rem), per = (blocks - x + 7) >> 3;           // tiles of this XCD, its workgroups
  const unsigned i = (b >> 3) + n * per;
  if (i >= mine) return false;
  unsigned t = (x < rem ? x * (q + 1) : rem * (q + 1) + (x - rem) * q) + i;
  layer = t / (tm * tn);
  t -= layer * (tm * tn);
  constexpr unsigned W = 8;
  const unsigned nfs = tn / W, full = nfs * tm * W;
  if (t < full) {
    const unsigned strip = t / (tm * W), r = t - strip * tm * W;
    ty = r / W;
    tx = strip * W + r % W;
  } else {
    const unsigned w = tn - nfs * W, r = t - full;
    ty = r / w;
    tx = nfs * W + r % w;
  }
  return true;
}

}  // namespace vocab
