// Losses over a large vocabulary from hidden states, in pieces of the vocabulary, without keeping the logits
// (pretrain_src/model/pretrain_cmt.py:131-153 multiplies the masked tokens with the tied decoder of 30 522 rows and calls
// cross_entropy on the logits):
//   scores          z_rj = (h_r . W_j + b_j) / T          L_r = log sum_j exp z_rj
//   cross entropy   loss_r = L_r - z_{r, y_r}             (T = 1)
//   distillation    loss_r = T^2 sum_s p_rs (log p_rs - z_{r, id_rs} + L_r),   p_r = softmax of the teacher's top logits / T
//   both            dS_rj = g_r T (exp(z_rj - L_r) - sum_{s: id_rs = j} p_rs)    (cross entropy: one slot, p = 1)
//                   dh = dS W,   dW = dS^T h,   db_j = sum_r dS_rj
// Forward: the score tile's epilogue leaves each row's (maximum, sum of exponentials) of its columns; a second, small kernel joins
// them.  Backward: the scores are computed again piece by piece, the epilogue turns them into 16-bit dS (one piece at a time, the
// workspace bounds its width), and two more products read it.  The entries of dS at a target come from the target's score as the
// forward's sums hold it: softmax - p is rounded once there.  A row keeps its maximum and its sum of exponentials apart, as the
// logarithm of both together has roundings of the maximum's size.
//
// Rows that do not count (label == ignore_index; no filled slot) are left out on the device: the counted rows are compacted into
// the packed copy of h, the grids are sized for all rows and workgroups past the count end at once -- no host read-back.
//
// Number formats.  bf16 / fp16 operands: one plane, products exact, sums fp32; dS in two planes of the operands' type, an entry off by
// 2^-16 (bf16) or 2^-22 (fp16) of itself, so that a gradient is rounded once, to its own type.  (One plane leaves 1.4 times that error, up to
// twice where a handful of entries makes up a sum; 8030 x 131072 x 2048 13.9 ms against 21.2.)  fp32 operands: two fp16 planes each after a
// power-of-two scale from the tensor's largest finite value: 22 bits of a value, or 25 of its row's largest, as long as the rows' largest
// values lie within 2^14 of each other, which the device finds out; rows further apart run on fp32 matrix instructions.  fp16
// planes of dS take a power-of-two scale for each row, from its |g T|.
// Bound by the products (vocab_gemm.h): 8030 x 131072 x 2048 bf16 forward and backward 21.1 ms, of it 3.4 scores, 4.1 dS, 6.7 dh, 6.8 dW (two planes
// of dS each); fp32 384 x 30522 x 768 334 - 350 us, of it 255 products (1.4 rounds of 128 x 128 tiles) and 60 for W's scale and packing.
// Everything runs in the base-2 domain: y = z log2 e, exp2, and ln 2 comes back in the losses.
#include <algorithm>

#include "vocab_gemm.h"

namespace {

using vocab::f32x16_t;
using vocab::Item;
using vocab::Operand;
using vocab::Tile;
using vocab::tile_of;

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int AMAX_H = 64, AMAX_W = 512;      // workgroups of the largest-value search (fp32 operands)
constexpr int PREP_T = 1024;
constexpr int64_t PIECE_MB = 512;
enum { F32 = 0, BF16 = 1, F16 = 2 };

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
  if (dtype == F32) return reinterpret_cast<const float*>(p)[i];
  const unsigned short u = reinterpret_cast<const unsigned short*>(p)[i];
  return dtype == BF16 ? bf16_bits_to_f32(u) : (float)__builtin_bit_cast(_Float16, u);
}
__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int wide) {
  return wide ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
}
// fp32 -> 16 bits, to nearest even; NaN stays NaN
__device__ __forceinline__ unsigned short to_f16(float x) { return __builtin_bit_cast(unsigned short, (_Float16)x); }
__device__ __forceinline__ unsigned short to_bf16(float x) { return (unsigned short)(cvt_pk_bf16(x, x) & 0xffffu); }
// four of them, two at a time
template <bool F16V>
__device__ __forceinline__ u16x4_t to_16x4(float a, float b, float c, float d) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
  if constexpr (F16V) {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    const u32x2_t u = {__builtin_bit_cast(unsigned, __builtin_convertvector(((f32x2_t){a, b}), f16x2_t)),
                       __builtin_bit_cast(unsigned, __builtin_convertvector(((f32x2_t){c, d}), f16x2_t))};
    return __builtin_bit_cast(u16x4_t, u);
  } else {
    const u32x2_t u = {cvt_pk_bf16(a, b), cvt_pk_bf16(c, d)};
    return __builtin_bit_cast(u16x4_t, u);
  }
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.4028234664e38f ? a : 0.f;
}
// power of two that brings values of at most `amax` under 2^(top + 1): exponent top - floor(log2 amax)
__device__ __forceinline__ int scale_exp(float amax, int top) {
  if (!(amax > 0.f)) return 0;
  int e;
  (void)frexpf(amax, &e);              // amax = f 2^e, f in [1/2, 1)
  return top + 1 - e;
}

// what the kernels share on the device: written by the preparation kernels, read by all that follow
struct Meta {
  int count;         // rows that count
  int sh, sw;        // power-of-two exponents of the packed h and W
  int wide;          // fp32 rows too far apart for one scale: nothing is packed, the products are fp32
};
// One scale leaves 22 bits of a value, but none below 2^-40 of the tensor's largest: with the rows' largest values within 2^14 of each
// other (rows of zeros aside) every value keeps 22 bits, or 25 of its row's largest.  Rows further apart -- an outlier row, be it of a
// column that its bias masks -- take the products on fp32 matrix instructions, from the operands as they
// lie: 384 x 30522 x 768 2.0 ms against 0.33, 2048 x 32000 x 1024 11.3 against 1.5.
constexpr int SPREAD = 14;
// the operands as they lie, for those products
struct Raw {
  const void *hidden, *weight;
  int64_t ldh, ldw, j0;          // j0: the piece's first column
  int K, vocab;
  const int* rowmap;
};

// Tiles of the products over the counted rows.  256 x 256 where they fill the chip (one workgroup of 8 waves a CU), else 128 x 128 (two
// of 4 waves a CU).  The host does not know the count: where both may be right it launches both, each sized for its own range, and the
// workgroups of the one whose turn it is not end at once.  256 x 256 from 1.5 rounds of 256 CUs on; the forward at 1024 hidden, us, 256 x 256 : 128 x
// 128, at 314, 384, 512 tiles: bf16 66 : 58, 64 : 64, 72 : 79; fp32 230 : 232, 191 : 205, 206 : 239.  (One full round, 256 tiles, is better off too,
// 45 : 48 and 127 : 143, but what follows it is not, and the rule has to rise with the count to spare most calls the second launch.)
constexpr int BIG_TILES = 384;
__host__ __device__ inline bool big_tiles(int64_t count, int64_t C) { return count > 256 && (count + 255) / 256 * (C / 256) >= BIG_TILES; }
// Contraction ranges of dh, so that its few tiles fill whole rounds of the chip: the cheapest of the numbers that fit into the first
// rounds, in stages of 64 columns a workgroup (1.2 us, and as much again for the second plane of 16 bits): rounds x (its share + what a
// tile costs beside its stages) + the ranges' sums written and read once more at ~4.7 TB/s.  136 tiles at 4099 x 2048 over 32768 columns of one
// plane: 1 range 752 us, 5 ranges 545 us; over 22016 of two planes 3 ranges 749, 5 ranges 717.
constexpr int64_t PART_MOST = 64 << 20;      // values of the ranges' partial products, if there are more than one
constexpr int MOST_SPLITS = 64;
__device__ __forceinline__ int hidden_splits(int64_t count, int64_t Kp, int64_t C, bool big, bool two) {
  const int T = big ? 256 : 128, slots = big ? 256 : 512;
  const int tiles = (int)((count + T - 1) / T) * (int)((Kp + T - 1) / T);
  const float stages = (float)(C / 64) * (two ? 2.f : 1.f), join = (float)(count * Kp) * (8.f / 4.7e6f / 1.2f);
  int most = (int)min((int64_t)MOST_SPLITS, C / 512);                   // at least 8 stages a range
  if (count > 0) most = (int)min((int64_t)most, PART_MOST / (count * Kp));
  int best = 1;
  float least = INFINITY;
  for (int k = 0, r0 = (tiles + slots - 1) / slots; k < 8; ++k) {
    const int s = max(1, min(most, (r0 + k) * slots / max(tiles, 1)));
    const float cost = (float)((tiles * s + slots - 1) / slots) * (stages / (float)s + 6.f) + (float)s * join;
    if (cost < least) { least = cost; best = s; }
  }
  return best;
}

__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {        // (maximum, sum of 2^(y - maximum))
  const float M = fmaxf(a.x, b.x), ref = M == -INFINITY ? 0.f : M;        // nothing but masked columns: sum 0
  return make_float2(M, a.y * __builtin_amdgcn_exp2f(a.x - ref) + b.y * __builtin_amdgcn_exp2f(b.x - ref));
}
// 2 ln 2 times half a base-2 score or loss; what is finite stays so
__device__ __forceinline__ float natural(float half) {
  const float x = half * (2.f * LN2);
  return fabsf(half) < INFINITY ? fminf(fmaxf(x, -3.4028234664e38f), 3.4028234664e38f) : x;
}
__device__ __forceinline__ void store_as(void* p, int64_t i, int dtype, float v) {
  if (dtype == F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<unsigned short*>(p)[i] = dtype == BF16 ? to_bf16(v) : to_f16(v);
}

// ---- targets of the distillation: one wave, one row: p = softmax(t / T) over the filled slots, sum of p log p; does the row count? ----
__device__ __forceinline__ bool teacher_row(const void* ids, int wide, int64_t ld_ids, const float* t, int64_t ld_t, int64_t r, int slots,
                                            float inv_t, float* p, float& plogp) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  bool nan = false;
  for (int s = lane; s < slots; s += 64) {
    if (load_index(ids, r * ld_ids + s, wide) < 0) continue;
    const float v = t[r * ld_t + s];
    nan |= v != v;
    m = fmaxf(m, v);
  }
  m = wave_max(m);
  plogp = 0.f;
  if (m == -INFINITY && !__any(nan)) {              // nothing to learn from
    for (int s = lane; s < slots; s += 64) p[r * slots + s] = 0.f;
    return false;
  }
  float sum = 0.f;
  for (int s = lane; s < slots; s += 64)
    if (load_index(ids, r * ld_ids + s, wide) >= 0) sum += expf((t[r * ld_t + s] - m) * inv_t);
  sum = wave_sum(sum);
  const float ls = logf(sum);
  float h = 0.f;
  for (int s = lane; s < slots; s += 64) {
    float q = 0.f;
    if (load_index(ids, r * ld_ids + s, wide) >= 0) {
      const float lp = (t[r * ld_t + s] - m) * inv_t - ls;      // (t / T may be past fp32 where the difference is not)
      q = expf(lp);
      if (q > 0.f || q != q) h += q * lp;
    }
    p[r * slots + s] = q;
  }
  plogp = wave_sum(h);
  return true;
}
__global__ __launch_bounds__(256) void kd_targets_kernel(const void* __restrict__ ids, int wide, int64_t ld_ids,
                                                         const float* __restrict__ t, int64_t ld_t, int rows, int slots,
                                                         float inv_t, float* __restrict__ p, float* __restrict__ plogp,
                                                         unsigned char* __restrict__ counts) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  float h;
  const bool live = teacher_row(ids, wide, ld_ids, t, ld_t, r, slots, inv_t, p, h);
  if ((threadIdx.x & 63) == 0) { counts[r] = live; plogp[r] = h; }
}

struct PrepArgs {
  const void *hidden, *weight, *bias, *labels;
  const unsigned char* counts;       // distillation; NULL: labels
  int64_t ldh, ldw, ignore;
  int rows, vocab, K, wide, dtype, bias_dtype, vp;
  float unit;
  Meta* meta;
  int *rowmap, *rowinv;
  float *loss, *biasz;
  int *amax_h, *amax_w;
};

__device__ __forceinline__ float amax_row(const float* x, int K, int lane) {
  float a = 0.f;
  if (K % 4 == 0 && ((uintptr_t)x & 15) == 0) {
    for (int k = lane * 4; k < K; k += 256) {
      const float4 v = *reinterpret_cast<const float4*>(x + k);
      a = fmaxf(fmaxf(a, fmaxf(finite_abs(v.x), finite_abs(v.y))), fmaxf(finite_abs(v.z), finite_abs(v.w)));
    }
  } else {
    for (int k = lane; k < K; k += 64) a = fmaxf(a, finite_abs(x[k]));
  }
  return a;
}

// One launch: workgroup 0 compacts the counted rows; the next `nb` copy the bias (/ T, base 2, -inf past the vocabulary); for fp32
// operands the rest find the largest finite |h| of the counted rows and |W|, one partial value a workgroup.
__global__ __launch_bounds__(PREP_T) void prep_kernel(const PrepArgs a, int nb) {
  __shared__ int part[16];
  __shared__ int part2[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto counted = [&](int r) {
    return a.counts ? a.counts[r] != 0 : load_index(a.labels, r, a.wide) != a.ignore;
  };
  int blk = blockIdx.x;
  if (blk == 0) {
    const int64_t per = (a.rows + PREP_T - 1) / PREP_T, r0 = tid * per, r1 = min((int64_t)a.rows, r0 + per);
    int n = 0;
    for (int64_t r = r0; r < r1; ++r) n += counted((int)r);
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(incl, o, 64);
      if (lane >= o) incl += up;
    }
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    int pos = incl - n, total = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) pos += part[w];
      total += part[w];
    }
    for (int64_t r = r0; r < r1; ++r) {
      const bool c = counted((int)r);
      a.rowinv[r] = c ? pos : -1;
      if (c) a.rowmap[pos++] = (int)r;
      else a.loss[r] = 0.f;
    }
    if (tid == 0) { a.meta->count = total; a.meta->sh = a.meta->sw = a.meta->wide = 0; }
    return;
  }
  blk -= 1;
  if (blk < nb) {
    const int64_t j = (int64_t)blk * PREP_T + tid;
    if (j < a.vp)
      a.biasz[j] = j >= a.vocab ? -INFINITY : a.bias ? load_as_f32(a.bias, j, a.bias_dtype) * a.unit : 0.f;
    return;
  }
  blk -= nb;
  const bool is_h = blk < AMAX_H;
  if (!is_h) blk -= AMAX_H;
  const int blocks = is_h ? AMAX_H : AMAX_W;
  const float* x = reinterpret_cast<const float*>(is_h ? a.hidden : a.weight);
  const int64_t ld = is_h ? a.ldh : a.ldw;
  const int rows = is_h ? a.rows : a.vocab;
  int top = 1 << 14, least = -(1 << 14);          // exponents of the scales that fit the largest row and the smallest one
  for (int64_t r = blk * 16 + wave; r < rows; r += blocks * 16)
    if (!is_h || counted((int)r)) {
      const float v = wave_max(amax_row(x + r * ld, a.K, lane));
      if (v > 0.f) { const int e = scale_exp(v, 14); top = min(top, e); least = max(least, e); }
    }
  if (lane == 0) { part[wave] = top; part2[wave] = least; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 16; ++w) { top = min(top, part[w]); least = max(least, part2[w]); }
    (is_h ? a.amax_h : a.amax_w)[blk] = top + (least << 16);
  }
}
// what comes of them, by a whole wave: the exponent of the scale that brings the tensor's largest value under 2^15, and whether the rows
// lie too far apart for it
__device__ __forceinline__ int tensor_scale(const int* amax, int n, bool& wide) {
  int top = 1 << 14, least = -(1 << 14);
  for (int k = threadIdx.x & 63; k < n; k += 64) {
    const int v = amax[k], t = (short)(v & 0xffff);
    top = min(top, t);
    least = max(least, (v - t) >> 16);
  }
  top = -(int)wave_max((float)-top);
  least = (int)wave_max((float)least);
  wide |= least - top > SPREAD;
  return top == 1 << 14 ? 0 : top;                // (nothing but zeros)
}
struct Scales { int sh, sw, wide; };
__device__ __forceinline__ Scales scales(const int* amax_h, const int* amax_w) {
  bool wide = false;
  const int sh = tensor_scale(amax_h, AMAX_H, wide), sw = tensor_scale(amax_w, AMAX_W, wide);
  return wide ? Scales{0, 0, 1} : Scales{sh, sw, 0};
}

// ---- packing: rows -> 16-bit rows of Kp columns (zero past K), fp32 as two fp16 planes under a power-of-two scale ----
__device__ __forceinline__ void pack8(const float (&v)[8], bool split, int sh, unsigned short* hi, unsigned short* lo) {
  u16x8_t h, l;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = split ? ldexpf(v[e], sh) : v[e];
    const _Float16 f = (_Float16)x;
    h[e] = __builtin_bit_cast(unsigned short, f);
    l[e] = to_f16(x - (float)f);
  }
  *reinterpret_cast<u16x8_t*>(hi) = h;
  if (split) *reinterpret_cast<u16x8_t*>(lo) = l;
}
__device__ __forceinline__ void pack_row(const void* src, int64_t off, int dtype, int K, int Kp, int lane, int sh, bool zero,
                                         unsigned short* hi, unsigned short* lo) {
  if (dtype == F32) {
    const float* x = reinterpret_cast<const float*>(src) + off;
    const bool vec = ((uintptr_t)x & 15) == 0;
    for (int k = lane * 8; k < Kp; k += 512) {
      float v[8];
      if (!zero && vec && k + 8 <= K) {
        const float4 p = *reinterpret_cast<const float4*>(x + k), q = *reinterpret_cast<const float4*>(x + k + 4);
        v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; v[4] = q.x; v[5] = q.y; v[6] = q.z; v[7] = q.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = !zero && k + e < K ? x[k + e] : 0.f;
      }
      pack8(v, true, sh, hi + k, lo + k);
    }
  } else {
    const unsigned short* x = reinterpret_cast<const unsigned short*>(src) + off;
    const bool vec = ((uintptr_t)x & 15) == 0;
    for (int k = lane * 8; k < Kp; k += 512) {
      u16x8_t v;
      if (!zero && vec && k + 8 <= K) {
        v = *reinterpret_cast<const u16x8_t*>(x + k);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = !zero && k + e < K ? x[k + e] : (unsigned short)0;
      }
      *reinterpret_cast<u16x8_t*>(hi + k) = v;
    }
  }
}

// rows [j0, j0 + C) of W -> Wp (zero past the vocabulary), one row a wave
__device__ __forceinline__ void pack_w(const void* W, int64_t ldw, int dtype, int K, int Kp, int64_t j0, int i, int C, int vocab, int sw,
                                       unsigned short* Wp) {
  if (i >= C) return;
  const bool zero = j0 + i >= vocab;
  unsigned short* hi = Wp + (int64_t)i * Kp * (dtype == F32 ? 2 : 1);
  pack_row(W, zero ? 0 : (j0 + i) * ldw, dtype, K, Kp, threadIdx.x & 63, sw, zero, hi, hi + Kp);
}
__global__ __launch_bounds__(256) void pack_w_kernel(const void* __restrict__ W, int64_t ldw, int dtype, int K, int Kp, int64_t j0,
                                                     int C, int vocab, const Meta* __restrict__ meta,
                                                     unsigned short* __restrict__ Wp) {
  if (meta->wide) return;
  pack_w(W, ldw, dtype, K, Kp, j0, blockIdx.x * 4 + (threadIdx.x >> 6), C, vocab, meta->sw, Wp);
}

// The scores' operands in fp32, for Tile::run_exact: counted rows of h, rows of W of the piece
template <class T>
__device__ __forceinline__ auto exact_scores(const Raw& raw, int count) {
  return [&raw, count](const Item& it, auto f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave / T::WAVES_N, wc = wave % T::WAVES_N, K = raw.K;
    const float *h[T::TM], *w[T::TN];
#pragma unroll
    for (int i = 0; i < T::TM; ++i) {
      const int64_t r = it.bm + wr * T::WM + i * 32 + (lane & 31);
      h[i] = (const float*)raw.hidden + (int64_t)raw.rowmap[r < count ? r : count - 1] * raw.ldh;
    }
#pragma unroll
    for (int c = 0; c < T::TN; ++c) {
      const int64_t j = raw.j0 + it.bn + wc * T::WN + c * 32 + (lane & 31);
      w[c] = (const float*)raw.weight + (j < raw.vocab ? j : raw.vocab - 1) * raw.ldw;
    }
    f([&](int i, int64_t k) { return k < K ? h[i][k] : 0.f; }, [&](int c, int64_t k) { return k < K ? w[c][k] : 0.f; });
  };
}

// ---- a teacher's targets by blocks of 64 columns: the score tiles hand over the scores at them ----
// Dot products of their own read rows x slots rows of W once more (4099 x 128 x 4 KB: 305 us; 2413 x 254 x 15.6 KB: 1.4 ms).
struct TargetLists {
  const unsigned short* begin;      // [compacted row][blocks + 1]
  const unsigned* entry;            // [compacted row][slots]: slot << 6 | column in its block
  int64_t blocks;
  int slots;
  float* zt;
  const void* bias;
  int bias_dtype;
  float half_unit;
};
constexpr int LIST_BLOCKS = 4096, LIST_SLOTS = 4096;
// ---- forward: per-row (maximum, sum of exponentials) of each tile's columns; LISTS: and the scores at the targets among them ----
template <class T, bool LISTS>
__global__ __launch_bounds__(T::THREADS, 2) void score_stats_kernel(Operand A, Operand B, int nk, int tn, const Meta* __restrict__ meta,
                                                                 const float* __restrict__ biasz, float unit,
                                                                 float2* __restrict__ stats, int64_t Rp, const TargetLists L, const Raw raw) {
  __shared__ __attribute__((aligned(16))) unsigned short smem[T::LDS];
  __shared__ float2 wst[T::WAVES_N][T::BM];
  const int count = __builtin_amdgcn_readfirstlane(meta->count), tm = (count + T::BM - 1) / T::BM;
  if (big_tiles(count, (int64_t)tn * T::BN) != (T::BM == 256)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave / T::WAVES_N, wc = wave % T::WAVES_N;
  const float sc = ldexpf(unit, -(meta->sh + meta->sw));
  auto work = [&](int n, Item& it) {
    unsigned ty, tx, layer;
    if (!tile_of(blockIdx.x, gridDim.x, n, tm, tn, 1, ty, tx, layer)) return false;
    it = Item{(int64_t)ty * T::BM, (int64_t)tx * T::BN, 0, nk, 0};
    return true;
  };
  auto done = [&](const Item& it, typename T::Acc& acc, const float*) {
        float m[T::TM];
#pragma unroll
        for (int i = 0; i < T::TM; ++i) m[i] = -INFINITY;
#pragma unroll
        for (int n = 0; n < T::TN; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 b = *reinterpret_cast<const float4*>(biasz + it.bn + wc * T::WN + n * 32 + q * 8 + (lane >> 5) * 4);
#pragma unroll
            for (int i = 0; i < T::TM; ++i) {
              f32x16_t& c = acc[i][n];
              c[q * 4 + 0] = fmaf(c[q * 4 + 0], sc, b.x);
              c[q * 4 + 1] = fmaf(c[q * 4 + 1], sc, b.y);
              c[q * 4 + 2] = fmaf(c[q * 4 + 2], sc, b.z);
              c[q * 4 + 3] = fmaf(c[q * 4 + 3], sc, b.w);
              m[i] = fmaxf(m[i], fmaxf(fmaxf(c[q * 4], c[q * 4 + 1]), fmaxf(c[q * 4 + 2], c[q * 4 + 3])));
            }
          }
        if constexpr (LISTS) {
          // entries of the rows and 64 columns of this wave; either half of the wave holds 4 of every 8 columns
          const int64_t block = (raw.j0 + it.bn + wc * T::WN) >> 6;
          static_assert(T::WN == 64, "64 columns a wave");
          unsigned e0[T::TM], e1[T::TM], next[T::TM];
#pragma unroll
          for (int i = 0; i < T::TM; ++i) {
            const int64_t r = it.bm + wr * T::WM + i * 32 + (lane & 31);
            const unsigned short* at = L.begin + (r < count ? r : 0) * (L.blocks + 1) + block;
            e0[i] = at[0];
            e1[i] = r < count ? at[1] : 0;
          }
#pragma unroll
          for (int i = 0; i < T::TM; ++i) {
            const int64_t r = it.bm + wr * T::WM + i * 32 + (lane & 31);
            next[i] = e0[i] < e1[i] ? L.entry[r * L.slots + e0[i]] : 0;
          }
#pragma unroll
          for (int i = 0; i < T::TM; ++i) {
            const int64_t r = it.bm + wr * T::WM + i * 32 + (lane & 31);
            while (e0[i] < e1[i]) {
              const unsigned v = next[i], c = v & 63;
              if (++e0[i] < e1[i]) next[i] = L.entry[r * L.slots + e0[i]];
              if (((c >> 2) & 1) != (unsigned)(lane >> 5)) continue;
              const int at = (c >> 5) * 16 + ((c & 31) >> 3) * 4 + (c & 3);
              float y = acc[i][0][0];
#pragma unroll
              for (int k = 1; k < 32; ++k) y = at == k ? acc[i][k >> 4][k & 15] : y;
              // half of it: a bias of the lowest finite number, -inf in base 2, is finite so
              L.zt[r * L.slots + (v >> 6)] = y == -INFINITY && L.bias ? load_as_f32(L.bias, block * 64 + c, L.bias_dtype) * L.half_unit : 0.5f * y;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
          m[i] = fmaxf(m[i], __shfl_xor(m[i], 32, 64));
          const float ref = m[i] == -INFINITY ? 0.f : m[i];      // a tile whose columns are all masked: sum 0
          float t = 0.f;
#pragma unroll
          for (int n = 0; n < T::TN; ++n)
#pragma unroll
            for (int q = 0; q < 16; ++q) t += __builtin_amdgcn_exp2f(acc[i][n][q] - ref);
          t += __shfl_xor(t, 32, 64);
          if (lane < 32) wst[wc][wr * T::WM + i * 32 + lane] = make_float2(m[i], t);
        }
        __syncthreads();
        for (int r = threadIdx.x; r < T::BM; r += T::THREADS) {
          float2 a = wst[0][r];
#pragma unroll
          for (int w = 1; w < T::WAVES_N; ++w) a = join_stats(a, wst[w][r]);
          stats[it.bn / 128 * Rp + it.bm + r] = a;
        }
  };
  if constexpr (T::PL == 2)
    if (meta->wide) return T::run_exact(work, [](const Item&) { return false; }, exact_scores<T>(raw, count), done);
  T::run(A, B, smem, work, [](const Item&) { return false; }, done);
}

// ---- scores at the targets: one workgroup 32 targets ----
struct TargetArgs {
  const void *hidden, *weight, *index, *bias;
  int64_t ldh, ldw, ld_index;
  int K, vocab, slots, wide, kd, bias_dtype;      // slots >= 1
  float unit;
  const Meta* meta;
  const int* rowmap;
  int* label;      // [compacted row], -1 outside the vocabulary; NULL: distillation
  float* zt;       // [compacted row][slots]: HALF the score in base 2, where a bias of the lowest finite number is still finite
};
// Values k .. k + 7 of a row as they lie, zero from K on.  Vectors on the boundaries of their elements where the rows are not on 16 bytes
// (value by value 6090 x 2 targets of 3055 fp16 took 170 us longer)
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* src, int64_t off, int k, int K, float (&v)[8]) {
  typedef float any4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef float all4 __attribute__((ext_vector_type(4)));
  using V4 = typename std::conditional<VEC, all4, any4>::type;
  const float* x = (const float*)src + off + k;
  if (k + 8 <= K) {
    const V4 p = *reinterpret_cast<const V4*>(x), q = *reinterpret_cast<const V4*>(x + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = p[i]; v[4 + i] = q[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = !VEC && k + i < K ? x[i] : 0.f;      // (VEC: K % 8 == 0)
  }
}
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* src, int64_t off, int k, int K, vocab::s16x8_t& v) {
  typedef short any8 __attribute__((ext_vector_type(8), aligned(2)));
  using V8 = typename std::conditional<VEC, vocab::s16x8_t, any8>::type;
  const short* x = (const short*)src + off + k;
  if (k + 8 <= K) {
    v = *reinterpret_cast<const V8*>(x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = !VEC && k + i < K ? x[i] : (short)0;
  }
}
// ... and as the tile products take them: one plane, or two under a scale (as pack8 makes them), `apart` vectors from each other
__device__ __forceinline__ void put8(vocab::s16x8_t* at, int apart, const float (&v)[8], int e) {
  vocab::s16x8_t hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = ldexpf(v[i], e);
    const _Float16 f = (_Float16)y;
    hi[i] = __builtin_bit_cast(short, f);
    lo[i] = (short)to_f16(y - (float)f);
  }
  at[0] = hi;
  at[apart] = lo;
}
__device__ __forceinline__ void put8(vocab::s16x8_t* at, int, const vocab::s16x8_t& v, int) { at[0] = v; }
// The score at a target has to be the very number that the log-sum-exp holds for it: where a row is sure of its target their difference
// is the loss, and a second product with roundings of its own left up to 2e-5 there, of either sign.  So it is computed as the tiles
// do, by the same matrix instructions in the same order, and equals the tile's bit for bit: the diagonal of a 32 x 32 product of 32
// targets' rows of W and their rows of h.  (32 times the operations of a dot product, and the same reads, which bound it.)  The four waves
// fetch and split the operands, the first one multiplies: one wave for all of it took 62 us at 384 x 768 fp32, longer than the packing beside it.
constexpr int TARGET_LDS = 1024;      // vectors of 8 values: 16 KB
template <int DT>
__device__ __forceinline__ void target_scores(const TargetArgs& a, int64_t block, const Scales sc, vocab::s16x8_t* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 31, half = lane >> 5;
  const int64_t pair = block * 32 + n, pairs = (int64_t)a.meta->count * a.slots;
  if (block * 32 >= pairs) return;
  const int64_t i = (pair < pairs ? pair : pairs - 1) / a.slots;
  const int s = (int)((pair < pairs ? pair : pairs - 1) - i * a.slots);
  const int64_t r = a.rowmap[i], id = load_index(a.index, r * a.ld_index + s, a.wide), at = id >= 0 && id < a.vocab ? id : 0;
  const bool vec = a.K % 8 == 0 && a.ldh % 8 == 0 && a.ldw % 8 == 0 && (((uintptr_t)a.hidden | (uintptr_t)a.weight) & 15) == 0;
  f32x16_t acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  constexpr int FR = DT == F32 ? 4 : 2, U = DT == F32 ? 1 : 2;      // fragments a step (16 columns), steps a wave fetches at a time
  static_assert(4 * U * FR * 64 == TARGET_LDS, "the steps of a round in LDS");
  using Raw = typename std::conditional<DT == F32, float[8], vocab::s16x8_t>::type;
  auto product = [&](auto v) {
    Raw h[U], w[U];
    auto fetch = [&](int k0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + 16 * (wave * U + u) + 8 * half;
        load8<DT, decltype(v)::value>(a.hidden, r * a.ldh, k, a.K, h[u]);
        load8<DT, decltype(v)::value>(a.weight, at * a.ldw, k, a.K, w[u]);
      }
    };
    fetch(0);
    for (int k0 = 0; k0 < a.K; k0 += 64 * U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        vocab::s16x8_t* to = lds + (wave * U + u) * FR * 64 + lane;
        put8(to, 64, h[u], sc.sh);
        put8(to + FR / 2 * 64, 64, w[u], sc.sw);
      }
      fetch(k0 + 64 * U);                    // (past the end: zeros, nothing is read)
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int u = 0; u < 4 * U; ++u) {
          const vocab::s16x8_t* from = lds + u * FR * 64 + lane;
          acc = vocab::mma<DT != BF16>(from[FR / 2 * 64], from[0], acc);
          if constexpr (DT == F32) {
            acc = vocab::mma<true>(from[3 * 64], from[0], acc);
            acc = vocab::mma<true>(from[2 * 64], from[64], acc);
          }
        }
      }
      __syncthreads();
    }
  };
  if (DT == F32 && sc.wide) {
    if (wave) return;
    const float *h = (const float*)a.hidden + r * a.ldh, *w = (const float*)a.weight + at * a.ldw;
#pragma unroll 8
    for (int k0 = 0; k0 < a.K; k0 += 2) {
      const bool in = k0 + half < a.K;
      acc = vocab::mma2(in ? w[k0 + half] : 0.f, in ? h[k0 + half] : 0.f, acc);
    }
  } else if (vec) {
    product(std::true_type{});
  } else {
    product(std::false_type{});
  }
  if (wave) return;
  // lane l holds column l & 31 at rows 8 (q >> 2) + 4 (l >> 5) + (q & 3)
  const int q = (n >> 3) * 4 + (n & 3);
  float z = acc[0];
#pragma unroll
  for (int k = 1; k < 16; ++k) z = q == k ? acc[k] : z;
  if (pair >= pairs || half != ((n >> 2) & 1)) return;
  // an id outside the vocabulary spoils its row; an empty slot has no score
  if (a.label) a.label[i] = id >= 0 && id < a.vocab ? (int)id : -1;
  const float b = a.bias ? load_as_f32(a.bias, at, a.bias_dtype) * a.unit : 0.f, y = fmaf(z, ldexpf(a.unit, -(sc.sh + sc.sw)), b);
  // half of it: a bias of the lowest finite number, -inf in base 2, is finite so
  const float out = y == -INFINITY && a.bias ? load_as_f32(a.bias, at, a.bias_dtype) * (0.5f * a.unit) : 0.5f * y;
  a.zt[pair] = a.kd && id < 0 ? 0.f : id < 0 || id >= a.vocab ? NAN : out;
}

// TargetLists: one compacted row a workgroup (the order within a block is whatever it is: each entry is its slot's own)
__global__ __launch_bounds__(256) void target_lists_kernel(const TargetArgs t, int blocks, unsigned short* __restrict__ begin,
                                                           unsigned* __restrict__ entry) {
  __shared__ unsigned at[LIST_BLOCKS];
  __shared__ unsigned part[4];
  const int64_t i = blockIdx.x;
  if (i >= t.meta->count) return;
  const int64_t r = t.rowmap[i];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int b = tid; b < blocks; b += 256) at[b] = 0;
  __syncthreads();
  for (int s = tid; s < t.slots; s += 256) {
    const int64_t id = load_index(t.index, r * t.ld_index + s, t.wide);
    if (id >= 0 && id < t.vocab) atomicAdd(&at[id >> 6], 1u);
    else t.zt[i * t.slots + s] = id < 0 ? 0.f : NAN;      // an empty slot has no score, an id outside the vocabulary spoils its row
  }
  __syncthreads();
  // thread t owns the blocks [per t, per (t + 1))
  const int per = (blocks + 255) / 256, b0 = min(blocks, tid * per), b1 = min(blocks, b0 + per);
  unsigned n = 0;
  for (int b = b0; b < b1; ++b) n += at[b];
  unsigned incl = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned up = __shfl_up(incl, o, 64);
    if (lane >= o) incl += up;
  }
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  unsigned pos = incl - n;
  for (int w = 0; w < wave; ++w) pos += part[w];
  unsigned short* mine = begin + i * (blocks + 1);
  for (int b = b0; b < b1; ++b) {
    const unsigned c = at[b];
    at[b] = pos;
    mine[b] = (unsigned short)pos;
    pos += c;
  }
  if (tid == 255) mine[blocks] = (unsigned short)pos;
  __syncthreads();
  for (int s = tid; s < t.slots; s += 256) {
    const int64_t id = load_index(t.index, r * t.ld_index + s, t.wide);
    if (id >= 0 && id < t.vocab) entry[i * t.slots + atomicAdd(&at[id >> 6], 1u)] = (unsigned)s << 6 | (unsigned)(id & 63);
  }
}

// exponent of the scale that brings a row of fp32 or fp16 under 2^15; NO_ROW: nothing but zeros
constexpr int NO_ROW = 1 << 14;
template <int DT>
__device__ __forceinline__ int row_exp(const void* h, int64_t off, int K, int lane) {
  float m = 0.f;
  if constexpr (DT == F32) m = amax_row((const float*)h + off, K, lane);
  else
    for (int k = lane; k < K; k += 64) m = fmaxf(m, finite_abs(load_as_f32(h, off + k, DT)));
  m = wave_max(m);
  return m > 0.f ? scale_exp(m, 14) : NO_ROW;
}

// One launch behind prep_kernel: the first `blocks` workgroups pack the counted rows of h into Hp (rows past the count up to a multiple
// of 256: zero), the next `targets` compute the scores at the targets, the rest pack the first C rows of W.
template <int DT>
__global__ __launch_bounds__(256) void rows_kernel(const TargetArgs t, int blocks, int targets, int Kp,
                                                     const int* __restrict__ amax_h,
                                                     const int* __restrict__ amax_w, Meta* __restrict__ meta,
                                                     unsigned short* __restrict__ Hp, int* __restrict__ hexp, int C,
                                                     unsigned short* __restrict__ Wp) {
  __shared__ vocab::s16x8_t lds[TARGET_LDS];
  const int b = blockIdx.x - blocks, lane = threadIdx.x & 63;
  Scales sc{0, 0, 0};
  if constexpr (DT == F32) sc = scales(amax_h, amax_w);
  const int sh = sc.sh;
  if (b >= 0 && b < targets) return target_scores<DT>(t, b, sc, lds);
  if (b >= 0) {
    if (sc.wide) return;
    return pack_w(t.weight, t.ldw, DT, t.K, Kp, 0, (b - targets) * 4 + (threadIdx.x >> 6), C, t.vocab, sc.sw, Wp);
  }
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int count = meta->count;
  if (DT == F32 && i == 0 && lane == 0) { meta->sh = sh; meta->sw = sc.sw; meta->wide = sc.wide; }
  if (sc.wide) return;
  if (i >= (count + 255) / 256 * 256) return;
  const bool zero = i >= count;
  unsigned short* hi = Hp + (int64_t)i * Kp * (DT == F32 ? 2 : 1);
  const int64_t off = zero ? 0 : (int64_t)t.rowmap[i] * t.ldh;
  pack_row(t.hidden, off, DT, t.K, Kp, lane, sh, zero, hi, hi + Kp);
  if constexpr (DT != BF16)
    if (!zero && hexp) {
      const int e = row_exp<DT>(t.hidden, off, t.K, lane);
      if (lane == 0) hexp[i] = e;
    }
}

// ---- joins the tiles' statistics and writes the losses: 16 rows a workgroup, 16 threads a row ----
__global__ __launch_bounds__(256) void loss_kernel(const float2* __restrict__ stats, int64_t Vp, int64_t C, int64_t Rp, const Meta* __restrict__ meta,
                                                   const int* __restrict__ rowmap, const float* __restrict__ zt, int slots,
                                                   const float* __restrict__ p, const float* __restrict__ plogp, float temperature,
                                                   float2* __restrict__ stat, float* __restrict__ loss) {
  __shared__ float2 part[16][17];
  __shared__ float2 acc[16][17];
  const int rr = threadIdx.x & 15, lanep = threadIdx.x >> 4;
  const int count = meta->count;
  const int64_t T = big_tiles(count, C) ? 256 : 128;
  // statistics of the tile at column j lie at j / 128 (a last piece may have taken the other tile)
  const int64_t last = Vp % C ? (big_tiles(count, Vp % C) ? 256 : 128) : T, whole = Vp / C * C;
  const int64_t i = (int64_t)blockIdx.x * 16 + rr;
  if ((int64_t)blockIdx.x * 16 >= count) return;
  float2 a = make_float2(-INFINITY, 0.f);
  if (i < count) {
    auto join = [&](int64_t j, int64_t end, int64_t step) {      // 8 loads in flight (one after the other: 10 us at 239 tiles)
      for (; j < end; j += 8 * step) {
        float2 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = stats[(j + u * step < end ? j + u * step : j) / 128 * Rp + i];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (j + u * step < end) a = join_stats(a, v[u]);
      }
    };
    join(lanep * T, whole, 16 * T);
    join(whole + lanep * last, Vp, 16 * last);
  }
  part[lanep][rr] = a;
  __syncthreads();
  a = part[0][rr];
  for (int w = 1; w < 16; ++w) a = join_stats(a, part[w][rr]);
  // The log-sum-exp stays in its two parts, maximum and logarithm of the sum: as one number it has the maximum's roundings, 2e-6 at 46
  const float ls = a.x == -INFINITY ? NAN : 0.5f * __builtin_amdgcn_logf(a.y);        // (halves, base 2; no column left: no number)
  float s = 0.f, mass = 0.f;
  bool bad = !(a.x == a.x && ls == ls);
  if (i < count) {
    if (p) {
      const int64_t r = rowmap[i];
#pragma unroll 4
      for (int k = lanep; k < slots; k += 16) {
        const float q = p[r * slots + k], z = zt[i * slots + k];
        bad |= z != z;
        if (!(q == 0.f)) { s += q * (0.5f * a.x - z); mass += q; }
      }
    }
  }
  acc[lanep][rr] = make_float2(bad ? NAN : s, mass);
  __syncthreads();
  if (lanep != 0 || i >= count) return;
  const int64_t r = rowmap[i];
  float out;
  if (p) {
    s = mass = 0.f;
    for (int w = 0; w < 16; ++w) { s += acc[w][rr].x; mass += acc[w][rr].y; }
    out = temperature * temperature * (plogp[r] + natural(fmaf(mass, ls, s)));
  } else {
    out = natural((0.5f * a.x - zt[i]) + ls);
    s = zt[i];
  }
  loss[r] = out;
  stat[i] = make_float2(a.x, s != s ? NAN : a.y);           // a bad target: its row's gradient is NaN too
}

// ---- backward ----
// dS in fp16 planes takes a scale for each row, from its |g T|: 2^13 at most, so that a row's entries keep 22 bits, or 2^-38 of its
// own |g T|, whatever the others are.  dh takes the scales out again row by row; dW = dS^T h sums over the rows, so h is laid out once
// more with the scales' inverses in it, and db's sums carry them as weights (2^15 to 2^-24).  Rows whose |g T| |h| are more than 2^20 apart do not
// fit into one layout of h (up to there a value is off by 2^-19 of its row's largest at most), |g T| more than 2^39 apart not into the weights: dS is fp32 then and dh and dW are products on fp32 matrix
// instructions.  bf16 has fp32's range and needs none of it.
constexpr int GRAD_SPREAD = 20, WEIGHT_SPREAD = 39;
struct Back {
  int wide;          // dS is fp32
  int c, least;      // dW's unit is 2^-c, db's 2^-least (fp32 dS: 1)
  int ranges;        // of dh
};
struct GradArgs {
  const float* g;              // upstream gradients of the rows as they came
  int64_t gs;
  float temperature;
  const int* rowmap;
  const int* label;            // of the compacted rows; NULL: distillation, whose targets a kernel of their own writes
  const float* zt;
  const float2* stat;          // (maximum, sum of 2^(y - maximum)): a softmax entry is 2^(y - maximum) / sum
  const int* rowexp;           // of the compacted rows: dS is 2^this times as large; NULL: 1
  const Back* back;            // NULL: bf16
  __device__ float scaled(int i) const {
    const float v = g[rowmap[i] * gs] * temperature;
    return rowexp ? ldexpf(v, rowexp[i]) : v;
  }
};
// The rows' scales, what they come to, and h with their inverses: H2 and weights.  Every workgroup goes through all rows' exponents for
// itself, one wave then lays a row out.
__global__ __launch_bounds__(256) void grad_scales_kernel(const GradArgs a, const Meta* __restrict__ meta, const int* __restrict__ hexp, int planes, int Kp,
                                                          const unsigned short* __restrict__ Hp, unsigned short* __restrict__ H2,
                                                          unsigned short* __restrict__ weights, int* __restrict__ rowexp, Back* __restrict__ back) {
  __shared__ int part[4][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, count = meta->count;
  auto exponent = [&](int i) {       // NO_ROW: a gradient of 0, or none that is a number
    const float v = finite_abs(a.g[a.rowmap[i] * a.gs] * a.temperature);
    return v > 0.f ? scale_exp(v, 13) : NO_ROW;
  };
  int e0 = NO_ROW, e1 = -NO_ROW, least = NO_ROW, most = -NO_ROW;
  if (!meta->wide) {
#pragma unroll 4
    for (int i = tid; i < count; i += 256) {
      const int x = exponent(i), h = hexp[i];
      if (x == NO_ROW) continue;
      least = min(least, x);
      most = max(most, x);
      if (h != NO_ROW) { e0 = min(e0, x + h); e1 = max(e1, x + h); }
    }
  }
  e0 = -(int)wave_max((float)-e0);
  e1 = (int)wave_max((float)e1);
  least = -(int)wave_max((float)-least);
  most = (int)wave_max((float)most);
  if (lane == 0) { part[wave][0] = e0; part[wave][1] = e1; part[wave][2] = least; part[wave][3] = most; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    e0 = min(e0, part[w][0]); e1 = max(e1, part[w][1]);
    least = min(least, part[w][2]); most = max(most, part[w][3]);
  }
  const bool wide = meta->wide || e1 - e0 > GRAD_SPREAD || most - least > WEIGHT_SPREAD;
  const int c = wide || e0 == NO_ROW ? 0 : e0;
  if (wide || least == NO_ROW) least = 0;
  if (blockIdx.x == 0 && tid == 0) { back->wide = wide; back->c = c; back->least = wide ? 0 : least + 15; }
  for (int i = blockIdx.x * 4 + wave; i < (count + 255) / 256 * 256; i += gridDim.x * 4) {
    const int x = i < count && !wide ? exponent(i) : NO_ROW;
    if (lane == 0) {
      rowexp[i] = x == NO_ROW ? 0 : x;
      weights[i] = x == NO_ROW ? (unsigned short)0 : to_f16(ldexpf(1.f, 15 + least - x));
    }
    if (wide) continue;
    // (zeros past the count and for a row whose gradient is 0 or no number, which its dS has already)
    const int64_t at = (int64_t)i * Kp * planes;
    for (int k = lane * 8; k < Kp * planes; k += 512) {
      u16x8_t v = *reinterpret_cast<const u16x8_t*>(Hp + at + k);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = x == NO_ROW ? (unsigned short)0 : to_f16(ldexpf((float)__builtin_bit_cast(_Float16, (unsigned short)v[e]), c - x - meta->sh));
      *reinterpret_cast<u16x8_t*>(H2 + at + k) = v;
    }
  }
}

// A wave's 32 x 64 values of an epilogue, of 16 or 32 bits, through its own LDS: lane l puts the runs of 4 columns it holds of row
// l & 31, and takes 16 bytes at a time of rows that lie whole in 8 (16 bits) or 16 (32 bits, 32 columns a pass) lanes: 128 contiguous
// bytes a row instead of 16 or 32.
template <class Patch, class Put>
__device__ __forceinline__ void rows_of_16(unsigned short* scratch, const u16x4_t (&v)[8], Patch patch, Put put) {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  // run n q (8 columns 8 (4 n + q) ..) half h: 8 bytes at column 32 n + 8 q + 4 h, 16-byte chunks swizzled by the row
#pragma unroll
  for (int i = 0; i < 8; ++i) *reinterpret_cast<u16x4_t*>(scratch + r * 64 + ((i ^ (r & 7)) * 8) + h * 4) = v[i];
  patch([&](int c) -> unsigned short& { return scratch[r * 64 + (((c >> 3) ^ (r & 7)) * 8) + (c & 7)]; });      // column c of row r
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int row = p * 8 + (lane >> 3), c = lane & 7;
    put(row, c * 8, *reinterpret_cast<const u16x8_t*>(scratch + row * 64 + ((c ^ (row & 7)) * 8)));
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
template <class Put>
__device__ __forceinline__ void rows_of_32(unsigned short* scratch, const float4 (&v)[4], Put put) {       // 32 x 32
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  float* s = reinterpret_cast<float*>(scratch);
#pragma unroll
  for (int q = 0; q < 4; ++q) *reinterpret_cast<float4*>(s + r * 32 + (((2 * q + h) ^ (r & 7)) * 4)) = v[q];
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int row = p * 8 + (lane >> 3), c = lane & 7;
    put(row, c * 4, *reinterpret_cast<const float4*>(s + row * 32 + ((c ^ (row & 7)) * 4)));
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// dS of the columns [j0, j0 + C): dS[r][j] = g_r T q_rj in two planes; at the row's label, from its fp32 score, g_r (q - 1)
template <class T>
__global__ __launch_bounds__(T::THREADS, 2) void score_grad_kernel(Operand A, Operand B, int nk, int tn, const Meta* __restrict__ meta,
                                                                const float* __restrict__ biasz, float unit, const GradArgs G, const Raw raw,
                                                                unsigned short* __restrict__ dS, int64_t plane) {
  __shared__ __attribute__((aligned(16))) unsigned short smem[T::LDS + T::SCRATCH];
  const int count = __builtin_amdgcn_readfirstlane(meta->count), tm = (count + T::BM - 1) / T::BM;
  if (big_tiles(count, (int64_t)tn * T::BN) != (T::BM == 256)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave / T::WAVES_N, wc = wave % T::WAVES_N;
  const float sc = ldexpf(unit, -(meta->sh + meta->sw));
  unsigned short* scratch = smem + T::LDS + wave * 2048;
  static_assert(T::TN == 2, "64 columns a wave");
  const int64_t ldS = 2 * plane;
  auto work = [&](int n, Item& it) {
    unsigned ty, tx, layer;
    if (!tile_of(blockIdx.x, gridDim.x, n, tm, tn, 1, ty, tx, layer)) return false;
    it = Item{(int64_t)ty * T::BM, (int64_t)tx * T::BN, 0, nk, 0};
    return true;
  };
  // in planes of 16 bits, or in fp32 (which takes the same room)
  auto done = [&](auto in_fp32) {
    return [&](const Item& it, typename T::Acc& acc, const float*) {
        const int64_t r0 = it.bm + wr * T::WM, c0 = it.bn + wc * T::WN;
        const float* bz = biasz + c0 + (lane >> 5) * 4;
        // what the rows need, its loads in flight together
        float Ms[T::TM], inv[T::TM], gs[T::TM];
        int ys[T::TM];
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
          const int r = (int)r0 + i * 32 + (lane & 31), rl = min(r, count - 1);
          const float2 st = G.stat[rl];
          const float g = G.scaled(rl);
          ys[i] = G.label && r < count ? G.label[rl] - (int)(raw.j0 + c0) : -1;
          Ms[i] = r < count ? st.x : INFINITY;          // (a row past the count: 0 times exp2(-inf))
          inv[i] = r < count ? 1.f / st.y : 1.f;
          gs[i] = r < count ? g : 0.f;
        }
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          const float M = Ms[i], gr = gs[i], gq = gr * inv[i];
          const int y = ys[i];
          const bool hit = y >= 0 && y < 64;
          float target = 0.f;
          if (hit) target = gr * fmaf(__builtin_amdgcn_exp2f(2.f * G.zt[r0 + i * 32 + (lane & 31)] - M), inv[i], -1.f);
          auto rounded = [](float x) {
            const unsigned short u = T::F16 ? to_f16(x) : to_bf16(x);
            return T::F16 ? (float)__builtin_bit_cast(_Float16, u) : bf16_bits_to_f32(u);
          };
          auto values = [&](int c, float (&v)[4]) {
            const float4 b = *reinterpret_cast<const float4*>(bz + c * 8);
            const float bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = gq * __builtin_amdgcn_exp2f(fmaf(acc[i][c >> 2][(c & 3) * 4 + e], sc, bb[e]) - M);
          };
          auto put = [&](const u16x4_t (&x)[8], float at_target, unsigned short* at) {
            rows_of_16(scratch, x, [&](auto column) { if (hit && lane < 32) column(y) = T::F16 ? to_f16(at_target) : to_bf16(at_target); },
                       [&](int row, int cc, u16x8_t v) { *reinterpret_cast<u16x8_t*>(at + row * ldS + cc) = v; });
          };
          if constexpr (decltype(in_fp32)::value) {
            float* at = reinterpret_cast<float*>(dS) + (r0 + i * 32) * plane + c0;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              float4 v[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                float x[4];
                values(4 * n + c, x);
                // (half of the wave holds 4 of every 8 columns; the label's among them)
                const int e = y - 32 * n - 8 * c - 4 * (lane >> 5);
                v[c] = make_float4(e == 0 ? target : x[0], e == 1 ? target : x[1], e == 2 ? target : x[2], e == 3 ? target : x[3]);
              }
              rows_of_32(scratch, v, [&](int row, int cc, float4 f) { *reinterpret_cast<float4*>(at + row * plane + n * 32 + cc) = f; });
            }
            continue;
          }
          unsigned short* at = dS + (r0 + i * 32) * ldS + c0;
          u16x4_t hi[8], lo[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float v[4];
            values(c, v);
            hi[c] = to_16x4<T::F16>(v[0], v[1], v[2], v[3]);
            lo[c] = to_16x4<T::F16>(v[0] - rounded(v[0]), v[1] - rounded(v[1]), v[2] - rounded(v[2]), v[3] - rounded(v[3]));
          }
          put(hi, target, at);
          put(lo, target - rounded(target), at + plane);
        }
    };
  };
  auto none = [](const Item&) { return false; };
  if constexpr (T::PL == 2)
    if (meta->wide) return T::run_exact(work, none, exact_scores<T>(raw, count), done(std::true_type{}));
  if constexpr (T::F16)
    if (G.back->wide) return T::run(A, B, smem, work, none, done(std::true_type{}));
  T::run(A, B, smem, work, none, done(std::false_type{}));
}

// the entries of dS at a teacher's targets in [j0, j0 + C): g_r T (q - sum of p over the slots of the same id)
struct FixArgs {
  const void* index;
  int64_t ld_index, j0, ldS, plane;
  int wide, slots, C, vocab, dtype;
  const Meta* meta;
  GradArgs G;
  const float* p;
  unsigned short* dS;
};
__device__ __forceinline__ void target_entry(const FixArgs& a, int64_t i, int s, int64_t id, float p) {
  const float2 st = a.G.stat[i];
  const float v = a.G.scaled((int)i) * fmaf(__builtin_amdgcn_exp2f(2.f * a.G.zt[i * a.slots + s] - st.x), 1.f / st.y, -p);
  if (a.G.back && a.G.back->wide) {
    reinterpret_cast<float*>(a.dS)[i * a.plane + (id - a.j0)] = v;
    return;
  }
  unsigned short* at = a.dS + i * a.ldS + (id - a.j0);
  at[0] = a.dtype == BF16 ? to_bf16(v) : to_f16(v);
  at[a.plane] = a.dtype == BF16 ? to_bf16(v - bf16_bits_to_f32(at[0])) : to_f16(v - (float)__builtin_bit_cast(_Float16, at[0]));
}
// one row a workgroup, 256 of its slots in LDS at a time; several slots may name one id: each of them writes the same value
__global__ __launch_bounds__(256) void target_grad_kernel(const FixArgs a) {
  __shared__ int sid[256];
  __shared__ float sp[256];
  const int64_t i = blockIdx.x;
  if (i >= a.meta->count) return;
  const int64_t r = a.G.rowmap[i];
  for (int s0 = 0; s0 < a.slots; s0 += 256) {
    const int s = s0 + threadIdx.x;
    const int64_t id = s < a.slots ? load_index(a.index, r * a.ld_index + s, a.wide) : -1;
    const bool mine = id >= a.j0 && id < a.j0 + a.C && id < a.vocab && id >= 0;
    float p = 0.f;
    for (int t0 = 0; t0 < a.slots; t0 += 256) {
      __syncthreads();
      const int t = t0 + threadIdx.x;
      if (t < a.slots) {
        const int64_t o = load_index(a.index, r * a.ld_index + t, a.wide);
        sid[threadIdx.x] = o < 0 || o >= a.vocab ? -1 : (int)o;
        sp[threadIdx.x] = a.p[r * a.slots + t];
      }
      __syncthreads();
      if (mine)
        for (int k = 0; k < min(256, a.slots - t0); ++k) p += sid[k] == (int)id ? sp[k] : 0.f;
    }
    if (mine) target_entry(a, i, s, id, p);
  }
}

// dh of this piece: partial products over the contraction ranges blockIdx.y, added to those of the pieces before.  `C`: the columns of
// a whole piece, which fix the tile and the number of ranges for all pieces.
template <class T>
__global__ __launch_bounds__(T::THREADS, 2) void hidden_grad_kernel(Operand A, Operand B, int steps, int tn, int64_t C,
                                                                 const Meta* __restrict__ meta, float* __restrict__ part, int64_t Kp,
                                                                 int first, Back* __restrict__ back, const Raw raw) {
  __shared__ __attribute__((aligned(16))) unsigned short smem[T::LDS + T::SCRATCH];
  const int count = __builtin_amdgcn_readfirstlane(meta->count), tm = (count + T::BM - 1) / T::BM;
  const bool big = big_tiles(count, C);
  if (big != (T::BM == 256)) return;
  constexpr bool TWO = T::PL == 1;       // dS's two planes one after the other
  const int splits = hidden_splits(count, Kp, C, big, TWO), per = (steps + splits - 1) / splits;
  if (blockIdx.x == 0 && threadIdx.x == 0) back->ranges = splits;
  const int wave = threadIdx.x >> 6, wr = wave / T::WAVES_N, wc = wave % T::WAVES_N;
  unsigned short* scratch = smem + T::LDS + wave * 2048;
  auto work = [&](int n, Item& it) {
    unsigned ty, tx, split;
    if (!tile_of(blockIdx.x, gridDim.x, n, tm, tn, splits, ty, tx, split)) return false;
    it = Item{(int64_t)ty * T::BM, (int64_t)tx * T::BN, (int64_t)split * per * T::BK, min(per, steps - (int)split * per), (int)split};
    return true;
  };
  auto done = [&](const Item& it, typename T::Acc& acc, const float*) {
    float* out = part + (int64_t)it.extra * count * Kp;
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int n = 0; n < T::TN; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        const int64_t r0 = it.bm + wr * T::WM + i * 32, c0 = it.bn + wc * T::WN + n * 32;
        float4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = make_float4(acc[i][n][q * 4], acc[i][n][q * 4 + 1], acc[i][n][q * 4 + 2], acc[i][n][q * 4 + 3]);
        rows_of_32(scratch, v, [&](int row, int cc, float4 x) {
          if (r0 + row >= count || c0 + cc >= Kp) return;
          float4* at = reinterpret_cast<float4*>(out + (r0 + row) * Kp + c0 + cc);
          if (!first) { const float4 o = *at; x.x += o.x; x.y += o.y; x.z += o.z; x.w += o.w; }
          *at = x;
        });
      }
  };
  if constexpr (T::F16)
    if (back->wide) {
      // dS in fp32, W where it lies
      auto rows = [&](const Item& it, auto f) {
        const int lane = threadIdx.x & 63;
        const float* s[T::TM];
        int64_t w[T::TN];
        bool in[T::TN];
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
          const int64_t r = it.bm + wr * T::WM + i * 32 + (lane & 31);
          s[i] = reinterpret_cast<const float*>(A.p) + (r < count ? r : count - 1) * A.cols;
        }
#pragma unroll
        for (int c = 0; c < T::TN; ++c) {
          const int64_t k = it.bn + wc * T::WN + c * 32 + (lane & 31);
          in[c] = k < raw.K;
          w[c] = in[c] ? k : 0;
        }
        f([&](int i, int64_t j) { return j < A.cols && raw.j0 + j < raw.vocab ? s[i][j] : 0.f; },
          [&](int c, int64_t j) { return in[c] && raw.j0 + j < raw.vocab ? load_as_f32(raw.weight, w[c] + (raw.j0 + j) * raw.ldw, T::PL == 2 ? F32 : F16) : 0.f; });
      };
      return T::run_exact(work, [](const Item&) { return false; }, rows, done);
    }
  T::run(A, B, smem, work, [](const Item&) { return false; }, done, TWO ? A.cols : 0);
}

// dh = the ranges' partial products in order, unscaled, to the rows they came from; zero for rows that do not count.  A workgroup
// takes 64 runs of 4 columns of one row, 4 threads a run, each every fourth range.
__global__ __launch_bounds__(256) void hidden_out_kernel(const float* __restrict__ part, int64_t Kp, int K, int rows,
                                                         const int* __restrict__ rowinv, const Meta* __restrict__ meta,
                                                         const int* __restrict__ rowexp, const Back* __restrict__ back, int dtype,
                                                         void* __restrict__ out) {
  __shared__ float4 sums[3][64];
  const int t = threadIdx.x & 63, sp = threadIdx.x >> 6;
  const int64_t r = blockIdx.x;
  const int k = blockIdx.y * 256 + t * 4;
  const int count = __builtin_amdgcn_readfirstlane(meta->count), pos = rowinv[r];
  const int e = !rowexp || pos < 0 || back->wide ? 0 : -(rowexp[pos] + meta->sw);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (pos >= 0 && k < Kp) {
    const int splits = back->ranges;
    const float* at = part + (int64_t)pos * Kp + k;
#pragma unroll 4
    for (int s = sp; s < splits; s += 4) {
      const float4 a = *reinterpret_cast<const float4*>(at + (int64_t)s * count * Kp);
      v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
    }
  }
  if (sp) sums[sp - 1][t] = v;
  __syncthreads();
  if (sp || k >= K) return;
#pragma unroll
  for (int s = 0; s < 3; ++s) { const float4 a = sums[s][t]; v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w; }
  const float f[4] = {ldexpf(v.x, e), ldexpf(v.y, e), ldexpf(v.z, e), ldexpf(v.w, e)};
  for (int x = 0; x < 4; ++x)
    if (k + x < K) store_as(out, r * K + k + x, dtype, f[x]);
}

// dW of this piece: rows [j0, j0 + C) complete (the contraction is all counted rows), written once in the weight's type; the first
// tile column also sums dS over the rows: db
template <class T>
__global__ __launch_bounds__(T::THREADS, 2) void weight_grad_kernel(Operand A, Operand B, int tm, int tn, const Meta* __restrict__ meta,
                                                                 const Back* __restrict__ back, const unsigned short* __restrict__ weights, int dtype, int64_t j0, int vocab, int K,
                                                                 void* __restrict__ dW, int bias_dtype, void* __restrict__ db, const Raw raw) {
  __shared__ __attribute__((aligned(16))) unsigned short smem[T::LDS + T::SCRATCH];
  const int count = __builtin_amdgcn_readfirstlane(meta->count);
  constexpr bool TWO = T::PL == 1;
  const int nk = (count + T::BK - 1) / T::BK;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave / T::WAVES_N, wc = wave % T::WAVES_N;
  const int eb = T::F16 ? -back->least : 0, e = T::F16 ? -back->c : 0;       // exponents of the units of db and dW
  unsigned short* scratch = smem + T::LDS + wave * 2048;
  static_assert(T::TN == 2, "64 columns a wave");
  auto work = [&](int n, Item& it) {
    unsigned ty, tx, layer;
    if (!tile_of(blockIdx.x, gridDim.x, n, tm, tn, 1, ty, tx, layer)) return false;
    it = Item{(int64_t)ty * T::BM, (int64_t)tx * T::BN, 0, nk, 0};
    return true;
  };
  auto want = [&](const Item& it) { return db && it.bn == 0 && wc == 0; };
  auto done = [&](const Item& it, typename T::Acc& acc, const float* sums) {
    const int64_t r0 = j0 + it.bm + wr * T::WM, c0 = it.bn + wc * T::WN;
    if (db && it.bn == 0 && wc == 0) {
#pragma unroll
      for (int i = 0; i < T::TM; ++i) {
        const float s = sums[i] + __shfl_xor(sums[i], 32, 64);
        const int64_t j = r0 + i * 32 + (lane & 31);
        if (lane < 32 && j < vocab) store_as(db, j, bias_dtype, ldexpf(s, eb));
      }
    }
    if (!dW) return;
#pragma unroll
    for (int i = 0; i < T::TM; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (dtype == F32) {
        float* out = reinterpret_cast<float*>(dW);
#pragma unroll
        for (int n = 0; n < T::TN; ++n) {
          float4 v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            v[q] = make_float4(ldexpf(acc[i][n][q * 4], e), ldexpf(acc[i][n][q * 4 + 1], e), ldexpf(acc[i][n][q * 4 + 2], e), ldexpf(acc[i][n][q * 4 + 3], e));
          rows_of_32(scratch, v, [&](int row, int cc, float4 x) {
            const int64_t r = r0 + i * 32 + row, c = c0 + n * 32 + cc;
            if (r >= vocab || c >= K) return;
            if (K % 4 == 0) {
              *reinterpret_cast<float4*>(out + r * K + c) = x;
            } else {
              const float f[4] = {x.x, x.y, x.z, x.w};
              for (int e = 0; e < 4; ++e)
                if (c + e < K) out[r * K + c + e] = f[e];
            }
          });
        }
      } else {
        unsigned short* out = reinterpret_cast<unsigned short*>(dW);
        u16x4_t v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const f32x16_t& x = acc[i][c >> 2];
          const int q = (c & 3) * 4;
          v[c] = to_16x4<T::F16>(ldexpf(x[q], e), ldexpf(x[q + 1], e), ldexpf(x[q + 2], e), ldexpf(x[q + 3], e));
        }
        rows_of_16(scratch, v, [](auto) {}, [&](int row, int cc, u16x8_t x) {
          const int64_t r = r0 + i * 32 + row, c = c0 + cc;
          if (r >= vocab || c >= K) return;
          if (K % 8 == 0) {
            *reinterpret_cast<u16x8_t*>(out + r * K + c) = x;
          } else {
            for (int e = 0; e < 8; ++e)
              if (c + e < K) out[r * K + c + e] = x[e];
          }
        });
      }
    }
  };
  if constexpr (T::F16)
    if (back->wide) {
      auto rows = [&](const Item& it, auto f) {
        const float* s[T::TM];
        int64_t h[T::TN];
        bool in[T::TN];
#pragma unroll
        for (int i = 0; i < T::TM; ++i) s[i] = reinterpret_cast<const float*>(A.p) + it.bm + wr * T::WM + i * 32 + (lane & 31);
#pragma unroll
        for (int c = 0; c < T::TN; ++c) {
          const int64_t k = it.bn + wc * T::WN + c * 32 + (lane & 31);
          in[c] = k < raw.K;
          h[c] = in[c] ? k : 0;
        }
        f([&](int i, int64_t r) { return r < count ? s[i][r * A.cols] : 0.f; },
          [&](int c, int64_t r) { return in[c] && r < count ? load_as_f32(raw.hidden, h[c] + (int64_t)raw.rowmap[r] * raw.ldh, T::PL == 2 ? F32 : F16) : 0.f; });
      };
      return T::template run_exact<true>(work, want, rows, done);
    }
  T::template run<true>(A, B, smem, work, want, done, TWO ? A.cols : 0, weights, scratch);
}

__global__ void zero_u16_kernel(unsigned short* __restrict__ p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = 0;
}

}  // namespace

#include "vocab_few.h"

namespace {

// ---------------------------------------------------------------------------------------------------------------------
// host side: what lies where, which tile, how wide a piece
// ---------------------------------------------------------------------------------------------------------------------
inline size_t up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// Which kernels.  Wall time of a call alone, us, few rows : tiles; a small call is the host's time, ~140 : 175 forward and backward, ~35 : 40
// - 50 the forward alone.
//   up to 32 rows (the forward alone of 16 bits: 16): forward and backward bf16 131072 x 2048 at 5, 16, 32, 48 rows 506 : 783, 507 : 777, 667 : 782,
//   1172 : 780; 30522 x 768 at 32, 48 rows 158 : 177, 193 : 176; fp32 131072 x 2048 at 16, 32 rows 810 : 2286, 989 : 2294; the forward alone
//   bf16 131072 x 2048 at 17, 32 rows 177 : 184, 221 : 179
//   small products: a workgroup of the weight gradient goes through groups x ceil(hidden / 256) steps one after another (bf16 8000 x 512 at 8, 16
//   of them 163 : 172, 233 : 173; 2216 x 512 at 16, 32 178 : 172, 284 : 174), and throughput counts from 3e8 scores x hidden on (fp32 30522 x
//   768 at 32, 64, 96 rows 162 : 223, 222 : 229, 305 : 234), where a score costs as much as 100 columns beside its product (16 bits);
//   the forward alone from 1e9 on (fp32 8000 x 2048 at 64, 128 rows 80 : 129, 114 : 130; bf16 8000 x 452 at 256, 512 rows 48 : 57, 66 : 58;
//   8000 x 16 at 512, 1024, 2048 rows 37 : 40, 48 : 41, 67 : 45)
//   a teacher's slots: every workgroup looks through all rows' ids; fp32 256 rows x 2000 x 64 at 64, 256, 1024 slots (3e7, 1e8, 5e8 comparisons)
//   147 : 191, 167 : 190, 691 : 463, the forward alone 44 : 53, 65 : 62, 318 : 103.  With few rows it is the tiles that suffer more (each row's slots
//   against each other, one workgroup): 16 rows x 131072 x 768 bf16 at 2048, 8192 slots (4e9, 2e10) 422 : 1507, 1018 : 18184
bool few_vectors(const gridmm_vocab_loss_t* d) {      // rows of h and W are whole 16-byte vectors on their boundaries
  const int A = d->dtype == F32 ? 4 : 8;
  return d->hidden_size % A == 0 && d->ld_hidden % A == 0 && d->ld_weight % A == 0 &&
         (((uintptr_t)d->hidden | (uintptr_t)d->weight) & 15) == 0;
}
bool few_rows(const gridmm_vocab_loss_t* d) {
  const double rv = (double)d->rows * d->vocab, K = d->hidden_size, targets = rv * d->slots;
  const bool fp32 = d->dtype == F32;
  if (targets > 2e10) return false;
  if (d->rows <= (fp32 || !d->forward_only ? 32 : 16)) return true;
  if (targets > 1e8) return false;
  if (d->forward_only) return rv * (K + 100) <= 1.1e9;
  const int steps = (d->rows + 31) / 32 * ((d->hidden_size + 255) / 256);
  return steps <= 16 && (fp32 ? rv * K <= 2.8e8 : rv * (K + 100) <= 7e8);
}

// Scores at a teacher's targets out of the score tiles where that is the cheaper: dot products read rows x slots rows of W at ~7 TB/s,
// the lists cost ~12 us and each tile's end ~4 us (0.28 us a million scores).  dot products : lists, us of the whole call: 4099 x 65537 x 2048
// bf16, 128 slots 4520 : 4336, 2413 x 3309 x 3904 fp32, 254 slots 1899 : 748, 2000 x 8000 x 1024 bf16, 64 slots 231 : 202, 2219 x 54900 x 1600
// fp16, 33 slots 405 : 414
bool target_lists(const gridmm_vocab_loss_t* d) {
  const double bytes = (double)d->rows * d->slots * d->hidden_size * (d->dtype == F32 ? 4 : 2);
  return d->slots && d->slots <= LIST_SLOTS && d->vocab <= LIST_BLOCKS * 64 - 256 && bytes / 7e6 > 12 + 2.8e-7 * d->rows * d->vocab;
}

struct Plan {
  int PL, slots;               // planes; target slots a row (cross entropy: 1)
  bool few, lists;
  int RP, groups, ranges, range;      // few rows: rows a group (16 or 32), groups; ranges of the vocabulary in dh and their rows
  int64_t Rp, Kp, Vp;
  bool pack_w;                 // W has to be split or padded; else it is read where it lies
  bool keep_w;                 // ... and its copy, one piece, stays for the backward (28 us of 396 at 30522 x 768 fp32)
  int64_t C_fwd, C_bwd;        // columns a piece
  // saved
  size_t o_meta, o_rowmap, o_rowinv, o_stat, o_zt, o_label, o_p, o_biasz, o_hexp, o_h, o_w, saved;
  // forward workspace
  size_t f_counts, f_plogp, f_amax, f_stats, f_w, f_begin, f_entry, fwd;
  // backward workspace
  size_t b_back, b_rowexp, b_weights, b_h2, b_ds, b_w, b_part, bwd;
};

bool make_plan(const gridmm_vocab_loss_t* d, Plan& P) {
  if (!d || d->rows < 0 || d->vocab < 1 || d->hidden_size < 1 || d->slots < 0 || d->dtype < 0 || d->dtype > 2 || d->bias_dtype < 0 ||
      d->bias_dtype > 2 || !(d->temperature >= 1e-6f) || !(d->temperature <= 1e6f) || d->rows > (1 << 20) || d->vocab > (1 << 27) ||
      d->hidden_size > (1 << 20) || d->slots > (1 << 16) || (!d->slots && d->temperature != 1.f))
    return false;
  P.PL = d->dtype == F32 ? 2 : 1;
  P.slots = d->slots ? d->slots : 1;
  P.Rp = (int64_t)up(d->rows, 256);
  P.Kp = (int64_t)up(d->hidden_size, 64);
  P.Vp = (int64_t)up(d->vocab, 256);
  // (a tile's 256 rows are addressed with 32-bit byte offsets: at most 2^31 from one row to the last where W lies)
  P.pack_w = d->packed || d->dtype == F32 || d->hidden_size % 64 || d->ld_weight % 8 || ((uintptr_t)d->weight & 15) || d->ld_weight > (1 << 22);
  // (grids: at most 2^32 threads)
  if ((P.Rp / 128) * (P.Vp / 128) > (1 << 23) || (int64_t)d->rows * ((P.slots + 7) / 8) > (1 << 25)) return false;
  // pieces: packed W and dS of at most `most` bytes each, whole tiles; but of dS 8192 columns (32 KB a row: more than that from 16384 rows
  // on), as dh's sums are read and written once a piece, and of W a tile's 256.  Forward and backward with 2048 : 8192 columns, ms:
  // 32768 x 32768 x 1024 bf16 16.3 : 12.8, 131072 rows of it 100 : 51, 131072 x 16384 x 4096 97 : 85, 131072 x 16384 x 1024 fp32 68 : 46
  const int64_t most = PIECE_MB << 20;
  auto piece = [&](int64_t bytes_a_column, int64_t least) {
    int64_t c = most / bytes_a_column / 256 * 256;
    if (c < least) c = least;
    if (c >= P.Vp) return P.Vp;
    const int64_t n = (P.Vp + c - 1) / c;                      // equal pieces
    return (int64_t)up((P.Vp + n - 1) / n, 256);
  };
  P.C_fwd = P.pack_w ? piece(P.Kp * 2 * P.PL, 256) : P.Vp;
  P.C_bwd = piece(std::max<int64_t>(P.Rp, 1) * 4, 8192);
  P.keep_w = P.pack_w && P.C_fwd == P.Vp;
  if (P.pack_w) P.C_bwd = std::min(P.C_bwd, P.C_fwd);
  P.few = few_rows(d);
  if (P.few) {
    P.RP = d->rows <= 16 ? 16 : 32;
    P.groups = std::max(1, (d->rows + P.RP - 1) / P.RP);
    // dh: four workgroups of 256 columns a CU (512, 1024, 2048 of them: 348, 238, 240 us at 131072 x 2048 fp32), at least 64
    // vocabulary rows a range
    const int64_t kb = (int64_t)((d->hidden_size + 255) / 256) * P.groups;
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>((1024 + kb - 1) / kb, d->vocab / 64));
    P.range = (int)up((d->vocab + n - 1) / n, 4);
    P.ranges = (d->vocab + P.range - 1) / P.range;
    size_t o = 0;
    auto take = [&](size_t bytes) { const size_t at = o; o += up(bytes, 256); return at; };
    const size_t V64 = up(d->vocab, 64), S = (size_t)d->rows * P.slots, GR = (size_t)P.groups * P.RP;
    P.o_stat = take(GR * 8);
    P.o_meta = take(GR * 4);                         // 1 for rows that count
    P.o_zt = take(S * 4);
    P.o_p = take(d->slots ? S * 4 : 0);
    P.o_h = take(d->forward_only ? 0 : V64 * GR * 4);      // the scores
    P.f_stats = take(V64 / 64 * GR * 8);             // (small enough to stay: no forward workspace)
    P.saved = o;
    P.fwd = 0;
    o = 0;
    P.b_ds = take(V64 * GR * 4);
    P.b_part = take((size_t)P.ranges * GR * up(d->hidden_size, 4) * 4);
    P.bwd = o;
    return true;
  }
  const size_t R = (size_t)std::max(d->rows, 1), Rp = (size_t)std::max<int64_t>(P.Rp, 256), S = P.slots;
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o += up(bytes, 256); return at; };
  P.o_meta = take(sizeof(Meta));
  P.o_rowmap = take(R * 4);
  P.o_rowinv = take(R * 4);
  P.o_stat = take(Rp * 8);
  P.o_zt = take(R * S * 4);
  P.o_label = take(d->slots ? 0 : R * 4);
  P.o_p = take(d->slots ? R * S * 4 : 0);
  P.o_biasz = take(P.Vp * 4);
  P.o_hexp = take(d->dtype == BF16 ? 0 : Rp * 4);
  P.o_h = take(Rp * P.Kp * 2 * P.PL);
  P.o_w = take(P.keep_w ? (size_t)P.Vp * P.Kp * 2 * P.PL : 0);
  P.saved = o;
  o = 0;
  P.f_counts = take(R);
  P.f_plogp = take(R * 4);
  P.f_amax = take((AMAX_H + AMAX_W) * 4);
  P.f_stats = take(Rp * (size_t)(P.Vp / 128) * 8);
  P.f_w = take(P.pack_w && !P.keep_w ? (size_t)P.C_fwd * P.Kp * 2 * P.PL : 0);
  P.lists = target_lists(d);
  P.f_begin = take(P.lists ? R * (P.Vp / 64 + 1) * 2 : 0);
  P.f_entry = take(P.lists ? R * S * 4 : 0);
  P.fwd = o;
  o = 0;
  P.b_back = take(sizeof(Back));
  P.b_rowexp = take(d->dtype == BF16 ? 0 : Rp * 4);
  P.b_weights = take(d->dtype == BF16 ? 0 : (Rp + 2048) * 2);
  P.b_h2 = take(d->dtype == BF16 ? 0 : Rp * P.Kp * 2 * P.PL);
  P.b_ds = take(Rp * (size_t)P.C_bwd * 4);
  P.b_w = take(P.pack_w && !P.keep_w ? (size_t)P.C_bwd * P.Kp * 2 * P.PL : 0);
  P.b_part = take(std::max<size_t>(Rp * (size_t)P.Kp, std::min<size_t>(MOST_SPLITS * Rp * (size_t)P.Kp, PART_MOST)) * 4);
  P.bwd = o;
  return true;
}

template <bool F16V, int PL, bool BIG, bool CA, bool CB>
using TileOf = typename std::conditional<BIG, Tile<F16V, PL, 256, 256, 128, 64, CA, CB>, Tile<F16V, PL, 128, 128, 64, 64, CA, CB>>::type;

// workgroups for so many tiles: what the chip holds at once, each then walks several
template <class T>
unsigned blocks(int64_t tiles) { return (unsigned)std::min<int64_t>(tiles, 256 * T::PER_CU); }

// calls f(type)
template <class F>
int by_dtype(const gridmm_vocab_loss_t* d, F f) {
  if (d->dtype == F32) return f(std::integral_constant<int, F32>{});
  if (d->dtype == BF16) return f(std::integral_constant<int, BF16>{});
  return f(std::integral_constant<int, F16>{});
}
// calls f(fp16?, planes) for the operands' type
template <class F>
int by_type(const gridmm_vocab_loss_t* d, F f) {
  using std::bool_constant;
  using std::integral_constant;
  if (d->dtype == F32) return f(bool_constant<true>{}, integral_constant<int, 2>{});
  if (d->dtype == F16) return f(bool_constant<true>{}, integral_constant<int, 1>{});
  return f(bool_constant<false>{}, integral_constant<int, 1>{});
}
// calls f(big?, rows) for each tile that a count of at most `rows` may ask for, with the most rows it is asked for
template <class F>
int by_tile(int rows, int64_t C, F f) {
  // the largest count that takes the small tile
  const int64_t small = std::max<int64_t>(256, (BIG_TILES + C / 256 - 1) / (C / 256) * 256 - 256);
  int rc = f(std::bool_constant<false>{}, (int)std::min<int64_t>(rows, small));
  if (rc == GRIDMM_OK && rows > small) rc = f(std::bool_constant<true>{}, rows);
  return rc;
}

// W's rows [j0, j0 + C) as an operand: packed into `buf` (kept: all of it in `kept`, where the forward packs it) or in place
int weight_piece(const gridmm_vocab_loss_t* d, const Plan& P, int64_t j0, int64_t C, const Meta* meta, unsigned short* kept, bool forward,
                 unsigned short* buf, hipStream_t st, Operand& W) {
  if (!P.pack_w) {
    W = Operand{(const unsigned short*)d->weight + j0 * d->ld_weight, d->ld_weight, 0, d->vocab - j0, P.Kp};
    return GRIDMM_OK;
  }
  if (P.keep_w) buf = kept + j0 * P.PL * P.Kp;
  if (forward ? j0 > 0 : !P.keep_w) {             // (the forward's first piece: rows_kernel)
    GRIDMM_LAUNCH(pack_w_kernel, dim3((unsigned)((C + 3) / 4)), dim3(256), 0, st, d->weight, d->ld_weight, d->dtype, d->hidden_size,
                  (int)P.Kp, j0, (int)C, d->vocab, meta, buf);
    GRIDMM_CHECK_LAUNCH();
  }
  W = Operand{buf, P.PL * P.Kp, P.Kp, C, P.Kp};
  return GRIDMM_OK;
}

bool bad_pointers(const gridmm_vocab_loss_t* d, const void* saved, bool forward) {
  if (!d->weight || !saved || d->ld_weight < d->hidden_size || ((uintptr_t)saved & 255)) return true;
  if (d->rows && (!d->hidden || d->ld_hidden < d->hidden_size)) return true;
  if (d->rows && d->slots && (!d->ids || d->ld_ids < d->slots)) return true;
  if (d->rows && d->slots && forward && (!d->teacher || d->ld_teacher < d->slots)) return true;
  if (d->rows && !d->slots && !d->labels) return true;
  return false;
}

// calls f(type, tiles of 16 rows, whole vectors)
template <class F>
int by_few(const gridmm_vocab_loss_t* d, const Plan& P, F f) {
  const bool vec = few_vectors(d);
  auto rows = [&](auto dt) {
    auto one = [&](auto rt) { return vec ? f(dt, rt, std::true_type{}) : f(dt, rt, std::false_type{}); };
    return P.RP == 16 ? one(std::integral_constant<int, 1>{}) : one(std::integral_constant<int, 2>{});
  };
  return by_dtype(d, rows);
}
FewArgs few_args(const gridmm_vocab_loss_t* d, const Plan& P, const void* saved) {
  FewArgs a{};
  char* sv = (char*)saved;
  a.hidden = d->hidden; a.weight = d->weight; a.bias = d->bias; a.index = d->slots ? d->ids : d->labels; a.teacher = d->teacher;
  a.ldh = d->ld_hidden; a.ldw = d->ld_weight; a.ld_index = d->slots ? d->ld_ids : 1; a.ld_teacher = d->ld_teacher; a.ignore = d->ignore_index;
  a.rows = d->rows; a.vocab = d->vocab; a.K = d->hidden_size; a.slots = P.slots; a.wide = d->index64; a.dtype = d->dtype;
  a.bias_dtype = d->bias_dtype; a.kd = d->slots > 0;
  a.inv_t = 1.f / d->temperature; a.unit = a.inv_t * LOG2E; a.temperature = d->temperature;
  a.stat = (float2*)(sv + P.o_stat); a.flag = (float*)(sv + P.o_meta); a.zt = (float*)(sv + P.o_zt);
  a.p = d->slots ? (float*)(sv + P.o_p) : nullptr;
  a.y = d->forward_only ? nullptr : (float*)(sv + P.o_h);
  a.ranges = P.ranges; a.range = P.range; a.groups = P.groups;
  a.group_dS = (int64_t)up(d->vocab, 64) * P.RP;
  return a;
}

}  // namespace

extern "C" size_t gridmm_vocab_loss_saved_bytes(const gridmm_vocab_loss_t* d) {
  Plan P;
  return make_plan(d, P) ? P.saved : 0;
}

extern "C" size_t gridmm_vocab_loss_workspace(const gridmm_vocab_loss_t* d, int backward) {
  Plan P;
  return make_plan(d, P) ? (backward ? P.bwd : P.fwd) : 0;
}

extern "C" int gridmm_vocab_loss_fwd(const gridmm_vocab_loss_t* d, float* loss, void* saved, size_t saved_bytes, void* workspace,
                                     size_t workspace_bytes, gridmm_stream_t stream) {
  Plan P;
  if (!make_plan(d, P) || bad_pointers(d, saved, true) || saved_bytes < P.saved || (P.fwd && !workspace) ||
      workspace_bytes < P.fwd || ((uintptr_t)workspace & 255) || (d->rows && !loss))
    return GRIDMM_EINVAL;
  if (d->rows == 0) return GRIDMM_OK;
  hipStream_t st = as_stream(stream);
  char *sv = (char*)saved, *ws = (char*)workspace;
  if (P.few) {
    FewArgs a = few_args(d, P, saved);
    a.stats = (float2*)(sv + P.f_stats);
    a.loss = loss;
    const int tiles = (d->vocab + 63) / 64;
    const int rc = by_few(d, P, [&](auto dt, auto rt, auto vec) {
      GRIDMM_LAUNCH((few_scores_kernel<decltype(dt)::value, decltype(rt)::value, decltype(vec)::value>), dim3(tiles, P.groups), dim3(256), 0, st, a);
      GRIDMM_CHECK_LAUNCH();
      return GRIDMM_OK;
    });
    if (rc != GRIDMM_OK) return rc;
    GRIDMM_LAUNCH(few_loss_kernel, dim3(d->rows), dim3(256), 0, st, a, (int64_t)tiles, P.RP);
    GRIDMM_CHECK_LAUNCH();
    return GRIDMM_OK;
  }
  Meta* meta = (Meta*)(sv + P.o_meta);
  int *rowmap = (int*)(sv + P.o_rowmap), *rowinv = (int*)(sv + P.o_rowinv);
  float2* stat = (float2*)(sv + P.o_stat);
  float *zt = (float*)(sv + P.o_zt), *p = d->slots ? (float*)(sv + P.o_p) : nullptr;
  float* biasz = (float*)(sv + P.o_biasz);
  unsigned short* Hp = (unsigned short*)(sv + P.o_h);
  unsigned char* counts = (unsigned char*)(ws + P.f_counts);
  float* plogp = (float*)(ws + P.f_plogp);
  int* amax = (int*)(ws + P.f_amax);
  float2* stats = (float2*)(ws + P.f_stats);
  const float inv_t = 1.f / d->temperature, unit = inv_t * LOG2E;

  if (d->slots) {
    GRIDMM_LAUNCH(kd_targets_kernel, dim3((d->rows + 3) / 4), dim3(256), 0, st, d->ids, d->index64, d->ld_ids, d->teacher,
                  d->ld_teacher, d->rows, d->slots, inv_t, p, plogp, counts);
    GRIDMM_CHECK_LAUNCH();
  }
  PrepArgs a;
  a.hidden = d->hidden; a.weight = d->weight; a.bias = d->bias; a.labels = d->labels;
  a.counts = d->slots ? counts : nullptr;
  a.ldh = d->ld_hidden; a.ldw = d->ld_weight; a.ignore = d->ignore_index;
  a.rows = d->rows; a.vocab = d->vocab; a.K = d->hidden_size; a.wide = d->index64; a.dtype = d->dtype; a.bias_dtype = d->bias_dtype;
  a.vp = (int)P.Vp; a.unit = unit; a.meta = meta; a.rowmap = rowmap; a.rowinv = rowinv; a.loss = loss; a.biasz = biasz;
  a.amax_h = amax; a.amax_w = amax + AMAX_H;
  const int nb = (int)((P.Vp + PREP_T - 1) / PREP_T);
  GRIDMM_LAUNCH(prep_kernel, dim3(1 + nb + (d->dtype == F32 ? AMAX_H + AMAX_W : 0)), dim3(PREP_T), 0, st, a, nb);
  GRIDMM_CHECK_LAUNCH();
  TargetArgs t;
  t.hidden = d->hidden; t.weight = d->weight; t.index = d->slots ? d->ids : d->labels;
  t.ldh = d->ld_hidden; t.ldw = d->ld_weight; t.ld_index = d->slots ? d->ld_ids : 1;
  t.K = d->hidden_size; t.vocab = d->vocab; t.slots = P.slots; t.wide = d->index64; t.kd = d->slots > 0;
  t.bias = d->bias; t.bias_dtype = d->bias_dtype; t.unit = unit; t.meta = meta; t.rowmap = rowmap; t.zt = zt;
  t.label = d->slots ? nullptr : (int*)(sv + P.o_label);
  const int rc = by_dtype(d, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const int hb = (int)(P.Rp / 4), tb = P.lists ? 0 : (int)(((int64_t)d->rows * P.slots + 31) / 32);
    const int C = P.pack_w ? (int)P.C_fwd : 0;
    unsigned short* Wp = (unsigned short*)(P.keep_w ? sv + P.o_w : ws + P.f_w);
    const dim3 grid((unsigned)(hb + tb + (C + 3) / 4));
    GRIDMM_LAUNCH((rows_kernel<DT>), grid, dim3(256), 0, st, t, hb, tb, (int)P.Kp, amax, amax + AMAX_H, meta, Hp,
                  d->forward_only ? nullptr : (int*)(sv + P.o_hexp), C, Wp);
    GRIDMM_CHECK_LAUNCH();
    return GRIDMM_OK;
  });
  if (rc != GRIDMM_OK) return rc;

  TargetLists lists{};
  if (P.lists) {
    unsigned short* begin = (unsigned short*)(ws + P.f_begin);
    unsigned* entry = (unsigned*)(ws + P.f_entry);
    lists = TargetLists{begin, entry, P.Vp / 64, P.slots, zt, d->bias, d->bias_dtype, 0.5f * unit};
    GRIDMM_LAUNCH(target_lists_kernel, dim3(d->rows), dim3(256), 0, st, t, (int)lists.blocks, begin, entry);
    GRIDMM_CHECK_LAUNCH();
  }
  const Operand H{Hp, P.PL * P.Kp, P.Kp, P.Rp, P.Kp};
  for (int64_t j0 = 0; j0 < P.Vp; j0 += P.C_fwd) {
    const int64_t C = std::min(P.C_fwd, P.Vp - j0);
    const Raw raw{d->hidden, d->weight, d->ld_hidden, d->ld_weight, j0, d->hidden_size, d->vocab, rowmap};
    Operand W;
    int rc = weight_piece(d, P, j0, C, meta, (unsigned short*)(sv + P.o_w), true, (unsigned short*)(ws + P.f_w), st, W);
    if (rc != GRIDMM_OK) return rc;
    rc = by_type(d, [&](auto f16, auto pl) {
      return by_tile(d->rows, C, [&](auto big, int rows) {
        using T = TileOf<decltype(f16)::value, decltype(pl)::value, decltype(big)::value, false, false>;
        const int64_t tn = C / T::BN, tm = (rows + T::BM - 1) / T::BM;
        auto run = [&](auto with) {
          GRIDMM_LAUNCH((score_stats_kernel<T, decltype(with)::value>), dim3(blocks<T>(tm * tn)), dim3(T::THREADS), 0, st, H, W,
                        (int)(P.Kp / T::BK), (int)tn, meta, biasz + j0, unit, stats + j0 / 128 * P.Rp, P.Rp, lists, raw);
          GRIDMM_CHECK_LAUNCH();
          return GRIDMM_OK;
        };
        return P.lists ? run(std::true_type{}) : run(std::false_type{});
      });
    });
    if (rc != GRIDMM_OK) return rc;
  }
  GRIDMM_LAUNCH(loss_kernel, dim3((d->rows + 15) / 16), dim3(256), 0, st, stats, P.Vp, P.C_fwd, P.Rp, meta, rowmap, zt, P.slots, p,
                plogp, d->temperature, stat, loss);
  GRIDMM_CHECK_LAUNCH();
  return GRIDMM_OK;
}

extern "C" int gridmm_vocab_loss_bwd(const gridmm_vocab_loss_t* d, const void* saved, size_t saved_bytes, const float* grad,
                                     int64_t grad_stride, void* d_hidden, void* d_weight, void* d_bias, void* workspace,
                                     size_t workspace_bytes, gridmm_stream_t stream) {
  Plan P;
  if (!make_plan(d, P) || bad_pointers(d, saved, false) || saved_bytes < P.saved || !workspace || workspace_bytes < P.bwd ||
      ((uintptr_t)workspace & 255) || (d->rows && (!grad || (!d_hidden && !d_weight && !d_bias))) || grad_stride < 0 ||
      (d_bias && !d->bias) || d->forward_only)
    return GRIDMM_EINVAL;
  hipStream_t st = as_stream(stream);
  if (d->rows == 0) {                       // nothing counts: the shared gradients are zero
    if (!d_weight && !d_bias) return GRIDMM_OK;
    const int64_t nw = (int64_t)d->vocab * d->hidden_size * (d->dtype == F32 ? 2 : 1), nb = (int64_t)d->vocab * (d->bias_dtype == F32 ? 2 : 1);
    if (d_weight) GRIDMM_LAUNCH(zero_u16_kernel, dim3((unsigned)std::min<int64_t>((nw + 255) / 256, 4096)), dim3(256), 0, st, (unsigned short*)d_weight, nw);
    if (d_bias) GRIDMM_LAUNCH(zero_u16_kernel, dim3((unsigned)std::min<int64_t>((nb + 255) / 256, 4096)), dim3(256), 0, st, (unsigned short*)d_bias, nb);
    GRIDMM_CHECK_LAUNCH();
    return GRIDMM_OK;
  }
  const char* sv = (const char*)saved;
  char* ws = (char*)workspace;
  if (P.few) {
    FewArgs a = few_args(d, P, saved);
    a.grad = grad; a.grad_stride = grad_stride;
    a.dS = (float*)(ws + P.b_ds); a.part = (float*)(ws + P.b_part);
    a.dh = d_hidden; a.dW = d_weight; a.db = d_bias;
    const int tiles = (d->vocab + 63) / 64, kb = (d->hidden_size + 255) / 256;
    const int hb = d_hidden ? kb * P.ranges * P.groups : 0, wb = d_weight || d_bias ? (d->vocab + 16 * FEW_J - 1) / (16 * FEW_J) : 0;
    const int rc = by_few(d, P, [&](auto dt, auto rt, auto vec) {
      GRIDMM_LAUNCH((few_grad_kernel<decltype(rt)::value>), dim3(tiles, P.groups), dim3(256), 0, st, a);
      GRIDMM_CHECK_LAUNCH();
      GRIDMM_LAUNCH((few_products_kernel<decltype(dt)::value, decltype(rt)::value, decltype(vec)::value>), dim3(hb + wb), dim3(256), 0, st, a, hb, kb);
      GRIDMM_CHECK_LAUNCH();
      return GRIDMM_OK;
    });
    if (rc != GRIDMM_OK) return rc;
    if (d_hidden) {
      GRIDMM_LAUNCH(few_hidden_kernel, dim3(d->rows, (d->hidden_size + 63) / 64), dim3(256), 0, st, a, P.RP);
      GRIDMM_CHECK_LAUNCH();
    }
    return GRIDMM_OK;
  }
  const Meta* meta = (const Meta*)(sv + P.o_meta);
  Back* back = (Back*)(ws + P.b_back);
  const bool scaled = d->dtype != BF16;
  int* rowexp = scaled ? (int*)(ws + P.b_rowexp) : nullptr;
  unsigned short* weights = scaled ? (unsigned short*)(ws + P.b_weights) : nullptr;
  const int *rowmap = (const int*)(sv + P.o_rowmap), *rowinv = (const int*)(sv + P.o_rowinv);
  const float2* stat = (const float2*)(sv + P.o_stat);
  const float* zt = (const float*)(sv + P.o_zt);
  const float *p = d->slots ? (const float*)(sv + P.o_p) : nullptr, *biasz = (const float*)(sv + P.o_biasz);
  const unsigned short* Hp = (const unsigned short*)(sv + P.o_h);
  float* part = (float*)(ws + P.b_part);
  unsigned short *dS = (unsigned short*)(ws + P.b_ds), *wbuf = (unsigned short*)(ws + P.b_w);
  const float unit = LOG2E / d->temperature;

  const GradArgs G{grad, grad_stride, d->temperature, rowmap, d->slots ? nullptr : (const int*)(sv + P.o_label), zt, stat, rowexp, scaled ? back : nullptr};
  const Operand H{Hp, P.PL * P.Kp, P.Kp, P.Rp, P.Kp};
  Operand H2 = H;                          // of dW
  if (scaled) {
    unsigned short* h2 = (unsigned short*)(ws + P.b_h2);
    GRIDMM_LAUNCH(grad_scales_kernel, dim3((unsigned)std::min<int64_t>(P.Rp / 4, 1024)), dim3(256), 0, st, G, meta, (const int*)(sv + P.o_hexp), P.PL,
                  (int)P.Kp, Hp, h2, weights, rowexp, back);
    GRIDMM_CHECK_LAUNCH();
    H2.p = h2;
  }
  for (int64_t j0 = 0; j0 < P.Vp; j0 += P.C_bwd) {
    const int64_t C = std::min(P.C_bwd, P.Vp - j0);
    const Raw raw{d->hidden, d->weight, d->ld_hidden, d->ld_weight, j0, d->hidden_size, d->vocab, rowmap};
    Operand W;
    int rc = weight_piece(d, P, j0, C, meta, (unsigned short*)(sv + P.o_w), false, wbuf, st, W);
    if (rc != GRIDMM_OK) return rc;
    const int64_t ldS = 2 * C;
    const Operand S{dS, ldS, C, P.Rp, C};
    rc = by_type(d, [&](auto f16, auto pl) {
      constexpr bool F = decltype(f16)::value;
      constexpr int L = decltype(pl)::value;
      int rc = by_tile(d->rows, C, [&](auto big, int rows) {
        using T = TileOf<F, L, decltype(big)::value, false, false>;
        const int64_t tn = C / T::BN, tm = (rows + T::BM - 1) / T::BM;
        GRIDMM_LAUNCH((score_grad_kernel<T>), dim3(blocks<T>(tm * tn)), dim3(T::THREADS), 0, st, H, W, (int)(P.Kp / T::BK), (int)tn, meta, biasz + j0,
                      unit, G, raw, dS, C);
        GRIDMM_CHECK_LAUNCH();
        return GRIDMM_OK;
      });
      if (rc != GRIDMM_OK) return rc;
      if (d->slots) {
        FixArgs f;
        f.index = d->ids; f.ld_index = d->ld_ids; f.j0 = j0; f.ldS = ldS; f.plane = C;
        f.wide = d->index64; f.slots = P.slots; f.C = (int)C; f.vocab = d->vocab; f.dtype = d->dtype; f.meta = meta; f.G = G;
        f.p = p; f.dS = dS;
        GRIDMM_LAUNCH(target_grad_kernel, dim3(d->rows), dim3(256), 0, st, f);
        GRIDMM_CHECK_LAUNCH();
      }
      if (d_hidden) {
        rc = by_tile(d->rows, P.C_bwd, [&](auto big, int rows) {
          using T = TileOf<F, L, decltype(big)::value, false, true>;
          const int64_t tn = (P.Kp + T::BN - 1) / T::BN, tm = (rows + T::BM - 1) / T::BM;
          GRIDMM_LAUNCH((hidden_grad_kernel<T>), dim3(blocks<T>(tm * tn * MOST_SPLITS)), dim3(T::THREADS), 0, st, S, W, (int)(C / T::BK), (int)tn,
                        P.C_bwd, meta, part, P.Kp, j0 == 0, back, raw);
          GRIDMM_CHECK_LAUNCH();
          return GRIDMM_OK;
        });
        if (rc != GRIDMM_OK) return rc;
      }
      if (d_weight || d_bias) {
        auto weight = [&](auto big) {
          using T = TileOf<F, L, decltype(big)::value, true, true>;
          const int64_t tn = d_weight ? (P.Kp + T::BN - 1) / T::BN : 1, tm = C / T::BM;      // (db alone: the first tile column)
          GRIDMM_LAUNCH((weight_grad_kernel<T>), dim3(blocks<T>(tm * tn)), dim3(T::THREADS), 0, st, S, H2, (int)tm, (int)tn, meta, back, weights, d->dtype, j0,
                        d->vocab, d->hidden_size, d_weight, d->bias_dtype, d_bias, raw);
          GRIDMM_CHECK_LAUNCH();
          return GRIDMM_OK;
        };
        rc = C / 256 * ((P.Kp + 255) / 256) >= BIG_TILES ? weight(std::true_type{}) : weight(std::false_type{});
        if (rc != GRIDMM_OK) return rc;
      }
      return GRIDMM_OK;
    });
    if (rc != GRIDMM_OK) return rc;
  }
  if (d_hidden) {
    GRIDMM_LAUNCH(hidden_out_kernel, dim3(d->rows, (unsigned)((P.Kp + 255) / 256)), dim3(256), 0, st, part, P.Kp, d->hidden_size,
                  d->rows, rowinv, meta, rowexp, back, d->dtype, d_hidden);
    GRIDMM_CHECK_LAUNCH();
  }
  return GRIDMM_OK;
}
