// The vocabulary losses for few rows, and for small products of any number of rows (few_rows() in vocab_loss.hip): a handful of tokens
// against the whole vocabulary is bound by the read of W and, backward, the write of dW, a small head by its launches; tiles of 128
// rows, packed copies and a dozen launches cost more than the work.  Two launches forward, three backward, rows where they lie,
// nothing packed.  Rows go in groups of RP = 16 RT:
//   few_scores   16 vocabulary rows a wave, a group's RT tiles of 16 rows of h: each W value is loaded once, straight into the fragment layout
//                of the 16x16 matrix instructions (fp32: 16x16x4 fp32, products and sums in fp32; 16 bits: 16x16x32, products exact).
//                Forward: each row's (maximum, sum of exponentials) of the workgroup's 64 columns, and the targets' scores.
//                The scores stay for the backward, fp32 [group][vocabulary][RP]: a few percent of W's size, whose third read they save
//   few_grad     scores -> dS, laid out alike
//   few_loss     joins the statistics, the teacher's softmax, the losses
//   few_products dh = dS W over ranges of the vocabulary and dW = dS^T h, db, on the fp32 matrix instruction (16-bit operands are
//                widened: exact), as two kinds of workgroups of one launch
//   few_hidden   joins the ranges of dh
// One token of 30522 x 768 fp32: 24 us (3.9 TB/s); 4 rows of 131072 x 2048 fp32 forward 257 us (4.2 TB/s); 32 rows 423, where the reads of h count.
// dS is never rounded to 16 bits here.  A row that does not count has dS = 0 and its h is read as 0.
#pragma once
#include "vocab_gemm.h"

namespace {

typedef float few_f4 __attribute__((ext_vector_type(4)));

struct FewArgs {
  const void *hidden, *weight, *bias, *index;
  const float* teacher;
  int64_t ldh, ldw, ld_index, ld_teacher, ignore;
  int rows, vocab, K, slots, wide, dtype, bias_dtype, kd;
  float inv_t, unit, temperature;
  float2* stats;                 // [workgroup][groups RP]
  float2* stat;                  // saved: [groups RP] maximum and sum
  float *zt, *p, *flag;          // saved: [rows][slots] (halves), [rows][slots], [groups RP]: 1 for rows that count
  float* y;                      // saved: the scores, base 2, laid out like dS; NULL: no backward will follow
  float* loss;
  const float* grad;
  int64_t grad_stride;
  float *dS, *part;              // [group][vocab up to 64][RP], [ranges][groups RP][K up to 4]
  void *dh, *dW, *db;
  int ranges, range;             // of the vocabulary in dh, rows a range (a multiple of 4)
  int groups;
  int64_t group_dS;              // values of dS a group
};

template <int DT>
__device__ __forceinline__ float few_1(const void* p, int64_t i) { return load_as_f32(p, i, DT); }

// Vectors on the boundaries of their elements: this chip's global loads take them, at up to twice the cache accesses.  Value by value
// they took 2 - 3 times as long (16 bits, 1379 hidden).
typedef float few_f4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short few_u4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef short few_s8_any __attribute__((ext_vector_type(8), aligned(2)));

// values k .. k + 3 of a row, widened.  FULL: all of them are the row's; else zero from K on
template <int DT, bool VEC, bool FULL>
__device__ __forceinline__ few_f4 few_load4(const void* p, int64_t off, int k, int K) {
  few_f4 v = {0.f, 0.f, 0.f, 0.f};
  if constexpr (VEC || FULL) {               // (VEC: K % 4 == 0)
    const int at = FULL || k < K ? k : 0;
    if constexpr (DT == F32) {
      if constexpr (VEC) v = *reinterpret_cast<const few_f4*>((const float*)p + off + at);
      else v = *reinterpret_cast<const few_f4_any*>((const float*)p + off + at);
    } else {
      u16x4_t u;
      if constexpr (VEC) u = *reinterpret_cast<const u16x4_t*>((const unsigned short*)p + off + at);
      else u = *reinterpret_cast<const few_u4_any*>((const unsigned short*)p + off + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = DT == BF16 ? bf16_bits_to_f32(u[e]) : (float)__builtin_bit_cast(_Float16, (unsigned short)u[e]);
    }
    if (!FULL && k >= K) v = (few_f4){0.f, 0.f, 0.f, 0.f};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < K) v[e] = few_1<DT>(p, off + k + e);
  }
  return v;
}
// values k .. k + 7 of a 16-bit row as they are, likewise
template <bool VEC, bool FULL>
__device__ __forceinline__ vocab::s16x8_t few_load8(const void* p, int64_t off, int k, int K) {
  vocab::s16x8_t v = {0, 0, 0, 0, 0, 0, 0, 0};
  const short* x = (const short*)p + off;
  if constexpr (VEC) {                                 // K % 8 == 0
    v = *reinterpret_cast<const vocab::s16x8_t*>(x + (FULL || k < K ? k : 0));
    if (!FULL && k >= K) v = (vocab::s16x8_t){0, 0, 0, 0, 0, 0, 0, 0};
  } else if constexpr (FULL) {
    v = *reinterpret_cast<const few_s8_any*>(x + k);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < K) v[e] = x[k + e];
  }
  return v;
}

// Scores of the wave's 16 vocabulary rows from j0 on: lane l has rows of h r0 + 16 t + (l & 15), columns j0 + 4 (l >> 4) + i, base 2, bias
// in; -inf past the vocabulary.
template <int DT, int RT, bool VEC>
__device__ __forceinline__ void few_tile(const FewArgs& a, int r0, int64_t j0, f32x4_t (&acc)[RT]) {
  const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
  const int64_t j = j0 + l15 < a.vocab ? j0 + l15 : a.vocab - 1;
  int64_t ho[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = r0 + t * 16 + l15;
    ho[t] = (int64_t)(r < a.rows ? r : a.rows - 1) * a.ldh;
    acc[t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
  using std::bool_constant;
  using std::integral_constant;
  // 16 bits: U steps' loads in flight together (fp32 measured slower so: 372 against 240 us at 131072 x 2048)
  if constexpr (DT == F32) {
    auto step = [&](int k0, auto full) {
      constexpr bool FULL = decltype(full)::value;
      const few_f4 w = few_load4<DT, VEC, FULL>(a.weight, j * a.ldw, k0 + 4 * g, a.K);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const few_f4 h = few_load4<DT, VEC, FULL>(a.hidden, ho[t], k0 + 4 * g, a.K);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[e], h[e], acc[t], 0, 0, 0);
      }
    };
    const int whole = a.K / 16 * 16;
#pragma unroll 4
    for (int k0 = 0; k0 < whole; k0 += 16) step(k0, bool_constant<true>{});
    if (whole < a.K) step(whole, bool_constant<false>{});
  } else {
    auto steps = [&](int k0, auto full, auto n) {
      constexpr bool FULL = decltype(full)::value;
      constexpr int N = decltype(n)::value;
      vocab::s16x8_t w[N], h[N][RT];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int k = k0 + 32 * u + 8 * g;
        w[u] = few_load8<VEC, FULL>(a.weight, j * a.ldw, k, a.K);
#pragma unroll
        for (int t = 0; t < RT; ++t) h[u][t] = few_load8<VEC, FULL>(a.hidden, ho[t], k, a.K);
      }
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if constexpr (DT == BF16)
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w[u]), __builtin_bit_cast(bf16x8_t, h[u][t]), acc[t], 0, 0, 0);
          else
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w[u]), __builtin_bit_cast(f16x8_t, h[u][t]), acc[t], 0, 0, 0);
        }
    };
    constexpr int U = RT == 1 ? 8 : 6;
    if constexpr (VEC) {
      for (int k0 = 0; k0 < a.K; k0 += 32 * U) steps(k0, bool_constant<false>{}, integral_constant<int, U>{});
    } else {
      int k0 = 0;
      for (; k0 + 32 * U <= a.K; k0 += 32 * U) steps(k0, bool_constant<true>{}, integral_constant<int, U>{});
      for (; k0 + 32 <= a.K; k0 += 32) steps(k0, bool_constant<true>{}, integral_constant<int, 1>{});
      if (k0 < a.K) steps(k0, bool_constant<false>{}, integral_constant<int, 1>{});
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = j0 + 4 * g + i;
    const float b = c >= a.vocab ? -INFINITY : a.bias ? load_as_f32(a.bias, c, a.bias_dtype) * a.unit : 0.f;
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t][i] = c >= a.vocab ? -INFINITY : fmaf(acc[t][i], a.unit, b);
  }
}

// The targets of a group's rows among a workgroup's 64 columns, found together: wave w looks through the rows w, w + 4, .. and keeps a
// list of its own, in the order of (row, slot).  With few slots, or more hits than a list holds, each lane looks through its row.
struct FewTargets {
  unsigned list[4][256];
  int n[4];
};
constexpr int FEW_SLOTS_EACH = 4;
template <int RP>
__device__ __forceinline__ void few_collect(const FewArgs& a, int r0, FewTargets& T) {
  if (a.slots <= FEW_SLOTS_EACH) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t j0 = (int64_t)blockIdx.x * 64;
  int n = 0;
  for (int r = wave; r < RP && r0 + r < a.rows; r += 4)
    for (int s0 = 0; s0 < a.slots; s0 += 64) {
      const int s = s0 + lane;
      const int64_t id = s < a.slots ? load_index(a.index, (int64_t)(r0 + r) * a.ld_index + s, a.wide) : -1;
      const bool hit = id >= j0 && id < j0 + 64 && id < a.vocab;
      const uint64_t b = __ballot(hit);
      const int at = n + __popcll(b & ((1ull << lane) - 1));
      if (hit && at < 256) T.list[wave][at] = (unsigned)r | (unsigned)(id - j0) << 5 | (unsigned)s << 11;
      n += __popcll(b);
    }
  if (lane == 0) T.n[wave] = n;
  __syncthreads();
}
// f(slot, d) for the targets of row r = r0 + local among the lane's 4 columns from jl on, in the order of the slots
template <class F>
__device__ __forceinline__ void few_targets(const FewArgs& a, const FewTargets& T, int r0, int local, int64_t jl, F f) {
  if (a.slots > FEW_SLOTS_EACH && T.n[0] <= 256 && T.n[1] <= 256 && T.n[2] <= 256 && T.n[3] <= 256) {
    const unsigned c0 = (unsigned)(jl - (int64_t)blockIdx.x * 64);
    const int w = local & 3;
    for (int e = 0; e < T.n[w]; ++e) {
      const unsigned v = T.list[w][e], d = ((v >> 5) & 63) - c0;
      if ((int)(v & 31) == local && d < 4) f((int)(v >> 11), (int)d);
    }
    return;
  }
  for (int k0 = 0; k0 < a.slots; k0 += 8) {
    int64_t d[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      d[u] = load_index(a.index, (int64_t)(r0 + local) * a.ld_index + (k0 + u < a.slots ? k0 + u : a.slots - 1), a.wide) - jl;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (k0 + u < a.slots && (uint64_t)d[u] < 4 && jl + d[u] < a.vocab) f(k0 + u, (int)d[u]);
  }
}

// VEC: the rows of h and W are whole 16-byte vectors on their boundaries (decided once a call: a choice at each load would wait for it)
template <int DT, int RT, bool VEC>
__global__ __launch_bounds__(256) void few_scores_kernel(const FewArgs a) {
  __shared__ float2 wst[4][RT * 16];
  __shared__ FewTargets T;
  constexpr int RP = RT * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int64_t j0 = (int64_t)blockIdx.x * 64 + wave * 16, jl = j0 + 4 * g;
  f32x4_t y[RT];
  const int r0 = blockIdx.y * RP;
  few_collect<RP>(a, r0, T);
  few_tile<DT, RT, VEC>(a, r0, j0, y);
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = r0 + t * 16 + l15;
    if (a.y) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a.y[blockIdx.y * a.group_dS + (jl + i) * RP + t * 16 + l15] = y[t][i];
    }
    float m = fmaxf(fmaxf(y[t][0], y[t][1]), fmaxf(y[t][2], y[t][3]));
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += __builtin_amdgcn_exp2f(y[t][i] - ref);
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    if (g == 0) wst[wave][t * 16 + l15] = make_float2(m, s);
    if (r < a.rows)                           // the scores at the row's targets
      few_targets(a, T, r0, t * 16 + l15, jl, [&](int k, int d) {
        const float v = d < 2 ? (d == 0 ? y[t][0] : y[t][1]) : (d == 2 ? y[t][2] : y[t][3]);
        // half of it: a bias of the lowest finite number, -inf in base 2, is finite so
        a.zt[(int64_t)r * a.slots + k] = v == -INFINITY && a.bias ? load_as_f32(a.bias, jl + d, a.bias_dtype) * (0.5f * a.unit) : 0.5f * v;
      });
  }
  __syncthreads();
  for (int r = threadIdx.x; r < RP; r += 256) {
    float2 s = wst[0][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) s = join_stats(s, wst[w][r]);
    a.stats[((int64_t)blockIdx.x * a.groups + blockIdx.y) * RP + r] = s;
  }
}

template <int RT>
__global__ __launch_bounds__(256) void few_grad_kernel(const FewArgs a) {
  __shared__ FewTargets T;
  constexpr int RP = RT * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int64_t jl = (int64_t)blockIdx.x * 64 + wave * 16 + 4 * g;
  const int r0 = blockIdx.y * RP;
  few_collect<RP>(a, r0, T);
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = r0 + t * 16 + l15;
    const bool live = r < a.rows && a.flag[r] != 0.f;
    const float gt = live ? a.grad[r * a.grad_stride] * a.temperature : 0.f;
    const float2 st = live ? a.stat[r] : make_float2(0.f, 1.f);
    const float inv = 1.f / st.y;
    float p[4] = {0.f, 0.f, 0.f, 0.f};
    if (live)
      few_targets(a, T, r0, t * 16 + l15, jl, [&](int k, int d) {
        const float q = a.kd ? a.p[(int64_t)r * a.slots + k] : 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] += d == i ? q : 0.f;
      });
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t at = blockIdx.y * a.group_dS + (jl + i) * RP + t * 16 + l15;
      a.dS[at] = live ? gt * fmaf(__builtin_amdgcn_exp2f(a.y[at] - st.x), inv, -p[i]) : 0.f;
    }
  }
}

// one row a workgroup: wave 0 the teacher's softmax, all the join of the statistics
__global__ __launch_bounds__(256) void few_loss_kernel(const FewArgs a, int64_t tiles, int RP) {
  __shared__ float2 part[4];
  const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float2 s = make_float2(-INFINITY, 0.f);
  for (int64_t t = threadIdx.x; t < tiles; t += 256) s = join_stats(s, a.stats[t * a.groups * RP + r]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s = join_stats(s, make_float2(__shfl_xor(s.x, o, 64), __shfl_xor(s.y, o, 64)));
  if (lane == 0) part[wave] = s;
  __syncthreads();
  if (wave) return;
  s = part[0];
  for (int w = 1; w < 4; ++w) s = join_stats(s, part[w]);
  const float ls = s.x == -INFINITY ? NAN : 0.5f * __builtin_amdgcn_logf(s.y);      // (halves, base 2; no column left: no number)
  float out = 0.f;
  bool live, bad = false;
  if (a.kd) {
    float plogp;
    live = teacher_row(a.index, a.wide, a.ld_index, a.teacher, a.ld_teacher, r, a.slots, a.inv_t, a.p, plogp);
    float cross = 0.f, mass = 0.f;
    for (int k = lane; k < a.slots; k += 64) {
      const int64_t id = load_index(a.index, r * a.ld_index + k, a.wide);
      const float q = a.p[(int64_t)r * a.slots + k];
      if (id < 0) continue;
      bad |= id >= a.vocab;
      if (id < a.vocab && !(q == 0.f)) { cross += q * (0.5f * s.x - a.zt[(int64_t)r * a.slots + k]); mass += q; }
    }
    cross = wave_sum(cross);
    mass = wave_sum(mass);
    bad = __any(bad);
    out = a.temperature * a.temperature * (plogp + natural(fmaf(mass, ls, cross)));
  } else {
    const int64_t y = load_index(a.index, r * a.ld_index, a.wide);
    live = y != a.ignore;
    bad = y < 0 || y >= a.vocab;                        // a label outside the vocabulary spoils its row
    if (!bad) out = natural((0.5f * s.x - a.zt[r]) + ls);
  }
  if (lane == 0) {
    a.loss[r] = !live ? 0.f : bad ? NAN : out;
    a.stat[r] = make_float2(s.x, bad ? NAN : s.y);
    a.flag[r] = live ? 1.f : 0.f;
  }
}

constexpr int FEW_J = 2;           // tiles of 16 vocabulary rows a wave of dW
template <int DT, int RT, bool VEC>
__global__ __launch_bounds__(256) void few_products_kernel(const FewArgs a, int h_blocks, int k_blocks) {
  constexpr int RP = RT * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  // Lane l of a first operand loads 4 columns from 4 perm on, one matrix instruction each; the result's rows 4 g + i are then the columns
  // 16 i + 4 g + e: a store of 4 columns is 64 contiguous bytes a row over the wave.
  const int perm = 4 * (l15 & 3) + (l15 >> 2);
  if ((int)blockIdx.x < h_blocks) {
    // dh: 256 columns a workgroup, 64 a wave; lane l ends with row 16 t + l15, columns k0 + 16 i + 4 g + e
    const int range = blockIdx.x % a.ranges, q = blockIdx.x / a.ranges, group = q / k_blocks, k0 = q % k_blocks * 256 + wave * 64;
    const float* dS = a.dS + group * a.group_dS;
    const int64_t j0 = (int64_t)range * a.range, j1 = j0 + a.range < a.vocab ? j0 + a.range : a.vocab;
    if (k0 >= a.K) return;
    f32x4_t acc[4][RT];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[e][t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    auto product = [&](auto full) {
      constexpr bool FULL = decltype(full)::value;
      constexpr int U = 8;
      for (int64_t jb = j0; jb < j1; jb += 4 * U) {
        few_f4 w[U];
        float s[U][RT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t j = jb + 4 * u + g, jj = j < j1 ? j : j1 - 1;
          w[u] = few_load4<DT, VEC, FULL>(a.weight, jj * a.ldw, k0 + 4 * perm, a.K);
#pragma unroll
          for (int t = 0; t < RT; ++t) s[u][t] = dS[jj * RP + t * 16 + l15];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            const float v = jb + 4 * u + g < j1 ? s[u][t] : 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[u][e], v, acc[e][t], 0, 0, 0);
          }
      }
    };
    if (k0 + 64 <= a.K) product(std::true_type{});      // (the same for the wave)
    else product(std::false_type{});
    const int64_t Kq = (a.K + 3) / 4 * 4;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k0 + 16 * i + 4 * g;
        if (k < a.K)
          *reinterpret_cast<float4*>(a.part + (((int64_t)range * a.groups + group) * RP + t * 16 + l15) * Kq + k) =
              make_float4(acc[0][t][i], acc[1][t][i], acc[2][t][i], acc[3][t][i]);
      }
    return;
  }
  // dW: 16 J vocabulary rows a workgroup, every fourth run of 64 columns a wave; lane l ends with rows jb + 16 u + l15, columns
  // k0 + 16 i + 4 g + e.  The first group's dS (few rows: all there is) stays in registers for all runs.  dh and dW of 5 x
  // 131072 x 2048 bf16: 305 us (dh 129 at 4.2 TB/s); loaded at each run, J = 1: 350; J = 4: 320, and 57 : 36 at 128 x 2216 x 512.
  constexpr int J = FEW_J;
  const int64_t jb = ((int64_t)blockIdx.x - h_blocks) * (16 * J) + l15;      // (dS has rows up to a multiple of 64)
  if (a.db && wave < J) {
    const int64_t j = jb + 16 * wave;
    float sum = 0.f;
    for (int group = 0; group < a.groups; ++group)
#pragma unroll
      for (int q = 0; q < 4 * RT; ++q) sum += a.dS[group * a.group_dS + j * RP + 4 * q + g];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (g == 0 && j < a.vocab) store_as(a.db, j, a.bias_dtype, sum);
  }
  if (!a.dW) return;
  float s0[J][4 * RT];
  int64_t at0[4 * RT];                // -1: a row that does not count
  auto load_group = [&](int group, float (&s)[J][4 * RT], int64_t (&at)[4 * RT]) {
#pragma unroll
    for (int q = 0; q < 4 * RT; ++q) {
      const int r = group * RP + 4 * q + g;
      at[q] = r < a.rows && a.flag[r] != 0.f ? r * a.ldh : -1;
#pragma unroll
      for (int u = 0; u < J; ++u) s[u][q] = a.dS[group * a.group_dS + (jb + 16 * u) * RP + 4 * q + g];
    }
  };
  load_group(0, s0, at0);
  for (int k0 = wave * 64; k0 < a.K; k0 += 256) {
    f32x4_t acc[J][4];
#pragma unroll
    for (int u = 0; u < J; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[u][e] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    auto product = [&](auto full) {
      constexpr bool FULL = decltype(full)::value;
      auto add = [&](const float (&s)[J][4 * RT], const int64_t (&at)[4 * RT]) {
        few_f4 h[4 * RT];
#pragma unroll
        for (int q = 0; q < 4 * RT; ++q) h[q] = few_load4<DT, VEC, FULL>(a.hidden, at[q] < 0 ? 0 : at[q], k0 + 4 * perm, a.K);
#pragma unroll
        for (int q = 0; q < 4 * RT; ++q) {
          if (at[q] < 0) h[q] = (few_f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int u = 0; u < J; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[u][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(h[q][e], s[u][q], acc[u][e], 0, 0, 0);
        }
      };
      add(s0, at0);
      for (int group = 1; group < a.groups; ++group) {
        float s[J][4 * RT];
        int64_t at[4 * RT];
        load_group(group, s, at);
        add(s, at);
      }
    };
    if (k0 + 64 <= a.K) product(std::true_type{});
    else product(std::false_type{});
#pragma unroll
    for (int u = 0; u < J; ++u) {
      const int64_t j = jb + 16 * u;
      if (j >= a.vocab) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k0 + 16 * i + 4 * g;
        const float f[4] = {acc[u][0][i], acc[u][1][i], acc[u][2][i], acc[u][3][i]};
        if (k + 4 <= a.K) {                     // (rows of any length: on their elements' boundaries)
          if constexpr (DT == F32) {
            *reinterpret_cast<few_f4_any*>(reinterpret_cast<float*>(a.dW) + j * a.K + k) = (few_f4_any){f[0], f[1], f[2], f[3]};
          } else {
            const u16x4_t x = to_16x4<DT == F16>(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<few_u4_any*>(reinterpret_cast<unsigned short*>(a.dW) + j * a.K + k) = (few_u4_any){x[0], x[1], x[2], x[3]};
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k + e < a.K) store_as(a.dW, j * a.K + k + e, DT, f[e]);
        }
      }
    }
  }
}

// dh = the ranges in order: 16 runs of 4 columns of one row a workgroup, 16 threads a run, each every 16th range
__global__ __launch_bounds__(256) void few_hidden_kernel(const FewArgs a, int RP) {
  __shared__ float4 sums[16][17];
  const int t = threadIdx.x & 15, sp = threadIdx.x >> 4, r = blockIdx.x, k = blockIdx.y * 64 + t * 4;
  const int64_t Kq = (a.K + 3) / 4 * 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (k < a.K) {
#pragma unroll 4
    for (int s = sp; s < a.ranges; s += 16) {
      const float4 x = *reinterpret_cast<const float4*>(a.part + ((int64_t)s * a.groups * RP + r) * Kq + k);
      v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    }
  }
  sums[sp][t] = v;
  __syncthreads();
  if (sp || k >= a.K) return;
  for (int s = 1; s < 16; ++s) { const float4 x = sums[s][t]; v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w; }
  const float f[4] = {v.x, v.y, v.z, v.w};
  for (int e = 0; e < 4; ++e)
    if (k + e < a.K) store_as(a.dh, (int64_t)r * a.K + k + e, a.dtype, f[e]);
}

}  // namespace
