// gridmm_top_logits: of every row of logits the k largest, their ids and the row's log-sum-exp -- what a teacher hands to
// gridmm_vocab_loss_fwd's distillation.  Order: value descending, id ascending among equal values (-0 equals +0), NaN above
// everything.  The value is mapped to an unsigned key of the same order; the k-th largest key comes from four rounds of 256
// digit counts, most significant digit first; what lies above it and the lowest ids that equal it are collected and sorted.
#include "common.h"

namespace {

constexpr int TOP_T = 1024;
enum { F32 = 0, BF16 = 1, F16 = 2 };

template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (DT == F32) return reinterpret_cast<const float*>(p)[i];
  const unsigned short u = reinterpret_cast<const unsigned short*>(p)[i];
  if constexpr (DT == BF16) return bf16_bits_to_f32(u);
  return (float)__builtin_bit_cast(_Float16, u);
}
__device__ __forceinline__ unsigned order_key(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// exp(a - b) of a <= b, where both may be the same infinity
__device__ __forceinline__ float exp_below(float a, float b) { return a == b ? 1.f : expf(a - b); }

template <int DT>
__global__ __launch_bounds__(TOP_T) void top_logits_kernel(const void* __restrict__ logits, int64_t ld, int V, int k, int kp,
                                                           void* __restrict__ values, int64_t* __restrict__ ids,
                                                           float* __restrict__ lse) {
  __shared__ unsigned hist[256];
  __shared__ unsigned long long best[1024];
  __shared__ float fm[16], fs[16];
  __shared__ unsigned wcount[16];
  __shared__ unsigned s_prefix, s_left, s_n;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x, base = r * ld;

  // log-sum-exp: running maximum and sum a thread, joined
  float m = -INFINITY, s = 0.f;
  for (int j = tid; j < V; j += TOP_T) {
    const float x = load1<DT>(logits, base + j);
    const float M = fmaxf(m, x);
    if (M > m) { s *= exp_below(m, M); m = M; }
    if (x != x) s = x;
    else if (x != -INFINITY) s += exp_below(x, m);
  }
  const float wm = wave_max(m);
  const float ref = wm == -INFINITY ? 0.f : wm;
  const float wsum = wave_sum(m == -INFINITY && s == 0.f ? 0.f : s * exp_below(m, ref));
  if (lane == 0) { fm[wave] = wm; fs[wave] = wsum; }
  __syncthreads();
  if (tid == 0) {
    float M = -INFINITY, S = 0.f;
    for (int w = 0; w < 16; ++w) M = fmaxf(M, fm[w]);
    const float R = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < 16; ++w) S += fs[w] * exp_below(fm[w] == -INFINITY ? R : fm[w], R);
    lse[r] = R + logf(S);
  }

  // the k-th largest key, digit by digit
  unsigned prefix = 0, left = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += TOP_T) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < V; j += TOP_T) {
      const unsigned key = order_key(load1<DT>(logits, base + j));
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      unsigned n = 0;
      int dig = 255;
      while (dig > 0 && n + hist[dig] < left) n += hist[dig--];
      s_prefix = prefix | ((unsigned)dig << shift);
      s_left = left - n;
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    __syncthreads();
  }
  // `left` of the keys equal to `prefix` belong to the k, the lowest ids of them
  if (tid == 0) s_n = 0;
  __syncthreads();
  unsigned eq_before = 0;
  for (int j0 = 0; j0 < V; j0 += TOP_T) {
    const int j = j0 + tid;
    const unsigned key = j < V ? order_key(load1<DT>(logits, base + j)) : 0u;
    const bool eq = j < V && key == prefix;
    const unsigned long long b = __ballot(eq);
    if (lane == 0) wcount[wave] = __popcll(b);
    __syncthreads();
    unsigned rank = eq_before + __popcll(b & ((1ull << lane) - 1));
    for (int w = 0; w < 16; ++w) {
      if (w < wave) rank += wcount[w];
      eq_before += wcount[w];
    }
    if (j < V && (key > prefix || (eq && rank < left)))
      best[atomicAdd(&s_n, 1u)] = ((unsigned long long)key << 32) | (unsigned)~j;
    __syncthreads();
  }
  for (int i = k + tid; i < kp; i += TOP_T) best[i] = 0;
  __syncthreads();
  // descending by (key, lowest id): bitonic over kp >= k entries
  for (int size = 2; size <= kp; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = tid; i < kp; i += TOP_T) {
        const int o = i ^ step;
        if (o > i) {
          const unsigned long long a = best[i], b = best[o];
          if ((a < b) == ((i & size) == 0)) { best[i] = b; best[o] = a; }
        }
      }
      __syncthreads();
    }
  for (int i = tid; i < k; i += TOP_T) {
    const unsigned j = ~(unsigned)(best[i] & 0xffffffffu);
    ids[r * k + i] = j;
    if (DT == F32) reinterpret_cast<float*>(values)[r * k + i] = reinterpret_cast<const float*>(logits)[base + j];
    else reinterpret_cast<unsigned short*>(values)[r * k + i] = reinterpret_cast<const unsigned short*>(logits)[base + j];
  }
}

}  // namespace

extern "C" size_t gridmm_top_logits_workspace(int rows, int vocab, int k) {
  (void)rows; (void)vocab; (void)k;
  return 0;
}

extern "C" int gridmm_top_logits(const void* logits, int64_t ld, int dtype, int rows, int vocab, int k, void* values, int64_t* ids,
                                 float* lse, void* workspace, size_t workspace_bytes, gridmm_stream_t stream) {
  if (rows < 0 || vocab < 1 || k < 1 || k > vocab || k > 1024 || ld < vocab || dtype < 0 || dtype > 2 ||
      workspace_bytes < gridmm_top_logits_workspace(rows, vocab, k))
    return GRIDMM_EINVAL;
  if (rows == 0) return GRIDMM_OK;
  if (!logits || !values || !ids || !lse) return GRIDMM_EINVAL;
  (void)workspace;
  hipStream_t st = as_stream(stream);
  int kp = 1;
  while (kp < k) kp <<= 1;
  if (dtype == F32) GRIDMM_LAUNCH(top_logits_kernel<F32>, dim3(rows), dim3(TOP_T), 0, st, logits, ld, vocab, k, kp, values, ids, lse);
  else if (dtype == BF16) GRIDMM_LAUNCH(top_logits_kernel<BF16>, dim3(rows), dim3(TOP_T), 0, st, logits, ld, vocab, k, kp, values, ids, lse);
  else GRIDMM_LAUNCH(top_logits_kernel<F16>, dim3(rows), dim3(TOP_T), 0, st, logits, ld, vocab, k, kp, values, ids, lse);
  GRIDMM_CHECK_LAUNCH();
  return GRIDMM_OK;
}
