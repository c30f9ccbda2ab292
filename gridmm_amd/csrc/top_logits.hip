// gridmm_top_logits: of every row of logits the k largest, their ids and the row's log-sum-exp -- what a teacher hands to
// gridmm_vocab_loss_fwd's distillation.  Order: value descending, id ascending among equal values (-0 equals +0), NaN above
// everything.
//
// Each value becomes an entry: a key, unsigned and of the same order, above the complement of its id.  Entries are distinct, so "the k
// largest" is one set whatever order things happen in.  A workgroup reads its part of a row ONCE, 16 bytes a lane and 4 loads ahead.
// The k-th largest of the first 2048 vectors' maxima is a floor of the k-th largest value (k values reach it); only values above it
// become entries in LDS -- about k + k ln(V / 16384) of a row in random order.  Where they outgrow the buffer (a rising row) they are
// cut down to k, and at the end: a radix selection over 11-bit digits, entries in registers, that stops as soon as a digit's bin is
// taken whole.  The same pass carries the running maximum and sum of the log-sum-exp.  With few rows a row is cut into segments,
// whose survivors a second kernel joins.  Bound by the read of the logits and, at 16 bits, nearly as much by the ~8 vector
// instructions a value needs: 4096 x 131072 bf16, k = 128 300 us (3.6 TB/s), 384 x 30522 fp32, k = 32 20.5 us, one row of 131071 20 us (9 the
// scan of its 32 segments, 11 their join).
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace {

constexpr int BINS = 2048, DIGIT = 11;
// With T threads a workgroup:
template <int T>
struct Size {
  static constexpr int CUT = 4 * T;      // more entries than this: cut down to k
  static constexpr int BUF = 2 * CUT;    // what does not fit is taken 4 values a thread at a time
  static constexpr int PER = BUF / T;    // entries a thread holds during a selection
  static constexpr int OWN = BINS / T;   // bins a thread owns
};
constexpr int MAX_K = 1024;
constexpr int GROUP = 4;               // chunks (of T vectors) read and looked at together
enum { F32 = 0, BF16 = 1, F16 = 2 };
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f, HUGE_F = 3.4028234664e38f;
typedef unsigned long long u64;

// a value's key: unsigned, of the same order, -0 equal to +0, NaN the largest, never 0 (16-bit types: 16 bits)
template <int DT>
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
  if constexpr (DT == F16) {
    const unsigned h = __builtin_bit_cast(unsigned short, (_Float16)x == (_Float16)0.f ? (_Float16)0.f : (_Float16)x);
    return x != x ? 0xffffu : h ^ ((h >> 15) ? 0xffffu : 0x8000u);
  }
  const unsigned key = x != x ? 0xffffffffu : u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return DT == BF16 ? key >> 16 : key;
}
// a value that no value of a key below `key` exceeds; +inf for the keys of NaN
template <int DT>
__device__ __forceinline__ float key_floor(unsigned key) {
  float x;
  if constexpr (DT == F16) {
    const unsigned short h = (unsigned short)(key ^ ((key >> 15) ? 0x8000u : 0xffffu));
    x = (float)__builtin_bit_cast(_Float16, h);
  } else {
    const unsigned full = DT == BF16 ? key << 16 : key;
    x = __uint_as_float(full ^ ((full >> 31) ? 0x80000000u : 0xffffffffu));
  }
  if (x != x) x = key >> (DT == F32 ? 31 : 15) ? INFINITY : -INFINITY;
  return x;
}
// inclusive sum over the wave's lanes, in lane order
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);      // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);      // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);      // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);      // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // row_bcast:15 into rows 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);      // row_bcast:31 into rows 2, 3
  return v;
}

template <int T>
struct Shared {
  u64 buf[Size<T>::BUF];
  unsigned hist[BINS];
  unsigned wsum[T / 64];
  unsigned n, bin, left, size, added[3];
};

// One digit of a radix selection: `count(add)` calls add(bin) for every entry that matches what is known; of the bins counted from the
// largest down the one that holds the left-th entry is returned, and `left` becomes its place in that bin.
template <int T, class Count>
__device__ __forceinline__ unsigned select_digit(Shared<T>& sh, unsigned& left, bool& whole, Count count) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int OWN = Size<T>::OWN;
#pragma unroll
  for (int b = 0; b < OWN; b += 4) *reinterpret_cast<uint4*>(&sh.hist[tid * OWN + b]) = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  count([&](unsigned bin) { atomicAdd(&sh.hist[bin], 1u); });
  __syncthreads();
  // thread t owns the bins BINS - OWN t - 1 .. BINS - OWN (t + 1), in that order
  unsigned c[OWN], own = 0;
#pragma unroll
  for (int b = 0; b < OWN; b += 4) {
    const uint4 c4 = *reinterpret_cast<const uint4*>(&sh.hist[BINS - 4 - b - tid * OWN]);
    c[b] = c4.w; c[b + 1] = c4.z; c[b + 2] = c4.y; c[b + 3] = c4.x;
    own += c4.w + c4.z + c4.y + c4.x;
  }
  const unsigned incl = wave_scan(own);
  if (lane == 63) sh.wsum[wave] = incl;
  __syncthreads();
  unsigned before = incl - own;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) before += w < wave ? sh.wsum[w] : 0u;
#pragma unroll
  for (int b = 0; b < OWN; ++b) {
    if (before < left && before + c[b] >= left) {
      sh.bin = BINS - 1 - (tid * OWN + b);
      sh.left = left - before;
      sh.size = c[b];
    }
    before += c[b];
  }
  __syncthreads();
  left = sh.left;
  whole = sh.size == left;
  return sh.bin;
}

// Of the n entries (of `bits` bits) in sh.buf keeps the k largest, in sh.buf[0, k) in any order, and sets sh.n = k; n > k.  Returns a
// floor of what is kept: entries below it are not.  Called by all threads with the same n; entries of 0 are "nothing" and lose to
// everything.
template <int T>
__device__ u64 keep_largest(Shared<T>& sh, int n, int k, int bits) {
  constexpr int PER = Size<T>::PER;
  const int tid = threadIdx.x, lane = tid & 63;
  u64 e[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * T + tid;
    e[i] = at < n ? sh.buf[at] : 0;
  }
  u64 prefix = 0;                   // what is known of the k-th largest: its bits from `low` up
  int low = bits;
  unsigned left = k;
  bool whole = false;
  do {
    const int width = min(DIGIT, low), at = low - width;
    const unsigned bin = select_digit(sh, left, whole, [&](auto add) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i * T < n && i * T + tid < n && (e[i] >> low) == prefix) add((unsigned)(e[i] >> at) & ((1u << width) - 1));
    });
    prefix = (prefix << width) | bin;
    low = at;
  } while (!whole && low > 0);
  // everything from here on is kept, k entries; or all that is something, fewer than k
  const bool few = prefix == 0 && low == 0;
  const u64 least = few ? 1 : prefix << low;
  if (tid == 0) sh.n = 0;
  __syncthreads();
  unsigned mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) mine += i * T < n && e[i] >= least;
  const unsigned incl = wave_scan(mine);
  unsigned at = 0;
  if (lane == 63) at = atomicAdd(&sh.n, incl);
  at = __builtin_amdgcn_readlane(at, 63) + incl - mine;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (i * T < n && e[i] >= least) sh.buf[at++] = e[i];
  __syncthreads();
  if (few) {
    for (int i = sh.n + tid; i < k; i += T) sh.buf[i] = 0;
    __syncthreads();
    if (tid == 0) sh.n = k;
    __syncthreads();
    return 0;
  }
  return least;
}

// The k largest of the n >= k entries of sh.buf, sorted, as values and ids: each entry's place is the number of larger ones.  n is at
// most RANK_MOST or k.
constexpr int RANK_MOST = 512;
template <int DT, int T>
__device__ void write_sorted(Shared<T>& sh, int n, int k, int id_bits, const void* logits, int64_t base, void* values, int64_t* ids,
                             int64_t at) {
  for (int i = threadIdx.x; i < n; i += T) sh.hist[i] = 0;
  __syncthreads();
  const int nr = (n + 63) / 64 * 64, parts = max(1, T / nr), len = (n + parts - 1) / parts;      // several threads an entry where n is small
  for (int w = threadIdx.x; w < nr * parts; w += T) {
    const int i = w % nr, j0 = w / nr * len, j1 = min(n, j0 + len);
    if (i >= n) continue;
    const u64 mine = sh.buf[i];
    unsigned larger = 0;
#pragma unroll 8
    for (int j = j0; j < j1; ++j) larger += sh.buf[j] > mine;
    if (larger) atomicAdd(&sh.hist[i], larger);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += T) {
    const int place = sh.hist[i];
    if (place >= k) continue;
    const int64_t id = (int64_t)(~sh.buf[i] & ((1ull << id_bits) - 1)), to = at + place;
    ids[to] = id;
    if constexpr (DT == F32) reinterpret_cast<float*>(values)[to] = reinterpret_cast<const float*>(logits)[base + id];
    else reinterpret_cast<unsigned short*>(values)[to] = reinterpret_cast<const unsigned short*>(logits)[base + id];
  }
}

__device__ __forceinline__ float2 join_sums(float2 a, float2 b) {       // (reference, sum of exp(x - reference)), the reference finite
  const float m = fmaxf(a.x, b.x);
  return make_float2(m, a.y * __builtin_amdgcn_exp2f((a.x - m) * LOG2E) + b.y * __builtin_amdgcn_exp2f((b.x - m) * LOG2E));
}

template <int DT, int T>
__global__ __launch_bounds__(T, 4) void top_scan_kernel(const void* __restrict__ logits, int64_t ld, int V, int k, int id_bits, int segs, int cap,
                                                        u64* __restrict__ kept, float2* __restrict__ sums, void* __restrict__ values,
                                                        int64_t* __restrict__ ids, float* __restrict__ lse) {
  constexpr int E = DT == F32 ? 4 : 8;          // values in 16 bytes
  constexpr int CUT = Size<T>::CUT, BUF = Size<T>::BUF;
  __shared__ Shared<T> sh;
  __shared__ float2 wst[T / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x / segs, seg = blockIdx.x % segs, base = r * ld;
  // vectors of E values counted from the 16-byte boundary at or in front of the row's first value
  const uintptr_t row = (uintptr_t)logits + (uintptr_t)base * (16 / E);
  const int lead = (int)(row & 15) / (16 / E);
  const char* origin = (const char*)(row & ~(uintptr_t)15);
  const int64_t vecs = ((int64_t)lead + V + E - 1) / E, per = (vecs + segs - 1) / segs;
  const int64_t v0 = seg * per, v1 = min(vecs, v0 + per);
  typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

  auto load = [&](int64_t v) -> u32x4_t {
    u32x4_t q = {0u, 0u, 0u, 0u};
    if (v >= v1) return q;
    const int64_t id = v * E - lead;
    if (id >= 0 && id + E <= V) {
      q = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(origin + v * 16));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (id + e >= 0 && id + e < V) {
          if constexpr (DT == F32) q[e] = reinterpret_cast<const unsigned*>(origin + v * 16)[e];
          else q[e / 2] |= (unsigned)reinterpret_cast<const unsigned short*>(origin + v * 16)[e] << (16 * (e & 1));
        }
    }
    return q;
  };
  auto value = [&](const u32x4_t& q, int e) -> float {
    if constexpr (DT == F32) return __uint_as_float(q[e]);
    else if constexpr (DT == BF16) return __uint_as_float((e & 1) ? q[e / 2] & 0xffff0000u : q[e / 2] << 16);
    else return (float)__builtin_bit_cast(_Float16, (unsigned short)(q[e / 2] >> (16 * (e & 1))));
  };

  const int bits = id_bits + (DT == F32 ? 32 : 16);
  auto entry = [&](float x, int64_t id) { return ((u64)order_key<DT>(x) << id_bits) | (~(u64)id & ((1ull << id_bits) - 1)); };
  auto valid = [&](int64_t v) -> unsigned {      // bit e: value e of vector v is the row's and the segment's
    if (v >= v1) return 0;
    const int64_t id = v * E - lead;
    unsigned bits = (1u << E) - 1;
    if (id + E > V) bits >>= (int)(id + E - V);
    if (id < 0) bits &= ~0u << (int)-id;
    return bits;
  };
  float m = -HUGE_F, s = 0.f;                 // reference (finite) and sum of exponentials
  // the values of one vector (-inf where there is none), their largest; into the running sums
  auto values_of = [&](const u32x4_t& q, unsigned have, float (&x)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = value(q, e);
    if (__all(have == (1u << E) - 1)) return;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = have >> e & 1 ? x[e] : -INFINITY;
  };
  auto entering = [&](const float (&x)[E], unsigned have, float least) -> unsigned {
    unsigned in = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) in |= (unsigned)!(x[e] <= least) << e;
    return in & have;
  };
  auto add_to_sums = [&](const float (&x)[E]) -> float {
    float top = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, x[e]);
    const float ref = fmaxf(m, fminf(top, HUGE_F));
    float t = 0.f;
    // One instruction less with the reference's product rounded: 2^-24 of the reference on the log-sum-exp, half its own step.  Only for
    // references up to 2^16: of 1e10, a mask's or a value's, that rounding is an exponent of its own, and the sum infinite
    if (__all(fabsf(ref) < 65536.f)) {
      const float r2 = ref * LOG2E;
#pragma unroll
      for (int e = 0; e < E; ++e) t += __builtin_amdgcn_exp2f(fmaf(x[e], LOG2E, -r2));
      s = fmaf(s, __builtin_amdgcn_exp2f(fmaf(m, LOG2E, -r2)), t);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) t += __builtin_amdgcn_exp2f((x[e] - ref) * LOG2E);
      s = fmaf(s, __builtin_amdgcn_exp2f((m - ref) * LOG2E), t);
    }
    m = ref;
    return top;
  };

  auto inside = [&](int64_t c) { return c * E >= lead && c + GROUP * T <= v1 && (c + GROUP * T) * E - lead <= V; };
  auto fetch = [&](int64_t c, u32x4_t (&q)[GROUP]) {
    if (inside(c)) {
#pragma unroll
      for (int i = 0; i < GROUP; ++i) q[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(origin) + c + i * T + tid);
    } else {
#pragma unroll
      for (int i = 0; i < GROUP; ++i) q[i] = load(c + i * T + tid);
    }
  };
  u32x4_t q[GROUP], next[GROUP];
  fetch(v0, q);
  if (tid < 3) sh.added[tid] = 0;
  // a value enters if it is not <= least (so a NaN always does; a least of NaN lets everything in)
  float least = NAN;
  int n = 0, turn = 0;
  for (int64_t c = v0; c < v1; c += GROUP * T) {
    const bool whole = inside(c);
    if (c + GROUP * T < v1) fetch(c + GROUP * T, next);
    float floor_after = least;
    float x[E];
    unsigned in = 0;                          // bit i E + e: value e of chunk i enters
    if (c == v0) {
      // a floor from the vectors' maxima: the k-th largest of them to 22 bits; k values at least reach it
      unsigned key[GROUP];
#pragma unroll
      for (int i = 0; i < GROUP; ++i) {
        key[i] = 0;
        if (c + i * T >= v1) continue;
        const unsigned have = whole ? (1u << E) - 1 : valid(c + i * T + tid);
        values_of(q[i], have, x);
        const float top = add_to_sums(x);
        key[i] = have ? order_key<DT>(top) : 0u;
      }
      constexpr int KEY = DT == F32 ? 32 : 16;
      unsigned left = k, prefix = 0;
      bool all = false;
      int low = KEY;
#pragma unroll 1
      for (int pass = 0; pass < 2; ++pass) {
        const int width = min(DIGIT, low), at = low - width;
        const unsigned bin = select_digit(sh, left, all, [&](auto add) {
#pragma unroll
          for (int i = 0; i < GROUP; ++i)
            if (pass == 0 || (key[i] >> low) == prefix) add((key[i] >> at) & ((1u << width) - 1));
        });
        prefix = (prefix << width) | bin;
        low = at;
      }
      prefix <<= low;
      if (prefix) {
        floor_after = key_floor<DT>(prefix);
        // the first values may equal it: let in what is above the next lower number
        const unsigned u = __float_as_uint(floor_after);
        least = floor_after == -INFINITY ? NAN : floor_after == 0.f ? -1.4e-45f : __uint_as_float(u + ((u >> 31) ? 1 : -1));
      }
#pragma unroll
      for (int i = 0; i < GROUP; ++i) {
        asm volatile("" : "+v"(q[i]));         // (unpacked again rather than kept unpacked)
        if (c + i * T >= v1) continue;
        const unsigned have = whole ? (1u << E) - 1 : valid(c + i * T + tid);
        values_of(q[i], have, x);
        in |= entering(x, have, least) << (i * E);
      }
    } else {
#pragma unroll
      for (int i = 0; i < GROUP; ++i) {
        if (c + i * T >= v1) continue;
        const unsigned have = whole ? (1u << E) - 1 : valid(c + i * T + tid);
        values_of(q[i], have, x);
        const float top = add_to_sums(x);
        if (__any(!(top <= least) || s != s)) in |= entering(x, have, least) << (i * E);
      }
    }
    // places for all of them; if they do not fit, in small parts with cuts between
    auto put = [&](unsigned bitsin, unsigned at) {
      while (bitsin) {
        const int b = __builtin_ctz(bitsin);
        bitsin &= bitsin - 1;
        const int w = DT == F32 ? b : b >> 1;
        unsigned word = q[0][0];
#pragma unroll
        for (int j = 1; j < 4 * GROUP; ++j) word = w == j ? q[j / 4][j % 4] : word;
        float val;
        if constexpr (DT == F32) val = __uint_as_float(word);
        else if constexpr (DT == BF16) val = __uint_as_float((b & 1) ? word & 0xffff0000u : word << 16);
        else val = (float)__builtin_bit_cast(_Float16, (unsigned short)(word >> (16 * (b & 1))));
        sh.buf[at++] = entry(val, (c + (b / E) * T + tid) * E - lead + b % E);
      }
    };
    auto places = [&](unsigned bitsin) -> unsigned {
      unsigned at = 0;
      if (__any(bitsin != 0)) {
        const unsigned mine = __popc(bitsin), incl = wave_scan(mine);
        if (lane == 63) at = atomicAdd(&sh.added[turn], incl);
        at = __builtin_amdgcn_readlane(at, 63) + incl - mine;
      }
      return at;
    };
    // (three counters in turn: one is added to, one is being read, one has been read by everyone and is cleared)
    auto settle = [&]() -> unsigned {
      __syncthreads();
      const unsigned added = sh.added[turn];
      turn = turn == 2 ? 0 : turn + 1;
      if (tid == 0) sh.added[turn == 2 ? 0 : turn + 1] = 0;
      return added;
    };
    unsigned at = places(in);
    unsigned added = settle();
    if (n + added <= BUF) {
      put(in, n + at);
      n += added;
    } else {
#pragma unroll 1
      for (int i = 0; i < GROUP * E; i += 4) {
        const unsigned part = in & (15u << i);
        at = places(part);
        added = settle();
        put(part, n + at);                    // n <= CUT, and these are at most BUF - CUT
        n += added;
        if (n > CUT) {
          __syncthreads();
          const u64 kept_floor = keep_largest(sh, n, k, bits);
          n = k;
          // what came later with the same value loses by its id; a bound that is higher than the floor so far
          const float f = kept_floor ? key_floor<DT>((unsigned)(kept_floor >> id_bits)) : -INFINITY;
          if (kept_floor && !(f < floor_after)) floor_after = f;
        }
      }
    }
    least = floor_after;
    if (n > CUT) {
      __syncthreads();
      const u64 kept_floor = keep_largest(sh, n, k, bits);
      n = k;
      const float f = kept_floor ? key_floor<DT>((unsigned)(kept_floor >> id_bits)) : -INFINITY;
      if (kept_floor && !(f < least)) least = f;
    }
#pragma unroll
    for (int i = 0; i < GROUP; ++i) q[i] = next[i];
  }
  __syncthreads();
  const int room = segs == 1 ? (k > RANK_MOST ? k : RANK_MOST) : cap;
  if (n > room) {
    keep_largest(sh, n, k, bits);
    n = k;
  }

  // the row's sums
  float2 a = make_float2(m, s);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = join_sums(a, make_float2(__shfl_xor(a.x, o, 64), __shfl_xor(a.y, o, 64)));
  if (lane == 0) wst[wave] = a;
  __syncthreads();
  for (int w = 0; w < T / 64; ++w) a = w ? join_sums(a, wst[w]) : wst[0];
  if (segs == 1) {
    if (tid == 0) lse[r] = fmaf(__builtin_amdgcn_logf(a.y), LN2, a.x);
    write_sorted<DT, T>(sh, n, k, id_bits, logits, base, values, ids, r * k);
  } else {
    if (tid == 0) sums[blockIdx.x] = a;
    for (int i = tid; i < cap; i += T) kept[(int64_t)blockIdx.x * cap + i] = i < n ? sh.buf[i] : 0;
  }
}

template <int DT, int T>
__global__ __launch_bounds__(T) void top_join_kernel(const void* __restrict__ logits, int64_t ld, int k, int id_bits, int segs, int cap,
                                                     const u64* __restrict__ kept, const float2* __restrict__ sums,
                                                     void* __restrict__ values, int64_t* __restrict__ ids, float* __restrict__ lse) {
  __shared__ Shared<T> sh;
  const int64_t r = blockIdx.x;
  int n = segs * cap;
  for (int i = threadIdx.x; i < n; i += T) sh.buf[i] = kept[r * n + i];
  if (threadIdx.x == 0) {
    float2 a = sums[r * segs];
    for (int w = 1; w < segs; ++w) a = join_sums(a, sums[r * segs + w]);
    lse[r] = fmaf(__builtin_amdgcn_logf(a.y), LN2, a.x);
  }
  __syncthreads();
  if (n > RANK_MOST && n > k) {
    keep_largest(sh, n, k, id_bits + (DT == F32 ? 32 : 16));
    n = k;
  }
  write_sorted<DT, T>(sh, n, k, id_bits, logits, r * ld, values, ids, r * k);
}

// Threads a workgroup: 256 where the rows fill the chip four times over (four rows a CU in different phases: 302 against 326 us at 4096 x
// 131072 bf16, 38 : 73 at 4096 x 2000), else 512 (20.6 : 33.7 at 384 x 30522 fp32); 512 also where k is more than a quarter of
// the vectors that the floor comes from.
int threads(int rows, int k) { return rows >= 1024 && k <= 256 ? 256 : 512; }
// segments a row: a workgroup a CU (one segment and no join at 384 rows: 20.6 us, two: 27.5), none shorter than 4096 values, their
// survivors no more than the joining workgroup's buffer
constexpr int JOIN_T = 512;
int segments(int rows, int vocab, int k) {
  int64_t s = (256 + rows - 1) / rows;
  s = std::min<int64_t>(s, (vocab + 4095) / 4096);
  s = std::min<int64_t>(s, Size<JOIN_T>::BUF / k);
  return s < 1 ? 1 : (int)s;
}
// entries a segment may hand over: what it holds is cut down to k only if it is more than this
int handed(int segs, int k) { return std::min(Size<JOIN_T>::BUF / segs, 4 * k); }

}  // namespace

extern "C" size_t gridmm_top_logits_workspace(int rows, int vocab, int k) {
  if (rows < 1 || vocab < 1 || k < 1 || k > MAX_K) return 0;
  const int s = segments(rows, vocab, k);
  return s == 1 ? 0 : (size_t)rows * s * (handed(s, k) * sizeof(u64) + sizeof(float2));
}

extern "C" int gridmm_top_logits(const void* logits, int64_t ld, int dtype, int rows, int vocab, int k, void* values, int64_t* ids,
                                 float* lse, void* workspace, size_t workspace_bytes, gridmm_stream_t stream) {
  if (rows < 0 || rows > (1 << 22) || vocab < 1 || k < 1 || k > vocab || k > MAX_K || ld < vocab || dtype < 0 || dtype > 2)
    return GRIDMM_EINVAL;
  if (rows == 0) return GRIDMM_OK;
  const size_t need = gridmm_top_logits_workspace(rows, vocab, k);
  if (!logits || !values || !ids || !lse || workspace_bytes < need || (need && (!workspace || ((uintptr_t)workspace & 255))))
    return GRIDMM_EINVAL;
  if ((uintptr_t)logits % (dtype == F32 ? 4 : 2)) return GRIDMM_EINVAL;
  hipStream_t st = as_stream(stream);
  const int segs = segments(rows, vocab, k);
  int id_bits = 1;
  while (id_bits < 32 && (vocab - 1) >> id_bits) ++id_bits;
  u64* kept = (u64*)workspace;
  const int cap = handed(segs, k);
  float2* sums = (float2*)(kept + (size_t)rows * segs * cap);
  auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    auto scan = [&](auto t) {
      constexpr int T = decltype(t)::value;
      GRIDMM_LAUNCH((top_scan_kernel<DT, T>), dim3((unsigned)(rows * segs)), dim3(T), 0, st, logits, ld, vocab, k, id_bits, segs, cap,
                    kept, sums, values, ids, lse);
    };
    if (threads(rows, k) == 256) scan(std::integral_constant<int, 256>{});
    else scan(std::integral_constant<int, 512>{});
    GRIDMM_CHECK_LAUNCH();
    if (segs > 1) {
      GRIDMM_LAUNCH((top_join_kernel<DT, JOIN_T>), dim3(rows), dim3(JOIN_T), 0, st, logits, ld, k, id_bits, segs, cap, kept, sums, values,
                    ids, lse);
      GRIDMM_CHECK_LAUNCH();
    }
    return GRIDMM_OK;
  };
  if (dtype == F32) return run(std::integral_constant<int, F32>{});
  if (dtype == BF16) return run(std::integral_constant<int, BF16>{});
  return run(std::integral_constant<int, F16>{});
}
