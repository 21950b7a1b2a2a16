// Class log-probabilities of margin rows, and their gradient: for a row x of margins,
// m = max x and d_j = scale * (x_j - m),
//
//   log_sum = log s,  s = sum_j e^{d_j}          lse     = scale * m + log_sum
//   logp_t  = d_t - log_sum                      entropy = log_sum - (sum_j e^{d_j} d_j) / s
//
// and the k largest margins (the lower index first among equal ones) with their logp.
// Both terms of the entropy have one sign, so no digits cancel between them. s holds the
// maximum's own 1: log_sum, and with it logp and entropy, are right absolutely, to the rounding of
// that sum, and other classes that have less than 2^-24 together do not count. A row whose
// margins are all -inf has m = lse = logp = -inf, log_sum = entropy = 0; a NaN or +inf among
// the margins makes the row's outputs NaN (m is what it is).
//
// The gradient of sum_i (g_i logp_i + e_i entropy_i), with p_j = e^{d_j - log_sum}:
//
//   dx_j = scale * (g (delta_jt - p_j) - e p_j (log p_j + entropy))
//
// It takes m and log_sum rather than lse: lse in 32 bits cannot hold log_sum beside a large
// m (the finite lowest value used as a mask).
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "rw_internal.cuh"
#include "rw_types.cuh"

namespace {

constexpr float kLowest = -1e30f;  // where differences are cut: e^d is 0 there, and 0 * d stays 0
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = INFINITY;

// The larger of two values, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// An order of the margins as whole numbers above 0 (NaN above +inf, -0 equal to +0), and with
// the index below it: larger margins first, lower indices first among equal ones. The
// addition makes -0 into +0 and every NaN into the one with all bits but the sign set.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float margin_of(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
using Key = unsigned long long;
__device__ __forceinline__ Key key_of(uint32_t order, uint32_t index) {
  return (Key)order << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t index_of(Key k) { return 0xffffffffu - (uint32_t)k; }

// A running softmax: the largest margin so far, s = sum e^{scale (x - m)} and
// t = sum e^{scale (x - m)} (x - m). c = scale * log2(e).
struct Sums {
  float m = -kInf, s = 0.0f, t = 0.0f;
};
// Restates the sums relative to a larger maximum (not -inf).
__device__ __forceinline__ void raise(Sums& a, float m, float c) {
  const float d = max_nan(a.m - m, kLowest), f = exp2_fast(d * c);
  a.t = f * (a.t + d * a.s);
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
  const float m = max_nan(a.m, b.m);
  if (m == -kInf) return a;
  raise(a, m, c);
  raise(b, m, c);
  a.s += b.s;
  a.t += b.t;
  return a;
}
__device__ __forceinline__ Sums shuffle_xor(const Sums& a, int o) {
  Sums b;
  b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
  b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
  b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
  return b;
}

// What the outputs of a row need of its sums.
struct RowEnd {
  float base, log_sum;  // base: the maximum, 0 in a row of -inf alone
};
__device__ __forceinline__ RowEnd row_end(const Sums& a) {
  const bool dead = a.m == -kInf;
  return {dead ? 0.0f : a.m, dead ? 0.0f : logf(a.s)};
}
// scale * (x - base), of halves: the difference of two margins may be past f32's range.
__device__ __forceinline__ float scaled_difference(float x, float base, float scale) {
  return (x * 0.5f - base * 0.5f) * scale * 2.0f;
}
// A row's target and its margin, two dependent loads: the target's is issued before the row's
// loads and the margin's after them, so that neither is waited for at the row's end.
__device__ __forceinline__ int64_t target_of(const LogprobsLaunch& a, uint64_t i) {
  if (!a.logp) return -1;
  return a.target_type == RW_I64 ? ((const int64_t*)a.targets)[i] : ((const int32_t*)a.targets)[i];
}
template <typename T>
__device__ __forceinline__ float margin_at(const LogprobsLaunch& a, uint64_t i, int64_t target, bool& in) {
  in = target >= 0 && (uint64_t)target < a.classes;
  return in ? rw_widen(((const T*)a.x)[i * a.ld_x + target]) : 0.0f;
}
__device__ __forceinline__ void write_row(const LogprobsLaunch& a, uint64_t i, const Sums& r, const RowEnd& e,
                                          float target, bool in) {
  if (a.row_max) a.row_max[i] = r.m;
  if (a.log_sum) a.log_sum[i] = e.log_sum;
  if (a.lse) a.lse[i] = a.scale * r.m + e.log_sum;
  if (a.entropy) a.entropy[i] = r.m == -kInf ? 0.0f : e.log_sum - a.scale * __fdividef(r.t, r.s);
  if (a.logp) a.logp[i] = in ? scaled_difference(target, e.base, a.scale) - e.log_sum : 0.0f;
}
__device__ __forceinline__ void write_top(const LogprobsLaunch& a, uint64_t i, uint32_t place, Key k, const RowEnd& e) {
  if (a.top_index) a.top_index[i * a.top_k + place] = index_of(k);
  if (a.top_logp)
    a.top_logp[i * a.top_k + place] = scaled_difference(margin_of((uint32_t)(k >> 32)), e.base, a.scale) - e.log_sum;
}

// =================================================================================
// Few classes: L lanes a row, at most E margins a lane, all in registers.

constexpr int kGroupThreads = 256;
// The places of at most 32 margins: one after another, or from more than kCountPlaces on by
// counting (431527 x 15 f32, top 15: 112 us and 68 us).
constexpr uint32_t kCountPlaces = 6;
// The bound of a warp's row: by warp reductions, one a place, or above kReducePlaces by counting
// (200000 x 100 bf16, top 5: 110 us and 123 us; top 10: 125 us and 128 us; top 20: 163 us and
// 143 us).
constexpr uint32_t kReducePlaces = 12;
// Up to 128 classes: four rows a warp, or with more than kSharedPlaces places a warp a row
// (200000 x 100 bf16, top 5: 80 us and 110 us; top 10: 132 us and 128 us; top 20: 235 us and
// 143 us).
constexpr uint32_t kSharedPlaces = 8;
constexpr int kGroupCand = 128;  // candidates for a row's top places that a warp keeps

template <typename T, int L, int E>
__global__ void __launch_bounds__(kGroupThreads, L < 32 ? 1 : E <= 8 ? 6 : E <= 16 ? 4 : 3) k_logprobs_few(LogprobsLaunch a) {
  __shared__ __align__(16) uint32_t s_cand[L == 32 ? kGroupThreads / 32 : 1][L == 32 ? kGroupCand : 1];
  __shared__ uint32_t s_cand_at[L == 32 ? kGroupThreads / 32 : 1][L == 32 ? kGroupCand : 1];
  const uint32_t lane = threadIdx.x % L, classes = (uint32_t)a.classes;
  const float c = a.scale * kLog2e;
  constexpr uint32_t kRows = kGroupThreads / L;  // rows of a CTA at a time
  for (uint64_t base = (uint64_t)blockIdx.x * kRows; base < a.n; base += (uint64_t)gridDim.x * kRows) {
    const uint64_t i = base + threadIdx.x / L;
    const bool real = i < a.n;
    const T* x = (const T*)a.x + (real ? i : a.n - 1) * a.ld_x;
    // rows that share a warp leave no registers for it (24.6 -> 26.8 us at 1000000 x 7 f32)
    int64_t target = L == 32 && real && lane == 0 ? target_of(a, i) : -1;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      const uint32_t j = lane + e * L;
      v[e] = j < classes ? rw_widen(x[j]) : -kInf;
    }
    bool in_row = false;
    float at_target = 0.0f;
    if (L == 32) at_target = margin_at<T>(a, i, target, in_row);
    Sums r;
#pragma unroll
    for (int e = 0; e < E; e++) r.m = max_nan(r.m, v[e]);
    const float own = r.m;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) r.m = max_nan(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
    if (r.m != -kInf) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float d = max_nan(v[e] - r.m, kLowest), p = exp2_fast(d * c);
        r.s += p;
        r.t += p * d;
      }
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
      r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
      r.t += __shfl_xor_sync(0xffffffffu, r.t, o);
    }
    const RowEnd end = row_end(r);
    if (real && lane == 0) {
      if (L < 32) at_target = margin_at<T>(a, i, target_of(a, i), in_row);
      write_row(a, i, r, end, at_target, in_row);
    }
    if (a.top_k == 0) continue;
    uint32_t order[E];  // 0: no margin, or one that has its place
#pragma unroll
    for (int e = 0; e < E; e++) order[e] = lane + e * L < classes ? order_of(v[e]) : 0;
    if constexpr (L == 32) {
      // The top_k-th largest of the lanes' maxima is a bound: top_k margins at least reach it.
      // Those that do (the bound's own included) are ranked by counting. Too many only if
      // many are equal or a lane holds many of the largest: then place by place, below.
      uint32_t left = order_of(own), bound = 0;
      if (a.top_k <= kReducePlaces) {  // maximum by maximum
        for (uint32_t found = 0;;) {
          bound = __reduce_max_sync(0xffffffffu, left);
          found += __popc(__ballot_sync(0xffffffffu, left == bound));
          if (found >= a.top_k) break;
          if (left == bound) left = 0;
        }
      } else {  // the largest that top_k lanes reach
        uint32_t reach = 0;
#pragma unroll
        for (int o = 0; o < 32; o++) reach += __shfl_sync(0xffffffffu, left, o) >= left;
        bound = __reduce_max_sync(0xffffffffu, reach >= a.top_k ? left : 0u);
      }
      // the candidates' orders and indices, in index order
      uint32_t* cand = s_cand[threadIdx.x / 32];
      uint32_t* cand_at = s_cand_at[threadIdx.x / 32];
      auto collect = [&](uint32_t from) {
        uint32_t count = 0;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < E; e++) {
          const uint32_t hits = __ballot_sync(0xffffffffu, order[e] >= from);
          if (hits == 0) continue;
          const uint32_t at = count + __popc(hits & ((1u << lane) - 1));
          if (order[e] >= from && at < kGroupCand) {
            cand[at] = order[e];
            cand_at[at] = lane + e * 32;
          }
          count += __popc(hits);
        }
        if (lane < 4 && count + lane < kGroupCand) cand[count + lane] = 0;
        __syncwarp();
        return count;
      };
      uint32_t count = collect(bound), ties = 0;
      if (count > kGroupCand && bound != 0xffffffffu) {
        // many equal the bound (a mask): those above it, then the first of the equal ones
        count = collect(bound + 1);
        ties = count < a.top_k ? a.top_k - count : 0;
      }
      if (count <= kGroupCand) {
        for (uint32_t q = lane; q < count; q += 32) {
          // those above it, and the equal ones before it: whole fours by >=, then its own four
          const uint32_t k = cand[q], four = q & ~3u;
          uint32_t place = 0;
          for (uint32_t w = 0; w < count; w += 4) {
            const uint4 o = *(const uint4*)(cand + w);
            const uint32_t than = w < four ? k - 1 : k;  // orders are above 0
            place += (o.x > than) + (o.y > than) + (o.z > than) + (o.w > than);
          }
          for (uint32_t w = four; w < q; w++) place += cand[w] == k;
          if (real && place < a.top_k) write_top(a, i, place, key_of(k, cand_at[q]), end);
        }
        uint32_t place = a.top_k - ties;
#pragma unroll
        for (int e = 0; e < E; e++) {
          if (place >= a.top_k) break;
          const bool in = order[e] == bound;
          const uint32_t hits = __ballot_sync(0xffffffffu, in);
          const uint32_t at = place + __popc(hits & ((1u << lane) - 1));
          if (real && in && at < a.top_k) write_top(a, i, at, key_of(bound, lane + e * 32), end);
          place += __popc(hits);
        }
        continue;
      }
    }
    if constexpr (L > 1 && L * E <= 32) {
      // many places of few margins: every margin counts those before it
      if (a.top_k > kCountPlaces) {
        uint32_t above[E];
#pragma unroll
        for (int e = 0; e < E; e++) above[e] = 0;
#pragma unroll
        for (int o = 0; o < L; o++) {
#pragma unroll
          for (int q = 0; q < E; q++) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, order[q], o);
#pragma unroll
            for (int e = 0; e < E; e++) {
              const bool lower = q < e || (q == e && (lane ^ o) < lane);
              above[e] += other > order[e] || (other == order[e] && lower);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < E; e++)
          if (real && order[e] && above[e] < a.top_k)
            write_top(a, i, above[e], key_of(order[e], lane + e * L), end);
        continue;
      }
    }
    // place by place
    for (uint32_t place = 0; place < a.top_k; place++) {
      uint32_t top = order[0], at = lane;
#pragma unroll
      for (int e = 1; e < E; e++) {
        if (order[e] > top) {
          top = order[e];
          at = lane + e * L;
        }
      }
      Key best = key_of(top, at);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
      at = index_of(best);
#pragma unroll
      for (int e = 0; e < E; e++)
        if (lane + e * L == at) order[e] = 0;
      if (real && lane == 0) write_top(a, i, place, best, end);
    }
  }
}

// =================================================================================
// Many classes: a CTA a row, or a part of one.

// Threads a CTA: 256, or for many rows of at most kShortBytes 64, since barriers and joins cost
// more than the margins of short rows (64 and 256 threads: 48056 x 2824 bf16 128 us and 344 us,
// 8000 x 32000 115 us and 125 us; 6000 x 50000 136 us and 118 us).
constexpr int kRowThreads = 256, kShortThreads = 64;
constexpr uint64_t kShortBytes = 64 << 10;
constexpr int kRowDepth = 4;       // vectors in flight a thread
constexpr uint32_t kGroups = 64;   // groups of threads whose maxima bound the top places
constexpr uint32_t kCand = 1024;   // candidates for the top places that a CTA keeps
constexpr uint32_t kMaxParts = 64;

// Where a row's sums and top keys are left when it is split: [row][part].
struct SplitRow {
  uint32_t parts;
  uint64_t part;  // classes a part
  Sums* sums;
  Key* keys;      // [row][part][top_k], descending
};

// Consecutive margins as 16-byte vectors with a ragged head and tail.
template <typename T>
struct Span {
  static constexpr int kV = 16 / sizeof(T);
  const T* x;
  uint32_t n, head, vecs;
  __device__ __forceinline__ Span(const T* p, uint32_t count) : x(p), n(count) {
    const uint32_t off = (uint32_t)((uintptr_t)p & 15) / sizeof(T);
    head = min(n, off ? kV - off : 0u);
    vecs = (n - head) / kV;
  }
  __device__ __forceinline__ uint32_t ragged() const { return n - vecs * kV; }
  // the position of ragged element r
  __device__ __forceinline__ uint32_t ragged_at(uint32_t r) const { return r < head ? r : vecs * kV + r; }
  __device__ __forceinline__ const T* vec(uint32_t v) const { return x + head + (size_t)v * kV; }
};

// Two f32 values in a 64-bit register: one instruction adds or multiplies both.
using Two = unsigned long long;
__device__ __forceinline__ Two two_of(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(Two v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// Elements 2 q and 2 q + 1 of a pack; CUT: not below low (as bf16 has it).
template <bool CUT, int V>
__device__ __forceinline__ Two pair_of(const Pack<float, V>& p, int q, float low) {
  const float a = p.v[2 * q], b = p.v[2 * q + 1];
  return CUT ? two_of(max_nan(a, low), max_nan(b, low)) : two_of(a, b);
}
template <bool CUT, int V>
__device__ __forceinline__ Two pair_of(const Pack<__nv_bfloat16, V>& p, int q, float low) {
  __nv_bfloat162 w = reinterpret_cast<const __nv_bfloat162*>(p.v)[q];
  if (CUT) w = __hmax2_nan(w, __float2bfloat162_rn(low));
  const uint32_t b = *reinterpret_cast<uint32_t*>(&w);
  return two_of(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
}
template <bool CUT, int V>
__device__ __forceinline__ Two pair_of(const Pack<__half, V>& p, int q, float low) {
  const float2 f = __half22float2(reinterpret_cast<const __half2*>(p.v)[q]);
  return CUT ? two_of(max_nan(f.x, low), max_nan(f.y, low)) : two_of(f.x, f.y);
}

// The largest element of N packs, NaN if one is.
template <int N, int V>
__device__ __forceinline__ float packs_max(const Pack<float, V>* p) {
  float m = p[0].v[0];
#pragma unroll
  for (int k = 1; k < N * V; k++) m = max_nan(m, p[k / V].v[k % V]);
  return m;
}
template <typename T2, int N, typename T, int V>
__device__ __forceinline__ T2 pairs_max(const Pack<T, V>* p) {
  T2 m = reinterpret_cast<const T2*>(p[0].v)[0];
#pragma unroll
  for (int k = 1; k < N * V / 2; k++) m = __hmax2_nan(m, reinterpret_cast<const T2*>(p[k / (V / 2)].v)[k % (V / 2)]);
  return m;
}
template <int N, int V>
__device__ __forceinline__ float packs_max(const Pack<__nv_bfloat16, V>* p) {
  const __nv_bfloat162 m = pairs_max<__nv_bfloat162, N>(p);
  return max_nan(__low2float(m), __high2float(m));
}
template <int N, int V>
__device__ __forceinline__ float packs_max(const Pack<__half, V>* p) {
  const __half2 m = pairs_max<__half2, N>(p);
  return max_nan(__low2float(m), __high2float(m));
}

template <int NT>
struct TopSpace {
  static constexpr int kWarps = NT / 32;
  static constexpr uint32_t kGroupSize = NT / kGroups;
  // Threads that hold a margin above the bound are fewer than top_k groups'. With more that
  // reach it, many margins equal it.
  static constexpr uint32_t kLook = kMaxTop * kGroupSize;
  uint32_t order[NT];  // each thread's largest
  alignas(16) uint32_t group[kGroups];
  Key cand[kCand];
  uint32_t warp[kWarps];
  Key warp_key[kWarps];
  uint32_t look[kLook];
  uint32_t count, bound, looking;
};

// The first two steps of top_places, each followed by a barrier of the caller's: every
// thread's largest margin, and the groups' largest. The threads of a group are far apart, so
// neighbours in a row fall into different groups.
template <int NT>
__device__ __forceinline__ void top_threads(float own, TopSpace<NT>& s) {
  s.order[threadIdx.x] = order_of(own);
  if (threadIdx.x == 0) s.count = s.looking = s.bound = 0;
}
template <int NT>
__device__ __forceinline__ void top_groups(TopSpace<NT>& s) {
  const uint32_t t = threadIdx.x;
  if (t < kGroups) {
    uint32_t g = s.order[t];
#pragma unroll
    for (uint32_t q = 1; q < TopSpace<NT>::kGroupSize; q++) g = max(g, s.order[t + q * kGroups]);
    s.group[t] = g;
  }
}

// The top_k places among the span's margins, in order, after top_threads and top_groups;
// emit(place, key) is called once a place. All threads of the CTA call it.
template <typename T, int NT, typename Emit>
__device__ void top_places(const Span<T>& sp, uint32_t offset, float own, uint32_t top_k, TopSpace<NT>& s, Emit emit) {
  constexpr int kRowThreads = NT, kRowWarps = NT / 32;
  constexpr uint32_t kGroupSize = TopSpace<NT>::kGroupSize, kLook = TopSpace<NT>::kLook;
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  constexpr int kV = Span<T>::kV;
  const uint32_t mine = order_of(own);
  // A bound that top_k margins at least reach: the largest of the groups' maxima that top_k
  // groups reach; the kGroupSize threads of a group share the comparisons.
  {
    constexpr uint32_t kEach = kGroups / kGroupSize;
    const uint32_t g = s.group[t / kGroupSize], first = t % kGroupSize * kEach;
    uint32_t reach = 0;
#pragma unroll
    for (uint32_t q = 0; q < kEach; q += 4) {
      const uint4 o = *(const uint4*)(s.group + first + q);
      reach += (o.x >= g) + (o.y >= g) + (o.z >= g) + (o.w >= g);
    }
#pragma unroll
    for (uint32_t o = kGroupSize / 2; o > 0; o >>= 1) reach += __shfl_xor_sync(0xffffffffu, reach, o);
    const uint32_t best = __reduce_max_sync(0xffffffffu, reach >= top_k ? g : 0u);
    if (lane == 0) atomicMax(&s.bound, best);
  }
  __syncthreads();
  const uint32_t bound = s.bound;
  // Collects the margins whose order is at least `from`: the threads that have one are
  // listed and their vectors read again, spread over all threads. False: too many have one.
  auto collect = [&](uint32_t from) {
    if (mine >= from) {
      const uint32_t at = atomicAdd(&s.looking, 1u);
      if (at < kLook) s.look[at] = t;
    }
    __syncthreads();
    const uint32_t looking = s.looking;
    if (looking > kLook) return false;
    auto offer = [&](float x, uint32_t j) {
      const uint32_t o = order_of(x);
      if (o < from) return;
      const uint32_t at = atomicAdd(&s.count, 1u);
      if (at < kCand) s.cand[at] = key_of(o, offset + j);
    };
    const uint32_t each = (sp.vecs + kRowThreads - 1) / kRowThreads;
    for (uint32_t q = t; q < looking * each; q += kRowThreads) {
      const uint32_t who = q / each, v = s.look[who] + (q - who * each) * kRowThreads;
      if (v >= sp.vecs) continue;
      Pack<T, kV> p;
      p.load(sp.vec(v));
      if (order_of(packs_max<1>(&p)) < from) continue;
#pragma unroll
      for (int k = 0; k < kV; k++) offer(p.get(k), sp.head + v * kV + k);
    }
    if (t < sp.ragged()) offer(rw_widen(sp.x[sp.ragged_at(t)]), sp.ragged_at(t));
    return true;
  };
  const bool rare = collect(bound);
  __syncthreads();
  uint32_t count = s.count;
  uint32_t ties = 0;  // places that go to margins equal to the bound, in index order
  if (!rare || count > kCand) {
    // Many margins equal to the bound (a mask, a constant row): only those above it are
    // candidates, and the first of the equal ones follow.
    __syncthreads();
    if (t == 0) s.count = s.looking = 0;
    __syncthreads();
    if (bound != 0xffffffffu) collect(bound + 1);
    __syncthreads();
    count = s.count;
    ties = count < top_k ? top_k - count : 0;
  }
  if (count <= kCand) {
    for (uint32_t q = t; q < count; q += kRowThreads) {
      const Key k = s.cand[q];
      uint32_t place = 0;
#pragma unroll 8
      for (uint32_t w = 0; w < count; w++) place += s.cand[w] > k;
      if (place < top_k) emit(place, k);
    }
    uint32_t place = top_k - ties;  // the next place for an equal one
    for (uint32_t j0 = 0; place < top_k && j0 < sp.n; j0 += kRowThreads) {
      const uint32_t j = j0 + t;
      const bool in = j < sp.n && order_of(rw_widen(sp.x[j])) == bound;
      const uint32_t hits = __ballot_sync(0xffffffffu, in);
      __syncthreads();
      if (lane == 0) s.warp[warp] = __popc(hits);
      __syncthreads();
      uint32_t before = 0, all = 0;
      for (int w = 0; w < kRowWarps; w++) {
        before += w < (int)warp ? s.warp[w] : 0;
        all += s.warp[w];
      }
      const uint32_t at = place + before + __popc(hits & ((1u << lane) - 1));
      if (in && at < top_k) emit(at, key_of(bound, offset + j));
      place += all;
    }
    return;
  }
  // The largest margins are more than the candidates' space and lie in few groups: place by
  // place over the whole span.
  Key last = 0;  // that of the place before
  for (uint32_t place = 0; place < top_k; place++) {
    Key best = 0;
    for (uint32_t j = t; j < sp.n; j += kRowThreads) {
      const Key k = key_of(order_of(rw_widen(sp.x[j])), offset + j);
      if ((place == 0 || k < last) && k > best) best = k;  // a NaN of class 0 has the largest key
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) s.warp_key[warp] = best;
    __syncthreads();
    for (int w = 0; w < kRowWarps; w++) best = max(best, s.warp_key[w]);
    last = best;
    if (t == 0) emit(place, best);
  }
}

// The whole CTA's maximum, and its sum of v.x and v.y, in a fixed order.
template <int W>
__device__ __forceinline__ float cta_max(float m, float (&s_tmp)[W]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) s_tmp[threadIdx.x >> 5] = m;
  __syncthreads();
  m = s_tmp[0];
#pragma unroll
  for (int w = 1; w < W; w++) m = max_nan(m, s_tmp[w]);
  return m;
}
template <int W>
__device__ __forceinline__ float2 cta_sum(float2 v, float2 (&s_tmp)[W]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if ((threadIdx.x & 31) == 0) s_tmp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s_tmp[0];
#pragma unroll
  for (int w = 1; w < W; w++) {
    v.x += s_tmp[w].x;
    v.y += s_tmp[w].y;
  }
  return v;
}

// One pass over a row (or part): 16-byte vectors, kRowDepth in flight beside the kRowDepth that
// are being summed (4096 x 128000 bf16 with entropy and top 5: 185 us alone, 5.7 TB/s of the bytes
// that have to move; 337 us without the second buffer), exponents as one
// fused multiply-add e = x * c - mc with mc = round(m * c); the rounding of mc is known
// exactly and taken out of the sums at the end. A thread restates its sums only when a block
// of kRowDepth vectors holds a new maximum.
//
// The rounding of m * c is up to half a unit in its last place, and 2 to that power is in the
// sums until the end: it has to stay near 1, not only finite. So the sums hold where the row's
// maximum is steady, |m c| below 2^22, where the rounding is at most 1/4; for a row or part
// whose maximum is not (one masked with large finite numbers, margins of 1e7 and more), and for
// scales far from 1, they are taken again as e^{scale (x - m)}. Under a steady maximum margins at
// or below -2^23 / c have e^{scale (x - m)} = 0: they count as that, and blocks whose maximum so
// far is not above it are left out, so that no exponent on the way passes 2^24 in size.
// ENT: with the entropy's sum.
constexpr float kSteady = 4194304.0f;  // 2^22
__device__ __forceinline__ bool steady(float m, float c) { return fabsf(m) * c < kSteady; }
__device__ __forceinline__ float lowest_of(float c) { return __fdividef(-2.0f * kSteady, c); }
__device__ __forceinline__ bool scale_in_range(float s) { return s >= 1e-6f && s <= 1e6f; }

template <typename T, bool ENT, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) k_logprobs_row(LogprobsLaunch a, SplitRow sr) {
  constexpr int kRowThreads = NT, kRowWarps = NT / 32;
  __shared__ TopSpace<NT> s_top;
  __shared__ float s_max[kRowWarps];
  __shared__ float2 s_sum[kRowWarps];
  constexpr int kV = Span<T>::kV;
  const uint32_t t = threadIdx.x;
  const uint64_t i = blockIdx.x / sr.parts;
  const uint32_t part = blockIdx.x % sr.parts;
  const uint64_t lo = part * sr.part, hi = min(lo + sr.part, a.classes);
  const Span<T> sp((const T*)a.x + i * a.ld_x + lo, (uint32_t)(hi - lo));
  rw_let_successor_start();  // k_logprobs_join of a split row waits for this kernel
  const float c = a.scale * kLog2e, low = lowest_of(c);
  const int64_t target = t == 0 && sr.parts == 1 ? target_of(a, i) : -1;

  float m = -kInf, mc = 0.0f;
  Two s = 0, w = 0, c2 = two_of(c, c), base = 0;  // base: -mc twice
  auto absorb = [&](const Pack<T, kV>* p, auto packs) {
    constexpr int kCount = decltype(packs)::value;
    float top = packs_max<kCount>(p);
    if (!(top <= m)) {
      top = max_nan(top, m);
      const float next = top * c;
      if (m > low) {
        const float d = mc - next, f = exp2_fast(max_nan(d, kLowest));
        const Two f2 = two_of(f, f), zero = 0;
        if (ENT) w = fma2(f2, fma2(two_of(d, d), s, w), zero);
        s = fma2(f2, s, zero);
      }
      m = top;
      mc = next;
      base = two_of(-next, -next);
    }
    if (m <= low) return;
#pragma unroll
    for (int u = 0; u < kCount; u++) {
#pragma unroll
      for (int q = 0; q < kV / 2; q++) {
        const Two d = fma2(pair_of<ENT>(p[u], q, low), c2, base);
        const float2 df = both(d);
        const Two e = two_of(exp2_fast(df.x), exp2_fast(df.y));
        s = add2(s, e);
        if (ENT) w = fma2(e, d, w);
      }
    }
  };
  const std::integral_constant<int, kRowDepth> kBlockPacks;
  const std::integral_constant<int, 1> kOnePack;
  // a block is summed while the next one's loads are in flight
  constexpr uint32_t kBlock = kRowDepth * kRowThreads;
  uint32_t v = t;
  auto fetch = [&](Pack<T, kV>* p, uint32_t from) {
#pragma unroll
    for (int u = 0; u < kRowDepth; u++) p[u].load(sp.vec(from + u * kRowThreads));
  };
  auto whole = [&](uint32_t from) { return from + (kRowDepth - 1) * kRowThreads < sp.vecs; };
  if (whole(v)) {
    Pack<T, kV> p[2][kRowDepth];
    fetch(p[0], v);
    for (;;) {
      v += kBlock;
      if (!whole(v)) {
        absorb(p[0], kBlockPacks);
        break;
      }
      fetch(p[1], v);
      absorb(p[0], kBlockPacks);
      v += kBlock;
      if (!whole(v)) {
        absorb(p[1], kBlockPacks);
        break;
      }
      fetch(p[0], v);
      absorb(p[1], kBlockPacks);
    }
  }
  for (; v < sp.vecs; v += kRowThreads) {
    Pack<T, kV> p;
    p.load(sp.vec(v));
    absorb(&p, kOnePack);
  }
  bool in_row;
  const float at_target = margin_at<T>(a, i, target, in_row);
  Sums r;
  r.m = m;
  if (!(m <= low)) {
    // the sums are those of e^{scale (x - m)} times 2^off
    const float off = __fmaf_rn(m, c, -mc), f = exp2_fast(-off);
    const float2 sf = both(s), wf = both(w);
    r.s = (sf.x + sf.y) * f;
    r.t = ENT ? ((wf.x + wf.y) - off * (sf.x + sf.y)) * f / c : 0.0f;
  }
  if (t < sp.ragged()) {
    Sums one;
    one.m = rw_widen(sp.x[sp.ragged_at(t)]);
    one.s = one.m == -kInf ? 0.0f : 1.0f;
    r = join(r, one, c);
  }
  const float own = r.m;
  if (a.top_k) top_threads(own, s_top);
  const float all = cta_max(own, s_max);
  if (a.top_k) top_groups(s_top);
  if (all != -kInf) {
    if (!(steady(all, c) && scale_in_range(a.scale))) {
      r.s = r.t = 0.0f;
      for (uint32_t j = t; j < sp.n; j += kRowThreads) {
        const float d = max_nan(rw_widen(sp.x[j]) - all, kLowest), e = exp2_fast(d * c);
        r.s += e;
        r.t += e * d;
      }
    } else {
      raise(r, all, c);
    }
  }
  const float2 sums = cta_sum(make_float2(r.s, r.t), s_sum);
  r = {all, sums.x, sums.y};
  if (sr.parts == 1) {
    const RowEnd end = row_end(r);
    if (t == 0) write_row(a, i, r, end, at_target, in_row);
    if (a.top_k)
      top_places(sp, 0u, own, a.top_k, s_top, [&](uint32_t place, Key k) { write_top(a, i, place, k, end); });
  } else {
    if (t == 0) sr.sums[blockIdx.x] = r;
    if (a.top_k) {
      Key* keys = sr.keys + (uint64_t)blockIdx.x * a.top_k;
      // a part may have fewer classes than places
      if (t < a.top_k) keys[t] = 0;
      const uint32_t places = min(a.top_k, sp.n);
      top_places(sp, (uint32_t)lo, own, places, s_top, [&](uint32_t place, Key k) { keys[place] = k; });
    }
  }
}

// Joins a split row: the parts' sums, and the top places of their sorted lists. The p-th of a
// list whose head has r heads above it has p + r keys above it, and no key below the
// top_k-th largest head has a place, so few keys need comparing.
constexpr int kJoinThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) k_logprobs_join(LogprobsLaunch a, SplitRow sr) {
  __shared__ Key s_head[kMaxParts];
  __shared__ uint32_t s_above[kMaxParts];
  __shared__ Key s_cand[kMaxTop * (kMaxTop + 1) / 2];
  __shared__ uint32_t s_count;
  __shared__ Key s_bound;
  constexpr int kHeld = kMaxParts / (kJoinThreads / 32);  // a list a warp, a key a lane
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint64_t i = blockIdx.x;
  const float c = a.scale * kLog2e;
  rw_dependent_start();
  // everything that is read is on its way before anything is waited for
  const int64_t target = t == kJoinThreads - 1 ? target_of(a, i) : -1;
  const Sums* sums = sr.sums + i * sr.parts;
  Sums r, r2;
  if (lane < sr.parts) r = sums[lane];
  if (lane + 32 < sr.parts) r2 = sums[lane + 32];
  const Key* keys = sr.keys + i * sr.parts * a.top_k;
  Key held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; u++) {
    const uint32_t list = warp + u * (kJoinThreads / 32);
    held[u] = list < sr.parts && lane < a.top_k ? keys[list * a.top_k + lane] : 0;
  }
  bool in_row;
  const float at_target = margin_at<T>(a, i, target, in_row);
  if (t < sr.parts && a.top_k) s_head[t] = keys[(uint64_t)t * a.top_k];
  if (t == 0) {
    s_count = 0;
    s_bound = 1;  // with fewer lists than places only the ends of short lists, 0, are below
  }
  r = join(r, r2, c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r = join(r, shuffle_xor(r, o), c);
  const RowEnd end = row_end(r);
  if (a.top_k == 0) {
    if (t == kJoinThreads - 1) write_row(a, i, r, end, at_target, in_row);
    return;
  }
  __syncthreads();
  if (t < sr.parts) {
    uint32_t above = 0;
#pragma unroll 8
    for (uint32_t q = 0; q < sr.parts; q++) above += s_head[q] > s_head[t];
    s_above[t] = above;
    if (above == a.top_k - 1) s_bound = s_head[t];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kHeld; u++) {
    if (held[u] < s_bound) continue;
    if (lane + s_above[warp + u * (kJoinThreads / 32)] < a.top_k) s_cand[atomicAdd(&s_count, 1u)] = held[u];
  }
  __syncthreads();
  const uint32_t count = s_count;
  for (uint32_t q = t; q < count; q += kJoinThreads) {
    const Key k = s_cand[q];
    uint32_t place = 0;
#pragma unroll 8
    for (uint32_t w = 0; w < count; w++) place += s_cand[w] > k;
    if (place < a.top_k) write_top(a, i, place, k, end);
  }
  if (t == kJoinThreads - 1) write_row(a, i, r, end, at_target, in_row);
}

// =================================================================================
// The gradient: elementwise, as dx = hit - 2^d (A + B d) with d = x * c - K and the row's
// constants K = m c + log_sum log2(e), A, B and (at the target) hit. K is rounded to f32 and
// what the rounding dropped, at most 1/2 where m is steady, is a factor of A and B. Rows whose
// maximum is not steady are computed by the formula, from x - m.

// Margins below it count as it. A steady maximum at a scale in range is above -3e12, so 2^d is 0
// there, and d, at least -2e13 c, leaves A + B d finite for every A and B in use.
constexpr float kGradLowest = -1e13f;

constexpr int kGradThreads = 256;
constexpr int kGradDepth = 4;

struct RowGrad {
  float k, a, b, hit;
  int32_t target;  // -1: none
  int32_t kind;    // 0: zeros, 1: by the constants, 2: by the formula
};

__device__ __forceinline__ RowGrad row_grad(const LogprobsGradLaunch& a, uint64_t i) {
  RowGrad r = {0.0f, 0.0f, 0.0f, 0.0f, -1, 0};
  const float m = a.row_max[i];
  if (m == -kInf) return r;
  float g = 0.0f;
  if (a.targets) {
    const int64_t t = a.target_type == RW_I64 ? ((const int64_t*)a.targets)[i] : ((const int32_t*)a.targets)[i];
    g = a.grad_logp[i];  // on its way whatever the target is
    if (t >= 0 && (uint64_t)t < a.classes) r.target = (int32_t)t;
    else g = 0.0f;
  }
  const float e = a.grad_entropy ? a.grad_entropy[i] : 0.0f;
  if (g == 0.0f && e == 0.0f) return r;
  const float c = a.scale * kLog2e;
  if (!(steady(m, c) && scale_in_range(a.scale))) {
    r.kind = 2;
    return r;
  }
  // k = m c + log_sum log2(e) in two f32: products and sum with their roundings
  constexpr float kLog2eRest = (float)(1.4426950408889634 - (double)kLog2e);
  const float s = a.log_sum[i];
  const float mc = m * c, sl = s * kLog2e;
  const float k = mc + sl, back = k - mc;
  const float rest = ((mc - (k - back)) + (sl - back)) +
                     (__fmaf_rn(m, c, -mc) + __fmaf_rn(s, kLog2e, -sl) + s * kLog2eRest);
  const float f = exp2_fast(-rest) * a.scale;
  r.k = k;
  const float h = a.grad_entropy ? a.entropy[i] : 0.0f;
  constexpr float kLn2 = 0.6931471805599453f;
  r.a = f * (g + e * (h - rest * kLn2));
  r.b = f * e * kLn2;
  r.hit = g * a.scale;
  r.kind = fabsf(r.a) < 1e30f && fabsf(r.b) * c < 1e24f ? 1 : 2;  // A + B d stays finite
  return r;
}
// One element by the formula. p is multiplied first: where it is 0 nothing else may overflow.
__device__ __forceinline__ float grad_of(const LogprobsGradLaunch& a, uint64_t i, float x, bool hit, bool in) {
  const float lp = max_nan((x - a.row_max[i]) * a.scale - a.log_sum[i], kLowest);
  const float g = in ? a.grad_logp[i] : 0.0f;
  const float e = a.grad_entropy ? a.grad_entropy[i] : 0.0f, h = a.grad_entropy ? a.entropy[i] : 0.0f;
  const float p = exp2_fast(lp * kLog2e);
  return ((hit ? g : 0.0f) - (p * g + e * (p * (lp + h)))) * a.scale;
}
__device__ __forceinline__ float grad_element(const LogprobsGradLaunch& a, uint64_t i, const RowGrad& r, float c,
                                              float x, uint32_t j) {
  const bool hit = (int32_t)j == r.target;
  if (r.kind == 2) return grad_of(a, i, x, hit, r.target >= 0);
  const float d = __fmaf_rn(max_nan(x, kGradLowest), c, -r.k);
  const float v = -exp2_fast(d) * __fmaf_rn(r.b, d, r.a);
  return hit ? v + r.hit : v;
}

// Many classes: a CTA takes kGradThreads * kGradDepth vectors of one row. x and dx lie the
// same distance from a 16-byte boundary (VEC), else it goes element by element (4096 x 32000
// bf16: 107 us and 348 us). 4096 x 128000 bf16 with entropy: 379 us, 5.5 TB/s, bound by the
// memory's mixed reads and writes; 405 us with the 48 registers that it takes unbounded.
template <typename T, bool VEC, bool ENT>
__global__ void __launch_bounds__(kGradThreads, sizeof(T) == 2 ? 6 : 5) k_logprobs_grad(LogprobsGradLaunch a, uint32_t chunks) {
  constexpr int kV = Span<T>::kV;
  const uint64_t i = blockIdx.x / chunks;
  const uint32_t chunk = blockIdx.x % chunks, t = threadIdx.x;
  const Span<T> sp((const T*)a.x + i * a.ld_x, (uint32_t)a.classes);
  T* dx = (T*)a.dx + i * a.ld_dx;
  const RowGrad r = row_grad(a, i);
  const float c = a.scale * kLog2e;
  if (!VEC) {
    constexpr uint32_t kPer = kGradThreads * kGradDepth * kV;
    const uint32_t end = min((uint32_t)a.classes, (chunk + 1) * kPer);
    for (uint32_t j = chunk * kPer + t; j < end; j += kGradThreads)
      dx[j] = rw_round<T>(r.kind ? grad_element(a, i, r, c, rw_widen(sp.x[j]), j) : 0.0f);
    return;
  }
  T* out = dx + sp.head;
  const uint32_t v0 = chunk * (kGradThreads * kGradDepth) + t;
  Pack<T, kV> p[kGradDepth];
  if (r.kind) {
#pragma unroll
    for (int u = 0; u < kGradDepth; u++)
      if (v0 + u * kGradThreads < sp.vecs) p[u].load(sp.vec(v0 + u * kGradThreads));
  }
  if (chunk == 0 && t < sp.ragged()) {
    const uint32_t j = sp.ragged_at(t);
    dx[j] = rw_round<T>(r.kind ? grad_element(a, i, r, c, rw_widen(sp.x[j]), j) : 0.0f);
  }
  // the target's vector, none: beyond the last
  const uint32_t hit = r.target >= (int32_t)sp.head ? ((uint32_t)r.target - sp.head) / kV : 0xffffffffu;
  const Two c2 = two_of(c, c), k2 = two_of(-r.k, -r.k), a2 = two_of(-r.a, -r.a), b2 = two_of(-r.b, -r.b);
#pragma unroll
  for (int u = 0; u < kGradDepth; u++) {
    const uint32_t v = v0 + u * kGradThreads;
    if (v >= sp.vecs) break;
    if (r.kind == 1 && v != hit) {
#pragma unroll
      for (int q = 0; q < kV / 2; q++) {
        const Two d = fma2(pair_of<ENT>(p[u], q, kGradLowest), c2, k2);
        const float2 df = both(d), w = ENT ? both(fma2(b2, d, a2)) : make_float2(-r.a, -r.a);
        p[u].set(2 * q, exp2_fast(df.x) * w.x);
        p[u].set(2 * q + 1, exp2_fast(df.y) * w.y);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kV; k++)
        p[u].set(k, r.kind ? grad_element(a, i, r, c, p[u].get(k), sp.head + v * kV + k) : 0.0f);
    }
    p[u].store(out + (size_t)v * kV);
  }
}

// Few classes: a CTA takes `rows` whole rows, their constants in shared memory. VEC: the
// matrices are contiguous and aligned, so the rows are one run of 16-byte vectors whose
// elements may lie in different rows; 1000000 x 7 f32, inputs out of the L2: 20 us, 3.5 TB/s, the
// rows' constants waited for before the first vector. Strided rows go element by element
// (100000 x 100 bf16: 17 us and 49 us). magic = ceil(2^32 / classes): an element's row is the
// high half of its index times magic, exactly, as index * classes < 2^32.
constexpr uint32_t kGradRows = 1024;
// Vectors a thread: 8, 4 and 2 take 20, 24 and 24 us at 1000000 x 7 f32, 17, 18 and 20 us at
// 27233 x 320 f32, 85, 93 and 94 us at 100000 x 1000 bf16, but 28, 27 and 29 us at 200000 x 100.
constexpr uint64_t kGradFewDepth = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kGradThreads) k_logprobs_grad_few(LogprobsGradLaunch a, uint32_t rows, uint32_t magic) {
  __shared__ float4 s_row[kGradRows];     // k (NaN: by the formula), a, b, hit
  __shared__ int32_t s_target[kGradRows];  // -1: none, -2: a row of zeros
  constexpr int kV = VEC ? 16 / (int)sizeof(T) : 1;
  const uint64_t first = (uint64_t)blockIdx.x * rows;
  const uint32_t count = (uint32_t)min((uint64_t)rows, a.n - first), classes = (uint32_t)a.classes;
  const float c = a.scale * kLog2e;
  const uint32_t total = count * classes;
  const T* x = (const T*)a.x + first * a.ld_x;
  T* dx = (T*)a.dx + first * a.ld_dx;
  bool formula = false;
  for (uint32_t k = threadIdx.x; k < count; k += kGradThreads) {
    const RowGrad r = row_grad(a, first + k);
    s_row[k] = make_float4(r.kind == 2 ? NAN : r.k, r.a, r.b, r.hit);
    s_target[k] = r.kind ? r.target : -2;
    formula |= r.kind == 2;
  }
  formula = __syncthreads_or(formula);
  auto element = [&](uint32_t at, uint32_t row, float in) {
    const uint32_t j = at - row * classes;
    const float4 r = s_row[row];
    const int32_t target = s_target[row];
    const bool hit = (int32_t)j == target;
    const float d = __fmaf_rn(max_nan(in, kGradLowest), c, -r.x);
    float v = -exp2_fast(d) * __fmaf_rn(r.z, d, r.y);
    v = hit ? v + r.w : v;
    return target == -2 ? 0.0f : v;
  };
  auto row_of = [&](uint32_t at) { return classes == 1 ? at : __umulhi(at, magic); };
  if (formula) {  // element by element, every row by its own rule
    for (uint32_t at = threadIdx.x; at < total; at += kGradThreads) {
      const uint32_t row = row_of(at), j = at - row * classes;
      const int32_t target = s_target[row];
      const float in = rw_widen(x[row * a.ld_x + j]);
      const bool by_formula = s_row[row].x != s_row[row].x;
      dx[row * a.ld_dx + j] = rw_round<T>(
          by_formula ? grad_of(a, first + row, in, (int32_t)j == target, target >= 0) : element(at, row, in));
    }
    return;
  }
  for (uint32_t j0 = threadIdx.x * kV; j0 < total; j0 += kGradThreads * kV) {
    if (VEC && j0 + kV <= total) {
      Pack<T, kV> p;
      p.load(x + j0);
      const uint32_t row = row_of(j0), j = j0 - row * classes;
      const int32_t target = s_target[row];
      if (kV > 1 && classes >= 16 * kV && j + kV <= classes && (uint32_t)(target - (int32_t)j) >= kV) {
        // one row's, and the target elsewhere
        const float4 r = s_row[row];
        const Two c2 = two_of(c, c), k2 = two_of(-r.x, -r.x), a2 = two_of(-r.y, -r.y), b2 = two_of(-r.z, -r.z);
#pragma unroll
        for (int q = 0; q < kV / 2; q++) {
          const Two d = fma2(pair_of<true>(p, q, kGradLowest), c2, k2);
          const float2 df = both(d), w = both(fma2(b2, d, a2));
          p.set(2 * q, target == -2 ? 0.0f : exp2_fast(df.x) * w.x);
          p.set(2 * q + 1, target == -2 ? 0.0f : exp2_fast(df.y) * w.y);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kV; k++) p.set(k, element(j0 + k, row_of(j0 + k), p.get(k)));
      }
      p.store(dx + j0);
    } else {
      for (uint32_t at = j0; at < min(total, j0 + kV); at++) {
        const uint32_t row = row_of(at), j = at - row * classes;
        const size_t from = VEC ? at : row * a.ld_x + j, to = VEC ? at : row * a.ld_dx + j;
        dx[to] = rw_round<T>(element(at, row, rw_widen(x[from])));
      }
    }
  }
}

uint32_t grid_of(uint64_t blocks, uint32_t per_sm) {
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(blocks, 148ull * per_sm));
}

// Rows in registers up to here, by CTAs above (20000 x 1000 bf16, top 5: 36 us and 47 us).
constexpr uint64_t kFewClasses = 1024;

// Parts a row: with fewer rows than four CTAs an SM, enough parts to make that many, of 4096
// classes at least (a vector a thread and more; top 5 of 8 x 128000 bf16: 7.7 us, 8.6 us from 2048
// on, 7.1 us from 8192 on; of 1 x 16384: 6.4, 5.8 and 6.1 us).
SplitRow split_of(uint64_t n, uint64_t classes) {
  SplitRow r = {1, classes, nullptr, nullptr};
  if (classes <= kFewClasses || n == 0 || n >= 148 * 4) return r;
  const uint64_t want = (148 * 4 + n - 1) / n;
  const uint64_t parts = std::min<uint64_t>({want, kMaxParts, std::max<uint64_t>(1, classes / 4096)});
  r.part = ((classes + parts - 1) / parts + 7) / 8 * 8;
  r.parts = (uint32_t)((classes + r.part - 1) / r.part);
  return r;
}

}  // namespace

uint64_t logprobs_workspace(uint64_t n, uint64_t classes, int, uint32_t top_k) {
  const SplitRow r = split_of(n, classes);
  if (r.parts == 1) return 0;
  const uint64_t cells = n * r.parts;
  return (cells * sizeof(Sums) + 255) / 256 * 256 + cells * top_k * sizeof(Key);
}

cudaError_t launch_logprobs(const LogprobsLaunch& a, void* workspace, cudaStream_t s, int* nl) {
  if (a.n == 0) return cudaSuccess;
  *nl += 1;
  if (a.classes <= kFewClasses)
    return rw_with_type(a.type, [&](auto t) {
      using T = decltype(t);
      auto go = [&](auto* k, uint64_t lanes) {
        const uint64_t rows = kGroupThreads / lanes;
        return rw_launch(k, dim3(grid_of((a.n + rows - 1) / rows, 32)), dim3(kGroupThreads), 0, s, false, a);
      };
      if (a.classes <= 8) return go(k_logprobs_few<T, 1, 8>, 1);
      if (a.classes <= 32) return go(k_logprobs_few<T, 4, 8>, 4);
      if (a.classes <= 128)
        return a.top_k <= kSharedPlaces ? go(k_logprobs_few<T, 8, 16>, 8) : go(k_logprobs_few<T, 32, 4>, 32);
      if (a.classes <= 256) return go(k_logprobs_few<T, 32, 8>, 32);
      if (a.classes <= 384) return go(k_logprobs_few<T, 32, 12>, 32);
      if (a.classes <= 512) return go(k_logprobs_few<T, 32, 16>, 32);
      if (a.classes <= 768) return go(k_logprobs_few<T, 32, 24>, 32);
      return go(k_logprobs_few<T, 32, 32>, 32);
    });
  SplitRow r = split_of(a.n, a.classes);
  const uint64_t cells = a.n * r.parts;
  if (cells > 0x7fffffffull) return cudaErrorInvalidValue;
  r.sums = (Sums*)workspace;
  r.keys = (Key*)((char*)workspace + (cells * sizeof(Sums) + 255) / 256 * 256);
  return rw_with_type(a.type, [&](auto t) {
    using T = decltype(t);
    const dim3 grid((uint32_t)cells);
    const bool narrow = a.n >= 148 * 4 && a.classes * sizeof(T) <= kShortBytes;
    auto go = [&](auto* k, int threads) { return rw_launch(k, grid, dim3(threads), 0, s, false, a, r); };
    cudaError_t e;
    if (narrow) e = a.entropy ? go(k_logprobs_row<T, true, kShortThreads>, kShortThreads)
                              : go(k_logprobs_row<T, false, kShortThreads>, kShortThreads);
    else e = a.entropy ? go(k_logprobs_row<T, true, kRowThreads>, kRowThreads)
                       : go(k_logprobs_row<T, false, kRowThreads>, kRowThreads);
    if (e != cudaSuccess || r.parts == 1) return e;
    *nl += 1;
    return rw_launch(k_logprobs_join<T>, dim3((uint32_t)a.n), dim3(kJoinThreads), 0, s, true, a, r);
  });
}

// Up to this many classes whole rows share CTAs where they are one run of vectors, since a CTA
// of one row would have too little to do (50000 x 2050 bf16: 84 us and 173 us, x 4096 with
// entropy 153 us and 233 us, but 20000 x 8192 135 us and 122 us), else up to kGradFewStrided.
constexpr uint64_t kGradFew = 8192, kGradFewStrided = 1024;

cudaError_t launch_logprobs_grad(const LogprobsGradLaunch& a, cudaStream_t s, int* nl) {
  if (a.n == 0 || a.classes == 0) return cudaSuccess;
  *nl += 1;
  return rw_with_type(a.type, [&](auto t) {
    using T = decltype(t);
    constexpr uint64_t kV = 16 / sizeof(T);
    const dim3 block(kGradThreads);
    const uintptr_t x = (uintptr_t)a.x, dx = (uintptr_t)a.dx;
    const bool one = a.n == 1;
    const bool run = x % 16 == 0 && dx % 16 == 0 && (one || (a.ld_x == a.classes && a.ld_dx == a.classes));
    if (a.classes <= (run ? kGradFew : kGradFewStrided)) {
      const bool vec = run;
      // about kGradFewDepth vectors a thread, whole vectors in whole rows
      uint64_t rows = kGradThreads * kGradFewDepth * kV / a.classes;
      rows = std::min<uint64_t>(std::max<uint64_t>(rows, 1) + kV - 1, kGradRows) / kV * kV;
      const uint64_t ctas = (a.n + rows - 1) / rows;
      if (ctas > 0x7fffffffull) return cudaErrorInvalidValue;
      const uint32_t magic = (uint32_t)(((1ull << 32) + a.classes - 1) / a.classes);
      const dim3 grid((uint32_t)ctas);
      return vec ? rw_launch(k_logprobs_grad_few<T, true>, grid, block, 0, s, false, a, (uint32_t)rows, magic)
                 : rw_launch(k_logprobs_grad_few<T, false>, grid, block, 0, s, false, a, (uint32_t)rows, magic);
    }
    const bool vec = x % 16 == dx % 16 && (one || (a.ld_x * sizeof(T)) % 16 == (a.ld_dx * sizeof(T)) % 16);
    const uint64_t per = kGradThreads * kGradDepth * kV, chunks = (a.classes + per - 1) / per;
    if (a.n * chunks > 0x7fffffffull) return cudaErrorInvalidValue;
    const dim3 grid((uint32_t)(a.n * chunks));
    if (!vec) return rw_launch(k_logprobs_grad<T, false, true>, grid, block, 0, s, false, a, (uint32_t)chunks);
    return a.grad_entropy ? rw_launch(k_logprobs_grad<T, true, true>, grid, block, 0, s, false, a, (uint32_t)chunks)
                          : rw_launch(k_logprobs_grad<T, true, false>, grid, block, 0, s, false, a, (uint32_t)chunks);
  });
}
