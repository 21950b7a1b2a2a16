// Embedding lookup, its gradient and dropout: the vector-valued side of the categorical
// columns (encode.cu looks up and sums one scalar per key).
//
//   lookup    out[i] = scale * table[ids[i]]
//   gradient  dtable[v] (+)= scale * sum over i with ids[i] = v of grad[i]
//   dropout   y[e] = keep(e) ? x[e] / (1 - p) : 0
//
// All three move bytes: nothing is computed that the memory does not bound. An id outside
// the table is padding: a zero row, and no gradient.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "rw_internal.cuh"
#include "rw_types.cuh"

namespace {

constexpr int kSms = 148;

// =================================================================================
// lookup

template <typename TI, typename TO, typename ID>
__global__ void __launch_bounds__(256) k_embed(EmbedLaunch a) {
  const TI* table = (const TI*)a.table;
  const ID* ids = (const ID*)a.ids;
  TO* out = (TO*)a.out;
  for (uint64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
    const int64_t id = (int64_t)ids[i];
    const bool in = id >= 0 && (uint64_t)id < a.vocab;
    const TI* row = table + (in ? (uint64_t)id : 0) * a.ld_table;
    for (uint64_t c = threadIdx.x; c < a.d; c += blockDim.x)
      out[i * a.ld_out + c] = rw_round<TO>(in ? a.scale * rw_widen(row[c]) : 0.0f);
  }
}

// =================================================================================
// gradient
//
// The positions 0..n-1 are sorted by id (stably, so a sum's order is the positions' order
// and the result does not depend on timing), then each run of equal ids is summed.
//
// The sort is a radix sort over (id, position) pairs, digits of at most 9 bits, two
// launches a pass: digit counts per part of the input, then a stable scatter in which
// every CTA derives its part's bases from the counts of all parts.

constexpr int kRadixBits = 9;
constexpr int kRadix = 1 << kRadixBits;
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortRounds = 8;
constexpr int kSortTile = kSortThreads * kSortRounds;

struct SortPass {
  const void* ids;             // first pass: the ids
  const unsigned long long* in;  // later passes: (id << 32 | position)
  unsigned long long* out;
  uint32_t* counts;            // [parts][kRadix]
  uint64_t n, part;            // items; items a part
  uint64_t vocab;              // ids outside 0..vocab-1 sort as vocab
  uint32_t parts, shift;
};

template <typename ID, bool FIRST>
__device__ __forceinline__ unsigned long long sort_item(const SortPass& p, uint64_t i) {
  if (!FIRST) return p.in[i];
  const int64_t id = (int64_t)((const ID*)p.ids)[i];
  const uint64_t key = id >= 0 && (uint64_t)id < p.vocab ? (uint64_t)id : p.vocab;
  return key << 32 | i;
}
__device__ __forceinline__ uint32_t sort_digit(const SortPass& p, unsigned long long item) {
  return (uint32_t)(item >> 32 >> p.shift) & (kRadix - 1);
}

template <typename ID, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) k_token_count(SortPass p) {
  __shared__ uint32_t s_count[kRadix];
  for (int d = threadIdx.x; d < kRadix; d += kSortThreads) s_count[d] = 0;
  __syncthreads();
  const uint64_t lo = (uint64_t)blockIdx.x * p.part, hi = min(lo + p.part, p.n);
  for (uint64_t i = lo + threadIdx.x; i < hi; i += kSortThreads)
    atomicAdd(&s_count[sort_digit(p, sort_item<ID, FIRST>(p, i))], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < kRadix; d += kSortThreads)
    p.counts[(uint64_t)blockIdx.x * kRadix + d] = s_count[d];
}

template <typename ID, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) k_token_scatter(SortPass p) {
  __shared__ uint32_t s_base[kRadix];               // next output slot of each digit
  __shared__ uint32_t s_warp[kSortWarps][kRadix];   // a warp's counts, then its bases
  __shared__ uint32_t s_sum[kSortWarps];
  static_assert(kRadix == kSortThreads, "one thread a digit");
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  uint32_t before = 0, total = 0;
  for (uint32_t q = 0; q < p.parts; q++) {
    const uint32_t c = p.counts[(uint64_t)q * kRadix + t];
    before += q < blockIdx.x ? c : 0;
    total += c;
  }
  uint32_t incl = total;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= (uint32_t)d) incl += y;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  uint32_t lower = 0;
  for (uint32_t w = 0; w < warp; w++) lower += s_sum[w];
  s_base[t] = lower + incl - total + before;

  const uint64_t lo = (uint64_t)blockIdx.x * p.part, hi = min(lo + p.part, p.n);
  for (uint64_t tile = lo; tile < hi; tile += kSortTile) {
#pragma unroll
    for (int w = 0; w < kSortWarps; w++) s_warp[w][t] = 0;
    __syncthreads();
    unsigned long long item[kSortRounds];
    uint32_t rank[kSortRounds];
    // warp w takes 32 * kSortRounds consecutive items, 32 a round
    const uint64_t first = tile + (uint64_t)warp * 32 * kSortRounds + lane;
#pragma unroll
    for (int r = 0; r < kSortRounds; r++)
      item[r] = first + r * 32 < hi ? sort_item<ID, FIRST>(p, first + r * 32) : 0;
#pragma unroll
    for (int r = 0; r < kSortRounds; r++) {
      const bool in = first + r * 32 < hi;
      const uint32_t d = sort_digit(p, item[r]);
      const uint32_t peers = __match_any_sync(0xffffffffu, in ? d : (uint32_t)kRadix);
      const uint32_t ahead = __popc(peers & ((1u << lane) - 1));
      rank[r] = in ? s_warp[warp][d] + ahead : 0;
      __syncwarp();
      if (in && ahead == 0) s_warp[warp][d] += __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    uint32_t run = s_base[t];
#pragma unroll
    for (int w = 0; w < kSortWarps; w++) {
      const uint32_t c = s_warp[w][t];
      s_warp[w][t] = run;
      run += c;
    }
    s_base[t] = run;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; r++)
      if (first + r * 32 < hi) p.out[s_warp[warp][sort_digit(p, item[r])] + rank[r]] = item[r];
    __syncthreads();
  }
}

// One CTA per sorted position; the CTA at the start of a run of equal ids sums the run.
template <typename TG, typename TD>
__global__ void __launch_bounds__(256) k_embed_sum(EmbedGradLaunch a, const unsigned long long* pairs) {
  for (uint64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
    const uint32_t id = (uint32_t)(pairs[i] >> 32);
    if (id >= a.vocab || (i > 0 && (uint32_t)(pairs[i - 1] >> 32) == id)) continue;
    TD* row = (TD*)a.dtable + (uint64_t)id * a.ld_dtable;
    for (uint64_t c = threadIdx.x; c < a.d; c += blockDim.x) {
      float acc = 0.0f;
      for (uint64_t j = i; j < a.n && (uint32_t)(pairs[j] >> 32) == id; j++)
        acc += rw_widen(((const TG*)a.grad)[(uint64_t)(uint32_t)pairs[j] * a.ld_grad + c]);
      acc *= a.scale;
      if (a.accumulate) acc += rw_widen(row[c]);
      row[c] = rw_round<TD>(acc);
    }
  }
}

template <typename TD>
__global__ void __launch_bounds__(256) k_zero_rows(TD* p, uint64_t rows, uint64_t d, uint64_t ld) {
  for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (uint64_t c = threadIdx.x; c < d; c += blockDim.x) p[r * ld + c] = rw_round<TD>(0.0f);
}

// =================================================================================
// dropout
//
// The keep decisions come from Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011), a function of the seed and a counter, so the
// mask is recomputed wherever it is needed and never stored. Counter (e / 8, sequence)
// gives the 128 bits that elements 8 (e / 8) .. 8 (e / 8) + 7 share, 16 bits each. 16 bits
// instead of 32 halve the generator's work; p is then a multiple of 2^-16 and the scale
// uses that p, so the expectation is exact.

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t group, uint64_t sequence, uint64_t seed) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32);
  uint32_t c2 = (uint32_t)sequence, c3 = (uint32_t)(sequence >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

template <typename T>
__global__ void __launch_bounds__(256) k_dropout(DropoutLaunch a) {
  const uint64_t total = a.rows * a.cols, groups = (total + 7) / 8;
  const T* x = (const T*)a.x;
  T* y = (T*)a.y;
  for (uint64_t g = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; g < groups;
       g += (uint64_t)gridDim.x * blockDim.x) {
    const Words w = philox(g, a.sequence, a.seed);
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const uint64_t e = g * 8 + k;
      if (e >= total) break;
      const uint64_t r = e / a.cols, c = e - r * a.cols;
      const uint32_t half = k & 1 ? w.w[k / 2] >> 16 : w.w[k / 2] & 0xffff;
      const float v = half >= a.limit ? rw_widen(x[r * a.ld_x + c]) * a.scale : 0.0f;
      y[r * a.ld_y + c] = rw_round<T>(v);
    }
  }
}

uint32_t grid_of(uint64_t blocks, uint32_t per_sm) {
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(blocks, (uint64_t)kSms * per_sm));
}

}  // namespace

cudaError_t launch_embed(const EmbedLaunch& a, cudaStream_t s, int* nl) {
  if (a.n == 0 || a.d == 0) return cudaSuccess;
  *nl += 1;
  return rw_with_type(a.table_type, [&](auto ti) {
    return rw_with_type(a.out_type, [&](auto to) {
      return rw_with_index(a.id_type, [&](auto id) {
        return rw_launch(k_embed<decltype(ti), decltype(to), decltype(id)>, dim3(grid_of(a.n, 8)),
                         dim3(256), 0, s, false, a);
      });
    });
  });
}

namespace {

// Sizes and workspace offsets of one gradient call.
struct GradPlan {
  uint64_t part;
  uint32_t parts, passes;
  uint64_t pairs0, pairs1, counts, bytes;  // offsets
};

GradPlan grad_plan(uint64_t n, uint64_t vocab) {
  GradPlan g;
  const uint64_t tiles = (n + kSortTile - 1) / kSortTile;
  const uint64_t per = std::max<uint64_t>(1, (tiles + kSms - 1) / kSms);
  g.part = per * kSortTile;
  g.parts = (uint32_t)((n + g.part - 1) / g.part);
  uint32_t bits = 1;
  while (bits < 32 && vocab >> bits) bits++;  // keys 0..vocab
  g.passes = (bits + kRadixBits - 1) / kRadixBits;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  g.pairs0 = take(n * 8);
  g.pairs1 = take(n * 8);
  g.counts = take((uint64_t)g.parts * kRadix * 4);
  g.bytes = at;
  return g;
}

}  // namespace

uint64_t embed_grad_workspace(uint64_t n, uint64_t d, uint64_t vocab) {
  return n == 0 || d == 0 || vocab == 0 ? 0 : grad_plan(n, vocab).bytes;
}

cudaError_t launch_embed_grad(const EmbedGradLaunch& a, void* workspace, cudaStream_t s, int* nl) {
  if (a.d == 0 || a.vocab == 0) return cudaSuccess;
  cudaError_t e = cudaSuccess;
  if (!a.accumulate) {
    *nl += 1;
    e = rw_with_type(a.dtable_type, [&](auto td) {
      using TD = decltype(td);
      return rw_launch(k_zero_rows<TD>, dim3(grid_of(a.vocab, 8)), dim3(256), 0, s, false,
                       (TD*)a.dtable, a.vocab, a.d, a.ld_dtable);
    });
  }
  if (a.n == 0 || e != cudaSuccess) return e;
  const GradPlan g = grad_plan(a.n, a.vocab);
  char* ws = (char*)workspace;
  unsigned long long* buf[2] = {(unsigned long long*)(ws + g.pairs0),
                                (unsigned long long*)(ws + g.pairs1)};
  SortPass p = {};
  p.ids = a.ids;
  p.counts = (uint32_t*)(ws + g.counts);
  p.n = a.n;
  p.part = g.part;
  p.vocab = a.vocab;
  p.parts = g.parts;
  for (uint32_t i = 0; i < g.passes && e == cudaSuccess; i++) {
    p.in = buf[(i + 1) & 1];
    p.out = buf[i & 1];
    p.shift = i * kRadixBits;
    *nl += 2;
    e = rw_with_index(a.id_type, [&](auto id) {
      using ID = decltype(id);
      const dim3 grid(g.parts), block(kSortThreads);
      cudaError_t r = i == 0 ? rw_launch(k_token_count<ID, true>, grid, block, 0, s, false, p)
                             : rw_launch(k_token_count<ID, false>, grid, block, 0, s, false, p);
      if (r != cudaSuccess) return r;
      return i == 0 ? rw_launch(k_token_scatter<ID, true>, grid, block, 0, s, false, p)
                    : rw_launch(k_token_scatter<ID, false>, grid, block, 0, s, false, p);
    });
  }
  if (e != cudaSuccess) return e;
  *nl += 1;
  return rw_with_type(a.grad_type, [&](auto tg) {
    return rw_with_type(a.dtable_type, [&](auto td) {
      return rw_launch(k_embed_sum<decltype(tg), decltype(td)>, dim3(grid_of(a.n, 8)), dim3(256), 0,
                       s, false, a, (const unsigned long long*)buf[(g.passes + 1) & 1]);
    });
  });
}

cudaError_t launch_dropout(const DropoutLaunch& a, cudaStream_t s, int* nl) {
  if (a.rows == 0 || a.cols == 0) return cudaSuccess;
  *nl += 1;
  const uint64_t groups = (a.rows * a.cols + 7) / 8;
  return rw_with_type(a.type, [&](auto t) {
    return rw_launch(k_dropout<decltype(t)>, dim3(grid_of((groups + 255) / 256, 8)), dim3(256), 0, s,
                     false, a);
  });
}
