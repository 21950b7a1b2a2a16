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
constexpr int kSortRounds = 4;
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
  rw_dependent_start();
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
  rw_dependent_start();
  uint32_t before = 0, total = 0;
  for (uint32_t q0 = 0; q0 < p.parts; q0 += 16) {  // 16 loads in flight
    uint32_t c[16];
#pragma unroll
    for (int u = 0; u < 16; u++)
      c[u] = q0 + u < p.parts ? p.counts[(uint64_t)(q0 + u) * kRadix + t] : 0;
#pragma unroll
    for (int u = 0; u < 16; u++) {
      before += q0 + u < blockIdx.x ? c[u] : 0;
      total += c[u];
    }
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

// Short inputs are sorted by counting instead, in one launch: a position's place is the
// number of positions before it in the order (id, position). n * n comparisons: 2 us at
// n = 512, and at kCountSort still less than the radix sort's launches.
constexpr uint64_t kCountSort = 4096;
constexpr int kCountThreads = 256;
constexpr int kCountShare = 8;  // threads that share a position's comparisons

template <typename ID>
__global__ void __launch_bounds__(kCountThreads)
    k_token_rank(const ID* __restrict__ ids, uint32_t n, uint32_t vocab, unsigned long long* __restrict__ out) {
  __shared__ uint32_t s_key[kCountSort];
  for (uint32_t i = threadIdx.x; i < n; i += kCountThreads) {
    const int64_t id = (int64_t)ids[i];
    s_key[i] = id >= 0 && id < (int64_t)vocab ? (uint32_t)id : vocab;
  }
  __syncthreads();
  const uint32_t t = blockIdx.x * kCountThreads + threadIdx.x, i = t / kCountShare, part = t % kCountShare;
  const uint32_t key = i < n ? s_key[i] : 0;
  uint32_t place = 0;
  if (i < n) {
#pragma unroll 4
    for (uint32_t j = part; j < n; j += kCountShare) {
      const uint32_t other = s_key[j];
      place += other < key || (other == key && j < i);
    }
  }
#pragma unroll
  for (int o = kCountShare / 2; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
  if (i < n && part == 0) out[place] = (unsigned long long)key << 32 | i;
}

// The sums. The sorted positions are cut into chunks of equal length; a slot of `tx`
// threads (V columns each) walks one chunk in order with its running sum in registers.
// A run of equal ids inside one chunk is finished there; a run that crosses chunks leaves
// an f32 partial sum in each of them, and k_embed_join adds those in the chunks' order. So
// a frequent id is summed by many slots, and the order of every addition is fixed by the
// ids and the sizes.

constexpr int kSumThreads = 256;
constexpr int kSumDepth = 4;    // rows in flight per thread
constexpr int kZeroRows = 64;   // table rows a zeroing CTA covers
constexpr int kJoinThreads = 512;
constexpr int kJoinCols = 128;  // columns of one join (a float4 a lane)
constexpr uint32_t kNone = 0xffffffffu;

struct ChunkPlan {
  uint32_t chunk;       // positions a chunk
  uint32_t chunks;
  uint32_t tx, slots;   // threads a slot, slots a CTA
  uint32_t col_blocks;  // CTAs that share a chunk group's columns
  uint32_t sum_ctas;    // CTAs that sum; the rest zero rows that no id names
  uint64_t dv;          // vectors a row
  uint64_t pitch;       // floats of one partial row (a multiple of 4)
};

__device__ __forceinline__ uint32_t key_of(unsigned long long pair) { return (uint32_t)(pair >> 32); }

// The first of n sorted pairs whose id is at least key.
__device__ __forceinline__ uint64_t lower_bound(const unsigned long long* pairs, uint64_t n, uint32_t key) {
  uint64_t lo = 0, hi = n;
  while (lo < hi) {
    const uint64_t mid = (lo + hi) / 2;
    if (key_of(pairs[mid]) < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

template <typename TG, typename TD, int V>
__global__ void __launch_bounds__(kSumThreads)
    k_embed_chunks(EmbedGradLaunch a, ChunkPlan cp, const unsigned long long* __restrict__ pairs,
                   float* __restrict__ partial) {
  const uint32_t slot = threadIdx.x / cp.tx, lane = threadIdx.x % cp.tx;
  TD* dtable = (TD*)a.dtable;
  rw_dependent_start();
  if (blockIdx.x >= cp.sum_ctas) {  // zero the rows of this block that no id names
    __shared__ bool s_absent[kZeroRows];
    const uint64_t first = (uint64_t)(blockIdx.x - cp.sum_ctas) * kZeroRows;
    if (threadIdx.x < kZeroRows && first + threadIdx.x < a.vocab) {
      const uint32_t key = (uint32_t)(first + threadIdx.x);
      const uint64_t at = lower_bound(pairs, a.n, key);
      s_absent[threadIdx.x] = at == a.n || key_of(pairs[at]) != key;
    }
    __syncthreads();
    if (slot >= cp.slots) return;
    Pack<TD, V> zero;
#pragma unroll
    for (int k = 0; k < V; k++) zero.set(k, 0.0f);
    for (uint64_t r = slot; r < kZeroRows && first + r < a.vocab; r += cp.slots) {
      if (!s_absent[r]) continue;
      TD* row = dtable + (first + r) * a.ld_dtable;
      for (uint64_t c = lane; c < cp.dv; c += cp.tx) zero.store(row + c * V);
    }
    return;
  }
  const uint64_t chunk = (uint64_t)(blockIdx.x / cp.col_blocks) * cp.slots + slot;
  const uint64_t col = (uint64_t)(blockIdx.x % cp.col_blocks) * cp.tx + lane;
  if (slot >= cp.slots || chunk >= cp.chunks || col >= cp.dv) return;
  const uint64_t lo = chunk * cp.chunk, hi = min(lo + cp.chunk, a.n);
  const TG* grad = (const TG*)a.grad + col * V;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; k++) acc[k] = 0.0f;
  uint32_t run = key_of(pairs[lo]);
  bool before = lo > 0 && key_of(pairs[lo - 1]) == run;

  auto flush = [&](bool after) {
    if (run >= a.vocab) return;
    if (before || after) {
      float* p = partial + (chunk * 2 + (before ? 0 : 1)) * cp.pitch + col * V;
      Pack<float, V> out;
#pragma unroll
      for (int k = 0; k < V; k++) out.v[k] = acc[k];
      out.store(p);
    } else {
      TD* p = dtable + run * a.ld_dtable + col * V;
      Pack<TD, V> out;
      if (a.accumulate) out.load(p);
#pragma unroll
      for (int k = 0; k < V; k++)
        out.set(k, a.accumulate ? out.get(k) + acc[k] * a.scale : acc[k] * a.scale);
      out.store(p);
    }
  };

  for (uint64_t j = lo; j < hi; j += kSumDepth) {
    unsigned long long pair[kSumDepth];
    Pack<TG, V> row[kSumDepth];
#pragma unroll
    for (int u = 0; u < kSumDepth; u++) pair[u] = j + u < hi ? pairs[j + u] : ~0ull;
#pragma unroll
    for (int u = 0; u < kSumDepth; u++)
      if (key_of(pair[u]) < a.vocab) row[u].load(grad + (uint64_t)(uint32_t)pair[u] * a.ld_grad);
#pragma unroll
    for (int u = 0; u < kSumDepth; u++) {
      if (j + u >= hi) break;
      const uint32_t key = key_of(pair[u]);
      if (key != run) {
        flush(false);
        run = key;
        before = false;
#pragma unroll
        for (int k = 0; k < V; k++) acc[k] = 0.0f;
      }
      if (key < a.vocab) {
#pragma unroll
        for (int k = 0; k < V; k++) acc[k] += row[u].get(k);
      }
    }
  }
  flush(hi < a.n && key_of(pairs[hi]) == run);
}

// Adds the partial sums of the runs that cross chunks: CTA (x, y) takes the runs that start
// in chunks x, x + gridDim.x, .. and the columns of block y. A run of a few chunks is one
// warp's, a longer one is shared by all warps and their sums are added in order.
template <typename TD>
__global__ void __launch_bounds__(kJoinThreads)
    k_embed_join(EmbedGradLaunch a, ChunkPlan cp, const unsigned long long* __restrict__ pairs,
                 const float* __restrict__ partial) {
  constexpr int kWarps = kJoinThreads / 32;
  constexpr uint32_t kLong = 24;  // chunks from which on a run is shared by the warps
  __shared__ uint32_t s_first[kJoinThreads], s_last[kJoinThreads];
  __shared__ uint32_t s_count;
  __shared__ float4 s_part[kWarps][32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t col = (uint64_t)blockIdx.y * kJoinCols + lane * 4;
  TD* dtable = (TD*)a.dtable;
  rw_dependent_start();

  auto row_sum = [&](uint32_t first, uint32_t lo, uint32_t hi) {
    // partials lo..hi-1 of the run that starts in chunk `first`, in order
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < cp.pitch) {
#pragma unroll 8
      for (uint32_t q = lo; q < hi; q++) {
        const float4 v = *(const float4*)(partial + ((uint64_t)q * 2 + (q == first ? 1 : 0)) * cp.pitch + col);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
    }
    return s;
  };
  auto finish = [&](uint32_t first, float4 s) {
    const uint64_t end = min((uint64_t)(first + 1) * cp.chunk, a.n);
    TD* p = dtable + (uint64_t)key_of(pairs[end - 1]) * a.ld_dtable + col;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (col + k >= a.d) break;
      p[k] = rw_round<TD>(a.accumulate ? rw_widen(p[k]) + v[k] * a.scale : v[k] * a.scale);
    }
  };

  for (uint64_t base = 0; base < cp.chunks; base += (uint64_t)gridDim.x * kJoinThreads) {
    __syncthreads();
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    const uint64_t c = base + blockIdx.x + (uint64_t)threadIdx.x * gridDim.x;
    if (c + 1 < cp.chunks) {
      const uint64_t lo = c * cp.chunk, hi = lo + cp.chunk;
      const uint32_t key = key_of(pairs[hi - 1]);
      if (key < a.vocab && key_of(pairs[hi]) == key && (lo == 0 || key_of(pairs[lo - 1]) != key)) {
        // the last chunk that begins with this id: in growing steps, then by halving
        uint64_t in = c + 1, out = cp.chunks;
        for (uint64_t step = 1; in + step < out; step *= 2) {
          if (key_of(pairs[(in + step) * cp.chunk]) == key) in += step;
          else out = in + step;
        }
        while (out - in > 1) {
          const uint64_t mid = (in + out) / 2;
          if (key_of(pairs[mid * cp.chunk]) == key) in = mid;
          else out = mid;
        }
        const uint32_t at = atomicAdd(&s_count, 1u);  // the list's order does not matter
        s_first[at] = (uint32_t)c;
        s_last[at] = (uint32_t)in;
      }
    }
    __syncthreads();
    const uint32_t count = s_count;
    for (uint32_t k = warp; k < count; k += kWarps) {
      const uint32_t first = s_first[k], last = s_last[k];
      if (last - first < kLong) finish(first, row_sum(first, first, last + 1));
    }
    for (uint32_t k = 0; k < count; k++) {
      const uint32_t first = s_first[k], last = s_last[k];
      if (last - first < kLong) continue;
      const uint32_t m = last + 1 - first, per = (m + kWarps - 1) / kWarps;
      const uint32_t lo = min(m, warp * per), hi = min(m, lo + per);
      s_part[warp][lane] = row_sum(first, first + lo, first + hi);
      __syncthreads();
      if (warp == 0) {
        float4 s = s_part[0][lane];
        for (int w = 1; w < kWarps; w++) {
          const float4 v = s_part[w][lane];
          s.x += v.x;
          s.y += v.y;
          s.z += v.z;
          s.w += v.w;
        }
        finish(first, s);
      }
      __syncthreads();
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

// Sizes and workspace offsets of one gradient call. The workspace covers either vector
// width: it depends on n, d and vocab alone.
struct GradPlan {
  uint64_t part;
  uint32_t parts, passes;
  uint64_t pairs0, pairs1, counts, partial, bytes;  // offsets
};

// Chunks: enough for about 16 CTAs an SM where a row takes two warps or more, so that the
// longest one does not decide the time; for narrower rows 4, whose slots are many and whose
// runs then cross fewer chunks; no shorter than 8 positions (the partial sums would be more
// than a quarter of the traffic) and no more than 32768 (k_embed_join looks at each).
ChunkPlan chunk_plan(uint64_t n, uint64_t d, int V) {
  ChunkPlan c = {};
  c.dv = (d + V - 1) / V;
  c.tx = (uint32_t)std::min<uint64_t>(c.dv, kSumThreads);
  c.slots = kSumThreads / c.tx;
  c.col_blocks = (uint32_t)((c.dv + c.tx - 1) / c.tx);
  c.pitch = (d + 3) / 4 * 4;
  const uint64_t want = std::max<uint64_t>(1, (uint64_t)kSms * (c.tx >= 64 ? 16 : 4) * c.slots / c.col_blocks);
  const uint64_t most = std::min<uint64_t>(want, 32768);
  c.chunk = (uint32_t)std::max<uint64_t>(8, (n + most - 1) / most);
  c.chunks = (uint32_t)((n + c.chunk - 1) / c.chunk);
  c.sum_ctas = (c.chunks + c.slots - 1) / c.slots * c.col_blocks;
  return c;
}

GradPlan grad_plan(uint64_t n, uint64_t d, uint64_t vocab) {
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
  const uint64_t chunks =
      std::max({chunk_plan(n, d, 1).chunks, chunk_plan(n, d, 4).chunks, chunk_plan(n, d, 8).chunks});
  g.partial = take(chunks * 2 * ((d + 3) / 4 * 4) * 4);
  g.bytes = at;
  return g;
}

}  // namespace

uint64_t embed_grad_workspace(uint64_t n, uint64_t d, uint64_t vocab) {
  return n == 0 || d == 0 || vocab == 0 ? 0 : grad_plan(n, d, vocab).bytes;
}

cudaError_t launch_embed_grad(const EmbedGradLaunch& a, void* workspace, cudaStream_t s, int* nl) {
  if (a.d == 0 || a.vocab == 0) return cudaSuccess;
  cudaError_t e = cudaSuccess;
  if (a.n == 0) {
    if (a.accumulate) return cudaSuccess;
    *nl += 1;
    return rw_with_type(a.dtable_type, [&](auto td) {
      using TD = decltype(td);
      return rw_launch(k_zero_rows<TD>, dim3(grid_of(a.vocab, 8)), dim3(256), 0, s, false,
                       (TD*)a.dtable, a.vocab, a.d, a.ld_dtable);
    });
  }
  const GradPlan g = grad_plan(a.n, a.d, a.vocab);
  char* ws = (char*)workspace;
  unsigned long long* buf[2] = {(unsigned long long*)(ws + g.pairs0),
                                (unsigned long long*)(ws + g.pairs1)};
  const bool count = a.n <= kCountSort;
  if (count) {
    *nl += 1;
    e = rw_with_index(a.id_type, [&](auto id) {
      using ID = decltype(id);
      const uint32_t blocks = (uint32_t)((a.n * kCountShare + kCountThreads - 1) / kCountThreads);
      return rw_launch(k_token_rank<ID>, dim3(blocks), dim3(kCountThreads), 0, s, false,
                       (const ID*)a.ids, (uint32_t)a.n, (uint32_t)a.vocab, buf[0]);
    });
  }
  SortPass p = {};
  p.ids = a.ids;
  p.counts = (uint32_t*)(ws + g.counts);
  p.n = a.n;
  p.part = g.part;
  p.vocab = a.vocab;
  p.parts = g.parts;
  for (uint32_t i = 0; i < g.passes && !count && e == cudaSuccess; i++) {
    p.in = buf[(i + 1) & 1];
    p.out = buf[i & 1];
    p.shift = i * kRadixBits;
    *nl += 2;
    e = rw_with_index(a.id_type, [&](auto id) {
      using ID = decltype(id);
      const dim3 grid(g.parts), block(kSortThreads);
      cudaError_t r = i == 0 ? rw_launch(k_token_count<ID, true>, grid, block, 0, s, false, p)
                             : rw_launch(k_token_count<ID, false>, grid, block, 0, s, true, p);
      if (r != cudaSuccess) return r;
      return i == 0 ? rw_launch(k_token_scatter<ID, true>, grid, block, 0, s, true, p)
                    : rw_launch(k_token_scatter<ID, false>, grid, block, 0, s, true, p);
    });
  }
  if (e != cudaSuccess) return e;
  const unsigned long long* pairs = count ? buf[0] : buf[(g.passes + 1) & 1];
  float* partial = (float*)(ws + g.partial);
  *nl += 2;
  ChunkPlan cp = {};
  e = rw_with_type(a.grad_type, [&](auto tg) {
    return rw_with_type(a.dtable_type, [&](auto td) {
      using TG = decltype(tg);
      using TD = decltype(td);
      constexpr int kV = 16 / sizeof(TG);
      const bool wide = rw_packs(a.grad, a.n, a.d, a.ld_grad, sizeof(TG), kV) &&
                        rw_packs(a.dtable, a.vocab, a.d, a.ld_dtable, sizeof(TD), kV);
      cp = chunk_plan(a.n, a.d, wide ? kV : 1);
      const uint64_t zero = a.accumulate ? 0 : (a.vocab + kZeroRows - 1) / kZeroRows;
      const dim3 grid((uint32_t)(cp.sum_ctas + zero));
      return wide ? rw_launch(k_embed_chunks<TG, TD, kV>, grid, dim3(kSumThreads), 0, s, true, a, cp,
                              pairs, partial)
                  : rw_launch(k_embed_chunks<TG, TD, 1>, grid, dim3(kSumThreads), 0, s, true, a, cp,
                              pairs, partial);
    });
  });
  if (e != cudaSuccess) return e;
  const uint32_t cols = (uint32_t)((a.d + kJoinCols - 1) / kJoinCols);
  const uint32_t gx = std::max(1u, std::min(cp.chunks, (uint32_t)kSms * 4 / cols));
  return rw_with_type(a.dtable_type, [&](auto td) {
    return rw_launch(k_embed_join<decltype(td)>, dim3(gx, cols), dim3(kJoinThreads), 0, s, true, a,
                     cp, pairs, (const float*)partial);
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
