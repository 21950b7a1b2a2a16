// Embedding lookup, its gradient and dropout: the vector-valued side of the categorical
// columns (encode.cu looks up and sums one scalar per key).
//
//   lookup    out[i] = scale * table[ids[i]]
//   gradient  dtable[v] (+)= scale * sum over i with ids[i] = v of grad[i]
//   dropout   y[e] = keep(e) ? x[e] / (1 - p) : 0
//
// All three are bound by the bytes they move. An id outside the table is padding: a zero row,
// and no gradient.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "rw_internal.cuh"
#include "rw_types.cuh"

namespace {

constexpr int kSms = 148;

// =================================================================================
// lookup

// `tx` threads a row, V columns a thread and access; a thread takes R rows and C vectors of
// each at a time, all in flight, so that short rows have as much in flight as long ones. Every
// CTA takes slots * R rows and is done. 65536 x 4096 bf16: 129 us, 5.4 TB/s of the bytes that
// have to move; 136 us with a resident grid, 167 us with two vectors in flight. Odd widths of
// 16-bit rows go two bytes at a time (30000 x 2001 bf16 93 us, x 2002 40 us, x 2048 31 us).
constexpr int kEmbedThreads = 256;

struct EmbedPlan {
  uint32_t tx, slots;
  uint32_t dv;     // vectors a row
  uint32_t split;  // CTAs that share a row's columns
};

template <typename TI, typename TO, int V, int R, int C>
__global__ void __launch_bounds__(kEmbedThreads) k_embed(EmbedLaunch a, EmbedPlan ep) {
  const uint32_t slot = threadIdx.x / ep.tx, lane = threadIdx.x % ep.tx;
  if (slot >= ep.slots) return;
  const uint32_t step = ep.tx * ep.split;
  const uint32_t first = blockIdx.x % ep.split * ep.tx + lane;
  const uint64_t i0 = (uint64_t)(blockIdx.x / ep.split) * ep.slots * R + slot;
  int64_t id[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint64_t i = i0 + (uint64_t)r * ep.slots;
    id[r] = -1;
    if (i < a.n) id[r] = a.id_type == RW_I64 ? ((const int64_t*)a.ids)[i] : ((const int32_t*)a.ids)[i];
    if (id[r] >= 0 && (uint64_t)id[r] >= a.vocab) id[r] = -1;
  }
  for (uint32_t c = first; c < ep.dv; c += step * C) {
    Pack<TI, V> v[R][C];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const TI* row = (const TI*)a.table + (uint64_t)max(id[r], (int64_t)0) * a.ld_table;
#pragma unroll
      for (int u = 0; u < C; u++)
        if (id[r] >= 0 && c + u * step < ep.dv) v[r][u].load(row + (uint64_t)(c + u * step) * V);
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      const uint64_t i = i0 + (uint64_t)r * ep.slots;
      if (i >= a.n) break;
      TO* out = (TO*)a.out + i * a.ld_out;
#pragma unroll
      for (int u = 0; u < C; u++) {
        if (c + u * step >= ep.dv) break;
        Pack<TO, V> o;
#pragma unroll
        for (int k = 0; k < V; k++) o.set(k, id[r] >= 0 ? a.scale * v[r][u].get(k) : 0.0f);
        o.store_streaming(out + (uint64_t)(c + u * step) * V);
      }
    }
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
// every CTA derives its part's bases from the counts of all parts. 65536 ids of 128000: two
// passes, 22 us of chained latencies for 2 MB.

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

// Rows of zeros, as bytes: `unit`-byte stores (16, or the element's size) by `threads` threads.
struct ZeroRows {
  char* p;
  uint64_t rows, row_units, pitch;  // pitch in bytes
  uint32_t unit;
};
__device__ __forceinline__ void zero_units(const ZeroRows& z, uint64_t t, uint64_t threads) {
  auto put = [&](char* p) {
    if (z.unit == 16) __stcs((uint4*)p, make_uint4(0, 0, 0, 0));
    else if (z.unit == 4) *(uint32_t*)p = 0;
    else *(uint16_t*)p = 0;
  };
  if (z.rows == 1) {
    for (uint64_t c = t; c < z.row_units; c += threads) put(z.p + c * z.unit);
    return;
  }
  const uint64_t warp = t / 32, warps = threads / 32;  // a warp a row
  for (uint64_t r = warp; r < z.rows; r += warps)
    for (uint64_t c = t % 32; c < z.row_units; c += 32) put(z.p + r * z.pitch + c * z.unit);
}

// Short inputs are sorted by counting instead, in one launch: a position's place is the
// number of positions before it in the order (id, position). n * n comparisons: 2 us at
// n = 512, and at kCountSort still less than the radix sort's launches.
constexpr uint64_t kCountSort = 4096;
constexpr int kCountThreads = 256;
constexpr int kCountShare = 8;  // threads that share a position's comparisons

// The CTAs from `blocks` on zero the table meanwhile, when there is one to zero.
template <typename ID>
__global__ void __launch_bounds__(kCountThreads)
    k_token_rank(const ID* __restrict__ ids, uint32_t n, uint32_t vocab, unsigned long long* __restrict__ out,
                 uint32_t blocks, ZeroRows z) {
  __shared__ uint32_t s_key[kCountSort];
  if (blockIdx.x >= blocks) {
    zero_units(z, (uint64_t)(blockIdx.x - blocks) * kCountThreads + threadIdx.x,
               (uint64_t)(gridDim.x - blocks) * kCountThreads);
    return;
  }
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
// ids and the sizes. Rows that no id names are zeroed by further CTAs of the same launch.
// 65536 x 4096 bf16 into 128000 rows f32: 438 us for 2.6 GB, 5.9 TB/s; 473 us with the sort
// and the join. Four CTAs an SM, as its launch bounds ask for, against the three that 78 registers
// leave: 36548 x 1128 bf16 into 8 rows 50 us and 54 us, 200000 x 1024 into 100 119 us and 127 us.

constexpr int kSumThreads = 256;
constexpr int kSumDepth = 4;    // rows in flight per thread
constexpr int kZeroRows = 128;  // the most table rows a zeroing CTA covers
constexpr int kJoinThreads = 512;
constexpr int kJoinCols = 128;  // columns of one join (a float4 a lane)

struct ChunkPlan {
  uint32_t chunk;       // positions a chunk
  uint32_t chunks;
  uint32_t tx, slots;   // threads a slot, slots a CTA
  uint32_t col_blocks;  // CTAs that share a chunk group's columns
  uint32_t sum_ctas;    // CTAs that sum; the rest zero rows that no id names
  uint64_t dv;          // vectors a row
  uint64_t pitch;       // floats of one partial row (a multiple of 4)
  uint32_t zero_rows;   // table rows a zeroing CTA covers
  uint32_t join_lanes;  // lanes of k_embed_join for a row: a power of two
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
__global__ void __launch_bounds__(kSumThreads, V * sizeof(TG) >= 16 ? 4 : 1)
    k_embed_chunks(EmbedGradLaunch a, ChunkPlan cp, const unsigned long long* __restrict__ pairs,
                   float* __restrict__ partial, uint2* __restrict__ ends) {
  const uint32_t slot = threadIdx.x / cp.tx, lane = threadIdx.x % cp.tx;
  TD* dtable = (TD*)a.dtable;
  rw_dependent_start();
  if (blockIdx.x >= cp.sum_ctas) {  // zero the rows of this block that no id names
    __shared__ bool s_absent[kZeroRows];
    const uint64_t first = (uint64_t)(blockIdx.x - cp.sum_ctas) * cp.zero_rows;
    if (threadIdx.x < cp.zero_rows && first + threadIdx.x < a.vocab) {
      const uint32_t key = (uint32_t)(first + threadIdx.x);
      const uint64_t at = lower_bound(pairs, a.n, key);
      s_absent[threadIdx.x] = at == a.n || key_of(pairs[at]) != key;
    }
    __syncthreads();
    if (slot >= cp.slots) return;
    Pack<TD, V> zero;
#pragma unroll
    for (int k = 0; k < V; k++) zero.set(k, 0.0f);
    for (uint64_t r = slot; r < cp.zero_rows && first + r < a.vocab; r += cp.slots) {
      if (!s_absent[r]) continue;
      TD* row = dtable + (first + r) * a.ld_dtable;
      for (uint64_t c = lane; c < cp.dv; c += cp.tx) zero.store_streaming(row + c * V);
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

  // the next round's pairs are on their way while this round's rows are
  unsigned long long next[kSumDepth];
#pragma unroll
  for (int u = 0; u < kSumDepth; u++) next[u] = lo + u < hi ? pairs[lo + u] : ~0ull;
  for (uint64_t j = lo; j < hi; j += kSumDepth) {
    unsigned long long pair[kSumDepth];
    Pack<TG, V> row[kSumDepth];
#pragma unroll
    for (int u = 0; u < kSumDepth; u++) pair[u] = next[u];
#pragma unroll
    for (int u = 0; u < kSumDepth; u++)
      if (key_of(pair[u]) < a.vocab) row[u].load(grad + (uint64_t)(uint32_t)pair[u] * a.ld_grad);
#pragma unroll
    for (int u = 0; u < kSumDepth; u++) next[u] = j + kSumDepth + u < hi ? pairs[j + kSumDepth + u] : ~0ull;
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
  if (col == 0) ends[chunk] = make_uint2(key_of(pairs[lo]), key_of(pairs[hi - 1]));
}

// Adds the partial sums of the runs that cross chunks: CTA (x, y) takes the runs that start
// in chunks x, x + gridDim.x, .. and the columns of block y. A run of a few chunks is one
// warp's, a longer one is shared by all warps and their sums are added in order. Where a row
// has fewer than 32 float4s, groups of lanes take every 2nd, 4th, .. chunk.
template <typename TD>
__global__ void __launch_bounds__(kJoinThreads)
    k_embed_join(EmbedGradLaunch a, ChunkPlan cp, const float* __restrict__ partial,
                 const uint2* __restrict__ ends) {  // a chunk's first and last id
  constexpr int kWarps = kJoinThreads / 32;
  // Chunks from which on a run is shared by the warps (24: 500000 x 64 f32 into 50000 rows 111 us
  // instead of 103 us, 60000 x 502 bf16 into 30000 78 us instead of 75 us).
  constexpr uint32_t kLong = 12;
  __shared__ uint32_t s_first[kJoinThreads], s_shared[kJoinThreads];  // runs; those all warps share
  __shared__ uint32_t s_count, s_long;
  __shared__ float4 s_part[kWarps][32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t width = cp.join_lanes, groups = 32 / width, group = lane / width;
  const uint64_t col = (uint64_t)blockIdx.y * kJoinCols + lane % width * 4;
  TD* dtable = (TD*)a.dtable;
  rw_dependent_start();

  auto row_sum = [&](uint32_t first, uint32_t lo, uint32_t hi) {
    // partials lo..hi-1 of the run that starts in chunk `first`, in order
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < cp.pitch) {
#pragma unroll 8
      for (uint32_t q = lo + group; q < hi; q += groups) {
        const float4 v = *(const float4*)(partial + ((uint64_t)q * 2 + (q == first ? 1 : 0)) * cp.pitch + col);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
    }
    for (uint32_t o = width; o < 32; o *= 2) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
      s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
      s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
    }
    return s;
  };
  auto finish = [&](uint32_t first, float4 s) {
    if (group != 0) return;
    TD* p = dtable + (uint64_t)ends[first].y * a.ld_dtable + col;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (col + k >= a.d) break;
      p[k] = rw_round<TD>(a.accumulate ? rw_widen(p[k]) + v[k] * a.scale : v[k] * a.scale);
    }
  };

  // The last chunk of the run that starts in chunk `first`, by a warp: 32 probes at a time, at
  // doubling distances and then evenly spaced.
  auto last_of = [&](uint32_t first) {
    const uint32_t key = ends[first].y;
    auto probe = [&](uint64_t q) {  // the number of lanes whose chunk begins with the run's id
      return (uint32_t)__popc(__ballot_sync(0xffffffffu, q < cp.chunks && ends[q].x == key));
    };
    uint32_t step = 1u << (probe((uint64_t)first + (1u << min(lane, 20u))) - 1);  // chunk first + 1 does
    uint64_t last = (uint64_t)first + step;
    while (step > 1) {  // the end is less than `step` chunks on
      step = (step + 31) / 32;
      last += (uint64_t)step * probe(last + (uint64_t)step * (lane + 1));
    }
    return (uint32_t)last;
  };

  for (uint64_t base = 0; base < cp.chunks; base += (uint64_t)gridDim.x * kJoinThreads) {
    __syncthreads();
    if (threadIdx.x == 0) s_count = s_long = 0;
    __syncthreads();
    const uint64_t c = base + blockIdx.x + (uint64_t)threadIdx.x * gridDim.x;
    if (c + 1 < cp.chunks) {
      const uint32_t key = ends[c].y;
      if (key < a.vocab && ends[c + 1].x == key && (c == 0 || ends[c - 1].y != key))
        s_first[atomicAdd(&s_count, 1u)] = (uint32_t)c;  // the list's order does not matter
    }
    __syncthreads();
    const uint32_t count = s_count;
    for (uint32_t k = warp; k < count; k += kWarps) {
      const uint32_t first = s_first[k], last = last_of(first);
      if (last - first < kLong) finish(first, row_sum(first, first, last + 1));
      else if (lane == 0) s_shared[atomicAdd(&s_long, 1u)] = first;
    }
    __syncthreads();
    for (uint32_t k = 0; k < s_long; k++) {
      const uint32_t first = s_shared[k], last = last_of(first);
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

// Few, narrow table rows (a categorical column) need no sort: a slot of d threads keeps a
// whole table of sums in shared memory, one column a thread, so no two threads share a sum
// and the order is fixed (a sum of no rows stays at its start, -0). The CTA streams its part
// of grad once, in memory order, through a ring of tiles in shared memory that asynchronous
// copies fill; a ninth warp turns the ids into offsets, so that a sum is two loads, an
// addition and a store. 1000003 x 33 f32 into 50 rows: 42 us, the shared-memory pipe busy for
// three quarters of it; 51 us with loads to registers, 130 us by sorting, whose walk reads
// rows of 132 bytes in category order. grad has to be contiguous and aligned. 300000 x 16 f32
// into 64 rows: 12 us, 55 us by sorting; 100000 x 256 bf16 into 30: 29 us and 45 us; 2000 x 16
// into 50: 6 us and 12 us. 64 rows is where shared memory is still cheap, not where the two
// meet: with 96, 1000003 x 33 f32 would take 60 us here and 129 us sorted, but 100000 x 256 bf16
// 45 us here and 42 us sorted.
constexpr uint32_t kTableRows = 64;
constexpr uint32_t kTableCols = kSumThreads;
constexpr int kTableStages = 4;
constexpr int kTableThreads = kSumThreads + 32;  // eight warps that copy and add, one for the ids
constexpr int kTableJoinThreads = 1024;
// the most that a plan asks for: 256 columns of 65 rows; tiles of 8 KB and 2048 ids (d = 1) in every
// stage, and the rows' offsets
constexpr int kTableSmem =
    (int)((kTableRows + 1) * kTableCols * 4 + kTableStages * (kTableCols * 32 + kTableCols * 8 * 8) +
          2 * kTableCols * 8 * 4);
static_assert(kTableSmem <= 227 * 1024, "fits a CTA");

struct TablePlan {
  uint32_t slots, ctas;
  uint32_t tile;        // positions a tile: eight a slot, so tiles start on 16 bytes
  uint32_t tile_bytes;  // of grad, a multiple of 16
  uint64_t part;        // positions a CTA, a multiple of tile
  size_t tables, smem;  // bytes
};

__device__ __forceinline__ void copy_async16(uint32_t to, const void* from, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
template <int B>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(B) : "memory");
}

template <typename TG, typename ID>
__global__ void __launch_bounds__(kTableThreads)
    k_embed_table(EmbedGradLaunch a, TablePlan tp, float* __restrict__ partial) {
  extern __shared__ __align__(16) char s_mem[];
  float* s_table = (float*)s_mem;               // [slots][vocab + 1][d]
  char* s_grad = s_mem + tp.tables;             // [stages][tile_bytes]
  ID* s_id = (ID*)(s_grad + kTableStages * tp.tile_bytes);       // [stages][tile]
  uint32_t* s_row = (uint32_t*)(s_id + kTableStages * tp.tile);  // [2][tile]: ids as offsets of rows
  const uint32_t t = threadIdx.x, d = (uint32_t)a.d, vocab = (uint32_t)a.vocab, cells = vocab * d;
  const uint64_t lo = (uint64_t)blockIdx.x * tp.part;
  const uint32_t count = (uint32_t)min(tp.part, a.n - lo);  // lo < n
  const uint32_t tiles = (count + tp.tile - 1) / tp.tile;

  const uint32_t at_grad = (uint32_t)__cvta_generic_to_shared(s_grad);
  // One group of copies a tile and thread (an empty one past the last tile). After done(),
  // this thread's copies of the tile after the current one have landed; the barrier that
  // follows shows them to all.
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  auto done = [] { asm volatile("cp.async.wait_group %0;" ::"n"(kTableStages - 2) : "memory"); };

  if (t >= kSumThreads) {  // the warp of the ids
    const uint32_t lane = t - kSumThreads;
    const ID* ids = (const ID*)a.ids + lo;
    const uint32_t at_id = (uint32_t)__cvta_generic_to_shared(s_id);
    auto fetch = [&](uint32_t tile) {
      const uint32_t first = tile * tp.tile, to = tile % kTableStages * tp.tile;
      if (tile < tiles)
        for (uint32_t q = lane; q < tp.tile && first + q < count; q += 32)
          copy_async<sizeof(ID)>(at_id + (to + q) * (uint32_t)sizeof(ID), ids + first + q);
      commit();
    };
    // ids outside the table, and places past the end, add to its last row, which is not read;
    // a lane reads the ids that it copied
    auto offsets = [&](uint32_t tile) {
      done();
      if (tile >= tiles) return;
      const ID* id = s_id + tile % kTableStages * tp.tile;
      uint32_t* row = s_row + tile % 2 * tp.tile;
      const uint32_t rows = min(tp.tile, count - tile * tp.tile);
      for (uint32_t q = lane; q < tp.tile; q += 32) {
        const ID key = q < rows ? id[q] : (ID)-1;
        row[q] = (key >= 0 && key < (ID)vocab ? (uint32_t)key : vocab) * d;
      }
    };
#pragma unroll
    for (int k = 0; k < kTableStages - 1; k++) fetch(k);
    offsets(0);
    __syncthreads();
    for (uint32_t tile = 0; tile < tiles; tile++) {
      fetch(tile + kTableStages - 1);  // into the stage of the tile before, which is done with
      offsets(tile + 1);
      __syncthreads();
    }
    return;
  }

  // a thread copies bytes 16 t .. of every 4 KB of a tile (at most 8 KB)
  const char* from = (const char*)((const TG*)a.grad + lo * d) + t * 16;
  uint64_t left = (uint64_t)count * d * sizeof(TG);  // bytes of this and later tiles
  uint32_t stage = 0;
  auto fetch = [&] {
#pragma unroll
    for (uint32_t b = 0; b < 2; b++) {
      const uint32_t at = t * 16 + b * kSumThreads * 16;
      if (at < tp.tile_bytes && at < left)
        copy_async16(at_grad + stage * tp.tile_bytes + at, from + b * kSumThreads * 16,
                     (uint32_t)min((uint64_t)16, left - at));
    }
    from += tp.tile_bytes;
    left = left > tp.tile_bytes ? left - tp.tile_bytes : 0;
    stage = stage + 1 == kTableStages ? 0 : stage + 1;
    commit();
  };
#pragma unroll
  for (int k = 0; k < kTableStages - 1; k++) fetch();
  const uint32_t slot = t / d, col = t % d, step = tp.slots * d;
  const bool mine = slot < tp.slots;
  float* table = s_table + slot * (cells + d) + col;
  if (mine)
    for (uint32_t v = 0; v <= vocab; v++) table[v * d] = -0.0f;
  done();
  __syncthreads();
  for (uint32_t tile = 0; tile < tiles; tile++) {
    fetch();
    if (mine) {
      const TG* g = (const TG*)(s_grad + tile % kTableStages * tp.tile_bytes) + slot * d + col;
      const uint32_t* row = s_row + tile % 2 * tp.tile + slot;
      uint32_t to[8];
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; u++) {  // a tile is eight positions a slot
        to[u] = row[u * tp.slots];
        v[u] = rw_widen(g[u * step]);
      }
#pragma unroll
      for (int u = 0; u < 8; u++) table[to[u]] += v[u];
    }
    done();
    __syncthreads();
  }
  // the last barrier above came after every sum
  for (uint32_t c = t; c < cells; c += kSumThreads) {
    float s = s_table[c];
    for (uint32_t k = 1; k < tp.slots; k++) s += s_table[k * (cells + d) + c];
    partial[(uint64_t)blockIdx.x * cells + c] = s;
  }
}

// dtable from the CTAs' tables: 32 cells a CTA, the tables shared by its warps in order.
template <typename TD>
__global__ void __launch_bounds__(kTableJoinThreads)
    k_embed_table_join(EmbedGradLaunch a, uint32_t tables, const float* __restrict__ partial) {
  constexpr int kWarps = kTableJoinThreads / 32;
  __shared__ float s_part[kWarps][32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cells = (uint32_t)(a.vocab * a.d), c = blockIdx.x * 32 + lane;
  rw_dependent_start();
  const uint32_t per = (tables + kWarps - 1) / kWarps;
  const uint32_t lo = min(tables, warp * per), hi = min(tables, lo + per);
  float s = -0.0f;
  if (c < cells) {
#pragma unroll 8
    for (uint32_t t = lo; t < hi; t++) s += partial[(uint64_t)t * cells + c];
  }
  s_part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= cells) return;
  for (int w = 1; w < kWarps; w++) s += s_part[w][lane];
  const uint32_t v = c / (uint32_t)a.d;
  TD* p = (TD*)a.dtable + v * a.ld_dtable + (c - v * (uint32_t)a.d);
  // -0 is the sum of no rows (or of -0 alone): nothing to add, whatever the scale is
  const bool none = __float_as_uint(s) == 0x80000000u;
  if (!a.accumulate) *p = rw_round<TD>(none ? 0.0f : s * a.scale);
  else if (!none) *p = rw_round<TD>(rw_widen(*p) + s * a.scale);
}

__global__ void __launch_bounds__(kCountThreads) k_zero_rows(ZeroRows z) {
  zero_units(z, (uint64_t)blockIdx.x * kCountThreads + threadIdx.x, (uint64_t)gridDim.x * kCountThreads);
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

// The generator's ten round keys are the same for all: computed once on the host.
struct PhiloxKeys {
  uint32_t k0[10], k1[10];
};

__device__ __forceinline__ Words philox(uint64_t group, uint64_t sequence, const PhiloxKeys& k) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32);
  uint32_t c2 = (uint32_t)sequence, c3 = (uint32_t)(sequence >> 32);
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k.k0[r];
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k.k1[r];
    c3 = (uint32_t)a;
  }
  return {{c0, c1, c2, c3}};
}

// high_limit = limit << 16: the other half of the word does not change the comparison.
__device__ __forceinline__ bool dropout_keep(const Words& w, int k, uint32_t high_limit) {
  return (k & 1 ? w.w[k / 2] : w.w[k / 2] << 16) >= high_limit;
}

constexpr int kDropoutCtas = 5;
template <typename T>
constexpr int kDropoutDepth = 8 / (int)sizeof(T);  // 64 bytes

// One thread takes the 8 elements of a counter, kDropoutDepth counters whose loads are all in
// flight before it computes, and is done: many short CTAs overlap better than a resident grid
// that walks the matrix with as many loads in flight (268M bf16: 182 us, 5.9 TB/s, against
// 209-221 us). VEC: the matrices are contiguous and 16-byte aligned, so a group is one or two
// 16-byte accesses; the last, partial one goes element by element. Other layouts do throughout:
// 65536 x 1024 bf16 45 us contiguous, 231 us strided.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, kDropoutCtas) k_dropout(DropoutLaunch a, PhiloxKeys keys) {
  const uint64_t total = a.rows * a.cols;
  const uint32_t limit = a.limit << 16;  // p = 1 does not come here
  const T* x = (const T*)a.x;
  T* y = (T*)a.y;
  const uint64_t t = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const uint64_t threads = (uint64_t)gridDim.x * blockDim.x;
  constexpr int kDepth = kDropoutDepth<T>;
  if (VEC) {
    const uint64_t whole = total / 8;
    const uint64_t first = (uint64_t)blockIdx.x * (256 * kDepth) + threadIdx.x;
    Pack<T, 8> v[kDepth];
#pragma unroll
    for (int b = 0; b < kDepth; b++)
      if (first + b * 256 < whole) v[b].load(x + (first + b * 256) * 8);
#pragma unroll
    for (int b = 0; b < kDepth; b++) {
      const uint64_t g = first + b * 256;
      if (g >= whole) break;
      const Words w = philox(g, a.sequence, keys);
#pragma unroll
      for (int k = 0; k < 8; k++)
        v[b].set(k, dropout_keep(w, k, limit) ? v[b].get(k) * a.scale : 0.0f);
      v[b].store_streaming(y + g * 8);
    }
    if (t == 0 && whole * 8 < total) {
      const Words w = philox(whole, a.sequence, keys);
#pragma unroll
      for (int k = 0; k < 7; k++) {
        const uint64_t e = whole * 8 + k;
        if (e < total) y[e] = rw_round<T>(dropout_keep(w, k, limit) ? rw_widen(x[e]) * a.scale : 0.0f);
      }
    }
    return;
  }
  for (uint64_t g = t; g * 8 < total; g += threads) {
    const Words w = philox(g, a.sequence, keys);
    uint64_t r = g * 8 / a.cols, c = g * 8 - r * a.cols;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      if (g * 8 + k >= total) break;
      y[r * a.ld_y + c] =
          rw_round<T>(dropout_keep(w, k, limit) ? rw_widen(x[r * a.ld_x + c]) * a.scale : 0.0f);
      if (++c == a.cols) {
        c = 0;
        r++;
      }
    }
  }
}

uint32_t grid_of(uint64_t blocks, uint32_t per_sm) {
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(blocks, (uint64_t)kSms * per_sm));
}

template <typename TI, typename TO, int V>
cudaError_t embed_launch(const EmbedLaunch& a, cudaStream_t s) {
  EmbedPlan ep;
  ep.dv = (uint32_t)(a.d / V);
  // few rows: a vector a thread, a row's columns over several CTAs; many: four a thread, of one
  // row where a row has four warps' worth, else of two or four rows. Rows of 256 bf16, few and
  // many: 600 of them 2.0 us and 2.5 us; of 4096: 2400 of them 9.1 us and 8.2 us.
  const bool many = a.n >= 8 * kSms;
  const uint32_t warps = (ep.dv + 31) / 32;
  int c = !many ? 1 : warps >= 4 ? 4 : warps >= 2 ? 2 : 1;
  const int r = many ? 4 / c : 1;
  if (V <= 2 && c == 4 && warps >= 8) c = 8;  // narrow loads: more of them
  uint64_t tx = ep.dv;
  if (c > 1) tx = ((ep.dv + c - 1) / c + 31) / 32 * 32;
  ep.tx = (uint32_t)std::min<uint64_t>(tx, kEmbedThreads);
  ep.slots = kEmbedThreads / ep.tx;
  const uint64_t groups = (a.n + ep.slots * r - 1) / (ep.slots * r);
  const uint64_t most = (ep.dv + ep.tx - 1) / ep.tx;
  ep.split = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(most, 2 * kSms / groups));
  if (groups * ep.split > 0x7fffffffull) return cudaErrorInvalidValue;
  const dim3 grid((uint32_t)(groups * ep.split)), block(kEmbedThreads);
  if constexpr (V <= 2)
    if (c == 8) return rw_launch(k_embed<TI, TO, V, 1, 8>, grid, block, 0, s, false, a, ep);
  if (c == 4) return rw_launch(k_embed<TI, TO, V, 1, 4>, grid, block, 0, s, false, a, ep);
  if (c == 2) return rw_launch(k_embed<TI, TO, V, 2, 2>, grid, block, 0, s, false, a, ep);
  return many ? rw_launch(k_embed<TI, TO, V, 4, 1>, grid, block, 0, s, false, a, ep)
              : rw_launch(k_embed<TI, TO, V, 1, 1>, grid, block, 0, s, false, a, ep);
}

}  // namespace

cudaError_t launch_embed(const EmbedLaunch& a, cudaStream_t s, int* nl) {
  if (a.n == 0 || a.d == 0) return cudaSuccess;
  *nl += 1;
  return rw_with_type(a.table_type, [&](auto ti) {
    return rw_with_type(a.out_type, [&](auto to) {
      using TI = decltype(ti);
      using TO = decltype(to);
      constexpr int kV = 16 / sizeof(TI);
      auto packs = [&](int V) {
        return rw_packs(a.table, a.vocab, a.d, a.ld_table, sizeof(TI), V) &&
               rw_packs(a.out, a.n, a.d, a.ld_out, sizeof(TO), V);
      };
      return packs(kV) ? embed_launch<TI, TO, kV>(a, s)
             : packs(2) ? embed_launch<TI, TO, 2>(a, s) : embed_launch<TI, TO, 1>(a, s);
    });
  });
}

namespace {

// Sizes and workspace offsets of one gradient call. The workspace covers every type and
// layout: it depends on n, d and vocab alone.
struct GradPlan {
  uint64_t part;
  uint32_t parts, passes;
  uint64_t pairs0, pairs1, counts, partial, ends, bytes;  // offsets
};

// How a row's d columns, V a thread, lie on CTAs.
void chunk_columns(ChunkPlan& c, uint64_t d, int V) {
  c.dv = (d + V - 1) / V;
  c.tx = (uint32_t)std::min<uint64_t>(c.dv, kSumThreads);
  c.slots = kSumThreads / c.tx;
  c.col_blocks = (uint32_t)((c.dv + c.tx - 1) / c.tx);
}

// The columns a thread takes where no stride or base stands in the way: a 16-byte vector of
// `elem`-byte elements, or what the width allows.
int widest(uint64_t d, size_t elem) {
  const int v = 16 / (int)elem;
  return d % v == 0 ? v : d % 2 == 0 ? 2 : 1;
}

// Chunks: enough for about 10 CTAs an SM where a row takes two warps or more, so that the
// longest one does not decide the time (16: 36548 x 1128 bf16 into 8 rows 59 us instead of 50 us,
// 65536 x 4096 bf16 into 128000 481 us instead of 475 us, f32 498 us instead of 506 us); for
// narrower rows 4, whose slots are many and whose runs then cross fewer chunks; no shorter than
// 8 positions (the partial sums would be more than a quarter of the traffic) and no more than
// 32768 (k_embed_join looks at each). Their length follows n, d and the type's widest vectors,
// not the V that strides and bases leave, so that the order of the sums does not depend on the
// layout.
ChunkPlan chunk_plan(uint64_t n, uint64_t d, size_t elem, int V) {
  ChunkPlan c = {};
  chunk_columns(c, d, widest(d, elem));
  const uint64_t want = std::max<uint64_t>(1, (uint64_t)kSms * (c.tx >= 64 ? 10 : 4) * c.slots / c.col_blocks);
  chunk_columns(c, d, V);
  c.pitch = (d + 3) / 4 * 4;
  c.join_lanes = 1;
  while (c.join_lanes < 32 && c.join_lanes * 4 < d) c.join_lanes *= 2;
  const uint64_t most = std::min<uint64_t>(want, 32768);
  c.chunk = (uint32_t)std::max<uint64_t>(8, (n + most - 1) / most);
  c.chunks = (uint32_t)((n + c.chunk - 1) / c.chunk);
  c.sum_ctas = (c.chunks + c.slots - 1) / c.slots * c.col_blocks;
  return c;
}

// The table path's sizes; whether it is taken also depends on grad's alignment.
bool table_fits(uint64_t d, uint64_t vocab) { return d <= kTableCols && vocab <= kTableRows; }

TablePlan table_plan(uint64_t n, uint64_t d, uint64_t vocab, size_t elem, size_t id) {
  TablePlan t;
  t.slots = (uint32_t)(kTableCols / d);
  t.tables = ((size_t)t.slots * (vocab + 1) * d * 4 + 15) / 16 * 16;
  t.tile = t.slots * 8;  // up to 4 or 8 KB
  t.tile_bytes = (uint32_t)(t.tile * d * elem);
  t.smem = t.tables + kTableStages * (t.tile_bytes + t.tile * id) + 2 * t.tile * 4;
  const uint64_t per_sm = std::max<uint64_t>(1, std::min<uint64_t>(4, (220u << 10) / (t.smem + 1024)));
  // as many CTAs as fit at once, of kTableStages tiles at least
  const uint64_t tiles = (n + t.tile - 1) / t.tile;
  const uint64_t ctas = std::max<uint64_t>(1, std::min<uint64_t>(kSms * per_sm, tiles / kTableStages));
  t.part = (tiles + ctas - 1) / ctas * t.tile;
  t.ctas = (uint32_t)((n + t.part - 1) / t.part);
  return t;
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
  // they do not depend on V
  const uint64_t chunks = std::max(chunk_plan(n, d, 2, 1).chunks, chunk_plan(n, d, 4, 1).chunks);
  g.partial = take(chunks * 2 * ((d + 3) / 4 * 4) * 4);
  g.ends = take(chunks * sizeof(uint2));
  // the table path keeps its CTAs' tables there instead
  if (table_fits(d, vocab))
    for (size_t elem : {2, 4})
      for (size_t id : {4, 8})
        at = std::max<uint64_t>(at, table_plan(n, d, vocab, elem, id).ctas * vocab * d * 4);
  g.bytes = at;
  return g;
}

ZeroRows zero_rows(void* p, uint64_t rows, uint64_t cols, uint64_t ld, uint64_t elem) {
  const uint64_t pitch = ld * elem;
  ZeroRows z = {(char*)p, rows, 0, pitch, (uint32_t)elem};
  uint64_t bytes = cols * elem;
  if (rows == 1 || ld == cols) {  // one run
    bytes *= rows;
    z.rows = 1;
  }
  if (bytes % 16 == 0 && (uintptr_t)p % 16 == 0 && (z.rows == 1 || pitch % 16 == 0)) z.unit = 16;
  z.row_units = bytes / z.unit;
  return z;
}
uint32_t zero_ctas(const ZeroRows& z) {
  return grid_of((z.rows * z.row_units + 4 * kCountThreads - 1) / (4 * kCountThreads), 8);
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
    const ZeroRows z = zero_rows(a.dtable, a.vocab, a.d, a.ld_dtable, rw_type_bytes(a.dtable_type));
    return rw_launch(k_zero_rows, dim3(zero_ctas(z)), dim3(kCountThreads), 0, s, false, z);
  }
  const GradPlan g = grad_plan(a.n, a.d, a.vocab);
  char* ws = (char*)workspace;
  if (table_fits(a.d, a.vocab) && (a.n == 1 || a.ld_grad == a.d) && (uintptr_t)a.grad % 16 == 0) {
    const TablePlan t = table_plan(a.n, a.d, a.vocab, rw_type_bytes(a.grad_type), a.id_type == RW_I64 ? 8 : 4);
    *nl += 2;
    e = rw_with_type(a.grad_type, [&](auto tg) {
      return rw_with_index(a.id_type, [&](auto id) {
        auto* k = k_embed_table<decltype(tg), decltype(id)>;
        cudaError_t r = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kTableSmem);
        if (r != cudaSuccess) return r;
        return rw_launch(k, dim3(t.ctas), dim3(kTableThreads), t.smem, s, false, a, t, (float*)ws);
      });
    });
    if (e != cudaSuccess) return e;
    return rw_with_type(a.dtable_type, [&](auto td) {
      return rw_launch(k_embed_table_join<decltype(td)>, dim3((uint32_t)((a.vocab * a.d + 31) / 32)),
                       dim3(kTableJoinThreads), 0, s, true, a, t.ctas, (const float*)ws);
    });
  }
  unsigned long long* buf[2] = {(unsigned long long*)(ws + g.pairs0),
                                (unsigned long long*)(ws + g.pairs1)};
  const bool count = a.n <= kCountSort;
  // Few ids, many rows: the whole table is zeroed beside the sort and the rows that ids name
  // are written again, instead of looking for each row among the ids (512 ids into 32000 x
  // 768: 30 -> 21 us).
  const bool zero_first = count && !a.accumulate && a.n <= a.vocab / 4;
  if (count) {
    *nl += 1;
    e = rw_with_index(a.id_type, [&](auto id) {
      using ID = decltype(id);
      const uint32_t blocks = (uint32_t)((a.n * kCountShare + kCountThreads - 1) / kCountThreads);
      const ZeroRows z = zero_rows(a.dtable, a.vocab, a.d, a.ld_dtable, rw_type_bytes(a.dtable_type));
      return rw_launch(k_token_rank<ID>, dim3(blocks + (zero_first ? zero_ctas(z) : 0)), dim3(kCountThreads),
                       0, s, false, (const ID*)a.ids, (uint32_t)a.n, (uint32_t)a.vocab, buf[0], blocks, z);
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
  uint2* ends = (uint2*)(ws + g.ends);
  *nl += 1;
  ChunkPlan cp = {};
  e = rw_with_type(a.grad_type, [&](auto tg) {
    return rw_with_type(a.dtable_type, [&](auto td) {
      using TG = decltype(tg);
      using TD = decltype(td);
      constexpr int kV = 16 / sizeof(TG);
      auto packs = [&](int V) {
        return rw_packs(a.grad, a.n, a.d, a.ld_grad, sizeof(TG), V) &&
               rw_packs(a.dtable, a.vocab, a.d, a.ld_dtable, sizeof(TD), V);
      };
      const int V = packs(kV) ? kV : packs(2) ? 2 : 1;
      cp = chunk_plan(a.n, a.d, sizeof(TG), V);
      // A zeroing CTA takes 128 KB, so that its search among the ids is a small part of it, or
      // more where that still leaves 32 an SM, so that the last ones do not decide the time.
      cp.zero_rows = (uint32_t)std::min<uint64_t>(
          kZeroRows, std::max<uint64_t>({4, a.vocab / (kSms * 32), (128u << 10) / (a.d * sizeof(TD))}));
      const uint64_t zero = a.accumulate || zero_first ? 0 : (a.vocab + cp.zero_rows - 1) / cp.zero_rows;
      const dim3 grid((uint32_t)(cp.sum_ctas + zero));
      auto* k = V == kV ? k_embed_chunks<TG, TD, kV> : V == 2 ? k_embed_chunks<TG, TD, 2> : k_embed_chunks<TG, TD, 1>;
      return rw_launch(k, grid, dim3(kSumThreads), 0, s, true, a, cp, pairs, partial, ends);
    });
  });
  if (e != cudaSuccess || cp.chunks == 1) return e;
  *nl += 1;
  const uint32_t cols = (uint32_t)((a.d + kJoinCols - 1) / kJoinCols);
  const uint32_t gx = std::max(1u, std::min(cp.chunks, (uint32_t)kSms * 4 / cols));
  return rw_with_type(a.dtable_type, [&](auto td) {
    return rw_launch(k_embed_join<decltype(td)>, dim3(gx, cols), dim3(kJoinThreads), 0, s, true, a,
                     cp, (const float*)partial, (const uint2*)ends);
  });
}

cudaError_t launch_dropout(const DropoutLaunch& a, cudaStream_t s, int* nl) {
  if (a.rows == 0 || a.cols == 0) return cudaSuccess;
  *nl += 1;
  if (a.limit >= 65536) {
    const ZeroRows z = zero_rows(a.y, a.rows, a.cols, a.ld_y, rw_type_bytes(a.type));
    return rw_launch(k_zero_rows, dim3(zero_ctas(z)), dim3(kCountThreads), 0, s, false, z);
  }
  const uint64_t groups = (a.rows * a.cols + 7) / 8;
  PhiloxKeys keys;
  for (uint32_t r = 0; r < 10; r++) {
    keys.k0[r] = (uint32_t)a.seed + r * 0x9E3779B9u;
    keys.k1[r] = (uint32_t)(a.seed >> 32) + r * 0xBB67AE85u;
  }
  const bool flat = a.rows == 1 || (a.ld_x == a.cols && a.ld_y == a.cols);
  const bool vec = flat && (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.y % 16 == 0;
  return rw_with_type(a.type, [&](auto t) {
    using T = decltype(t);
    constexpr uint64_t kPer = 256 * kDropoutDepth<T>;
    const uint64_t ctas = (groups + kPer - 1) / kPer;
    if (ctas > 0x7fffffffull) return cudaErrorInvalidValue;
    const dim3 grid(vec ? (uint32_t)ctas : grid_of((groups + 255) / 256, 8)), block(256);
    return vec ? rw_launch(k_dropout<T, true>, grid, block, 0, s, false, a, keys)
               : rw_launch(k_dropout<T, false>, grid, block, 0, s, false, a, keys);
  });
}
