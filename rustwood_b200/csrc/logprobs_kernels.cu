// Class log-probabilities of margin rows, and their gradient: for a row x of margins,
// m = max x and d_j = scale * (x_j - m),
//
//   log_sum = log s,  s = sum_j e^{d_j}          lse     = scale * m + log_sum
//   logp_t  = d_t - log_sum                      entropy = log_sum - (sum_j e^{d_j} d_j) / s
//
// and the k largest margins (the lower index first among equal ones) with their logp.
// Both terms of the entropy have one sign, so it loses nothing to cancellation. A row whose
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
#include <math_constants.h>
#include <stdint.h>

#include <algorithm>

#include "rw_internal.cuh"
#include "rw_types.cuh"

namespace {

constexpr int kRowThreads = 256;
constexpr float kLowest = -1e30f;  // where d is cut: e^d is 0 there, and 0 * d stays 0

// The larger of two values, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Orders margins (NaN above +inf, -0 equal to +0), then lower indices first.
__device__ __forceinline__ unsigned long long rank_key(float x, uint32_t index) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t o = x != x ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
  return (unsigned long long)o << 32 | (0xffffffffu - index);
}

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* s_tmp, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_tmp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s_tmp[0];
  for (int w = 1; w < kRowThreads / 32; w++) v = f(v, s_tmp[w]);
  return v;
}

template <typename T, typename ID>
__global__ void __launch_bounds__(kRowThreads) k_logprobs(LogprobsLaunch a) {
  __shared__ float s_f[kRowThreads / 32];
  __shared__ unsigned long long s_k[kRowThreads / 32];
  for (uint64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
    const T* x = (const T*)a.x + i * a.ld_x;
    float m = -CUDART_INF_F;
    for (uint64_t j = threadIdx.x; j < a.classes; j += kRowThreads) m = max_nan(m, rw_widen(x[j]));
    m = block_reduce(m, s_f, max_nan);
    const bool dead = m == -CUDART_INF_F;
    const float base = dead ? 0.0f : m;
    float s = 0.0f, t = 0.0f;
    for (uint64_t j = threadIdx.x; j < a.classes; j += kRowThreads) {
      const float d = max_nan((rw_widen(x[j]) - base) * a.scale, kLowest);
      const float e = expf(d);
      s += e;
      t += e * d;
    }
    auto add = [](float p, float q) { return p + q; };
    s = block_reduce(s, s_f, add);
    t = block_reduce(t, s_f, add);
    const float log_sum = dead ? 0.0f : logf(s);
    if (threadIdx.x == 0) {
      if (a.row_max) a.row_max[i] = m;
      if (a.log_sum) a.log_sum[i] = log_sum;
      if (a.lse) a.lse[i] = a.scale * m + log_sum;
      if (a.entropy) a.entropy[i] = dead ? 0.0f : log_sum - t / s;
      if (a.logp) {
        const int64_t c = (int64_t)((const ID*)a.targets)[i];
        const bool in = c >= 0 && (uint64_t)c < a.classes;
        a.logp[i] = in ? (rw_widen(x[c]) - base) * a.scale - log_sum : 0.0f;
      }
    }
    unsigned long long last = ~0ull;
    for (uint32_t k = 0; k < a.top_k; k++) {
      unsigned long long best = 0;
      for (uint64_t j = threadIdx.x; j < a.classes; j += kRowThreads) {
        const unsigned long long key = rank_key(rw_widen(x[j]), (uint32_t)j);
        if ((k == 0 || key < last) && key > best) best = key;
      }
      best = last = block_reduce(best, s_k, [](unsigned long long p, unsigned long long q) {
        return p > q ? p : q;
      });
      if (threadIdx.x == 0) {
        const uint32_t j = 0xffffffffu - (uint32_t)best;
        if (a.top_index) a.top_index[i * a.top_k + k] = j;
        if (a.top_logp) a.top_logp[i * a.top_k + k] = (rw_widen(x[j]) - base) * a.scale - log_sum;
      }
    }
    __syncthreads();
  }
}

template <typename T, typename ID>
__global__ void __launch_bounds__(kRowThreads) k_logprobs_grad(LogprobsGradLaunch a) {
  for (uint64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
    const T* x = (const T*)a.x + i * a.ld_x;
    T* dx = (T*)a.dx + i * a.ld_dx;
    const float m = a.row_max[i], log_sum = a.log_sum[i];
    const bool dead = m == -CUDART_INF_F;
    int64_t c = a.targets ? (int64_t)((const ID*)a.targets)[i] : -1;
    if (c < 0 || (uint64_t)c >= a.classes) c = -1;
    const float g = c >= 0 ? a.grad_logp[i] : 0.0f;
    const float e = a.grad_entropy ? a.grad_entropy[i] : 0.0f;
    const float h = a.grad_entropy ? a.entropy[i] : 0.0f;
    for (uint64_t j = threadIdx.x; j < a.classes; j += kRowThreads) {
      const float lp = max_nan((rw_widen(x[j]) - m) * a.scale - log_sum, kLowest);
      const float p = expf(lp);
      float v = (int64_t)j == c ? g : 0.0f;
      v -= p * (g + e * (lp + h));
      dx[j] = rw_round<T>(dead ? 0.0f : v * a.scale);
    }
  }
}

uint32_t grid_of(uint64_t blocks, uint32_t per_sm) {
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(blocks, 148ull * per_sm));
}

}  // namespace

uint64_t logprobs_workspace(uint64_t, uint64_t, int, uint32_t) { return 0; }

cudaError_t launch_logprobs(const LogprobsLaunch& a, void*, cudaStream_t s, int* nl) {
  if (a.n == 0) return cudaSuccess;
  *nl += 1;
  return rw_with_type(a.type, [&](auto t) {
    return rw_with_index(a.target_type, [&](auto id) {
      return rw_launch(k_logprobs<decltype(t), decltype(id)>, dim3(grid_of(a.n, 8)),
                       dim3(kRowThreads), 0, s, false, a);
    });
  });
}

cudaError_t launch_logprobs_grad(const LogprobsGradLaunch& a, cudaStream_t s, int* nl) {
  if (a.n == 0 || a.classes == 0) return cudaSuccess;
  *nl += 1;
  return rw_with_type(a.type, [&](auto t) {
    return rw_with_index(a.target_type, [&](auto id) {
      return rw_launch(k_logprobs_grad<decltype(t), decltype(id)>, dim3(grid_of(a.n, 8)),
                       dim3(kRowThreads), 0, s, false, a);
    });
  });
}
