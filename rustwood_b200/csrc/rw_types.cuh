// Element types of the token operators (embedding, dropout, class log-probabilities):
// loads that widen to f32 and stores that round once to the output's type.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <tuple>

#include "rw_internal.cuh"

__device__ __forceinline__ float rw_widen(float v) { return v; }
__device__ __forceinline__ float rw_widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float rw_widen(__half v) { return __half2float(v); }
// one rounding, to nearest even
template <typename T>
__device__ __forceinline__ T rw_round(float v);
template <>
__device__ __forceinline__ float rw_round<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 rw_round<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half rw_round<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements as they lie in memory, moved in pieces of at most 16 bytes; the
// address is a multiple of a piece.
template <typename T, int V>
struct Pack {
  static constexpr int kBytes = (int)sizeof(T) * V;
  static constexpr int kPiece = kBytes < 16 ? kBytes : 16;
  static constexpr int kPieces = kBytes / kPiece;
  union alignas(kPiece) {
    T v[V];
    uint4 q[kBytes >= 16 ? kPieces : 1];
    uint2 d;
    uint32_t w;
    uint16_t h;
  };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kPieces; i++) q[i] = ((const uint4*)p)[i];
    } else if constexpr (kBytes == 8) {
      d = *(const uint2*)p;
    } else if constexpr (kBytes == 4) {
      w = *(const uint32_t*)p;
    } else {
      h = *(const uint16_t*)p;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kPieces; i++) ((uint4*)p)[i] = q[i];
    } else if constexpr (kBytes == 8) {
      *(uint2*)p = d;
    } else if constexpr (kBytes == 4) {
      *(uint32_t*)p = w;
    } else {
      *(uint16_t*)p = h;
    }
  }
  // a store that does not displace what the L2 holds of the inputs
  __device__ __forceinline__ void store_streaming(T* p) const {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kPieces; i++) __stcs((uint4*)p + i, q[i]);
    } else {
      store(p);
    }
  }
  __device__ __forceinline__ float get(int i) const { return rw_widen(v[i]); }
  __device__ __forceinline__ void set(int i, float f) { v[i] = rw_round<T>(f); }
};

// Whether a matrix of `elem`-byte elements can be read V elements at a time.
inline bool rw_packs(const void* p, uint64_t rows, uint64_t cols, uint64_t ld, size_t elem, int V) {
  const size_t piece = std::min<size_t>(elem * V, 16);
  return cols % V == 0 && (uintptr_t)p % piece == 0 && (rows <= 1 || ld * elem % piece == 0);
}

inline size_t rw_type_bytes(int type) { return type == RW_F32 ? 4 : 2; }

// Calls f with a value of the element type `type` names.
template <typename F>
inline cudaError_t rw_with_type(int type, F f) {
  switch (type) {
    case RW_F32: return f(float{});
    case RW_BF16: return f(__nv_bfloat16{});
    case RW_F16: return f(__half{});
  }
  return cudaErrorInvalidValue;
}
// Calls f with a value of the index type `type` names.
template <typename F>
inline cudaError_t rw_with_index(int type, F f) {
  switch (type) {
    case RW_I32: return f(int32_t{});
    case RW_I64: return f(int64_t{});
  }
  return cudaErrorInvalidValue;
}

// Programmatic dependent launch: a kernel launched as `dependent` (rw_launch) lets its
// successor start, then waits until its predecessors' writes are visible.
__device__ __forceinline__ void rw_let_successor_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void rw_dependent_start() {
  rw_let_successor_start();
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// A launch whose error is its own (an earlier, unrelated error of the thread stays where
// it is). dependent: the launch may start while its predecessor on the stream runs; the
// kernel calls rw_dependent_start() before it touches global memory.
template <typename... KArgs, typename... Args>
inline cudaError_t rw_launch(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                             bool dependent, Args... args) {
  if (!dependent) {
    std::tuple<std::remove_const_t<KArgs>...> held(args...);
    return std::apply(
        [&](auto&... a) {
          void* at[] = {&a...};
          return cudaLaunchKernel((const void*)k, grid, block, at, smem, s);
        },
        held);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, KArgs(args)...);
}
