// Activation types and small device helpers of the decoder's element-wise and recurrent kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "gsq_common.h"

namespace gsq {

enum { MD_F32 = 0, MD_F16 = 1, MD_BF16 = 2 };

template <int DT> struct Elem;
template <> struct Elem<MD_F32> {
  using T = float;
  __device__ static float ld(const T* p) { return *p; }
  __device__ static T mk(float v) { return v; }
};
template <> struct Elem<MD_F16> {
  using T = _Float16;
  __device__ static float ld(const T* p) { return (float)*p; }
  __device__ static T mk(float v) { return (_Float16)v; }
};
template <> struct Elem<MD_BF16> {
  using T = uint16_t;
  __device__ static float ld(const T* p) { return __builtin_bit_cast(float, (uint32_t)*p << 16); }
  __device__ static T mk(float v) { return (uint16_t)f32_to_bf16_bits(v); }
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Workgroup barrier that waits for this wave's LDS operations only: global loads issued before
// it stay in flight. The kernels here exchange data between threads through LDS only.
__device__ __forceinline__ void lds_sync() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float silu_f(float x) { return x / (1.f + expf(-x)); }

}  // namespace gsq
