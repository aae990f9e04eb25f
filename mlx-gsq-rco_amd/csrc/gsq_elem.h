// Activation types and small device helpers of the decoder's element-wise and recurrent kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

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

// fn(v of lane l, v of its partner) over the wave, in every lane and without LDS (whose round trips are what the
// norm of a row waits for): partners 1, 2, 4 and 8 lanes away, then the rows of 16 lanes. T: float or double.
template <typename T, typename F>
__device__ __forceinline__ T lanes_reduce(T v, F fn) {
  constexpr int N = sizeof(T) / 4;
  struct W { uint32_t w[N]; };
  auto dpp = [&](auto ctrl) {
    W a = __builtin_bit_cast(W, v);
    for (int i = 0; i < N; ++i)
      a.w[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a.w[i], decltype(ctrl)::value, 0xF, 0xF, false);
    v = fn(v, __builtin_bit_cast(T, a));
  };
  dpp(std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  dpp(std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  dpp(std::integral_constant<int, 0x141>{});  // row_half_mirror
  dpp(std::integral_constant<int, 0x140>{});  // row_mirror
  W a = __builtin_bit_cast(W, v), b = a;
  for (int i = 0; i < N; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
    a.w[i] = (uint32_t)r[0];
    b.w[i] = (uint32_t)r[1];
  }
  v = fn(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
  a = b = __builtin_bit_cast(W, v);
  for (int i = 0; i < N; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false);
    a.w[i] = (uint32_t)r[0];
    b.w[i] = (uint32_t)r[1];
  }
  return fn(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
}
template <typename T>
__device__ __forceinline__ T lanes_sum(T v) {
  return lanes_reduce(v, [](T x, T y) { return x + y; });
}

__device__ __forceinline__ float silu_f(float x) { return x / (1.f + expf(-x)); }

}  // namespace gsq
