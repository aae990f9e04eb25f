// What the kernels over packed sequences and paged caches share: the 16-bit activation types, and the sequence a
// packed token belongs to.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "gsq_common.h"

namespace gsq {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// A 16-bit activation type: single values, pairs (rounded to nearest) and its matrix instruction.
template <bool BF>
struct Half;
template <>
struct Half<false> {
  __device__ static float ld(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
  __device__ static uint16_t mk(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
  __device__ static uint32_t pack(f32x2 v) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2)); }
  __device__ static f32x2 unpack(uint32_t w) { return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2); }
  // towards zero, so that what is left of a positive value is not negative
  __device__ static uint32_t chop(f32x2 v) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(v.x, v.y)); }
  // a pair of values less what is cut off, rounded: one instruction each takes the 16-bit values off
  __device__ static uint32_t rest(f32x2 v, uint32_t cut) {
    const f16x2 h = __builtin_bit_cast(f16x2, cut);
    return pack((f32x2){__builtin_fmaf((float)h.x, -1.f, v.x), __builtin_fmaf((float)h.y, -1.f, v.y)});
  }
  static constexpr uint16_t kLeast = 1;  // least positive value that the matrix instruction does not take for 0
  __device__ static f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Half<true> {
  __device__ static float ld(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
  __device__ static uint16_t mk(float v) { return (uint16_t)f32_to_bf16_bits(v); }
  __device__ static uint32_t pack(f32x2 v) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2)); }
  __device__ static f32x2 unpack(uint32_t w) { return (f32x2){ld((uint16_t)w), ld((uint16_t)(w >> 16))}; }
  __device__ static uint32_t chop(f32x2 v) {
    const float x = v.x, y = v.y;  // a bit cast of a vector's element takes the first
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
  }
  __device__ static uint32_t rest(f32x2 v, uint32_t cut) { return pack(v - unpack(cut)); }
  static constexpr uint16_t kLeast = 0x80;
  __device__ static f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// v_exp_f32: 2^x to one ulp (results below the normal range are 0)
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// 1 / (1 + e^-x) from the hardware's power of two and reciprocal, to a few ulps of float32
__device__ __forceinline__ float sigmoid_raw(float x) {
  return __builtin_amdgcn_rcpf(1.f + exp2_raw(x * -1.44269504088896340736f));
}

// The sequence of packed token t: how many of the B sequences end at or before it (B: t lies behind the last). Called
// by whole waves with one t; every load is in flight before the first is used.
__device__ __forceinline__ int seq_of(const int32_t* cu, int B, int t) {
  int n = 0;
  for (int i = threadIdx.x & 63; i - (int)(threadIdx.x & 63) < B; i += 64)
    n += __popcll(__ballot(i < B && cu[min(i, B - 1) + 1] <= t));
  return n;
}

// What lies at p[i], by a scalar load: i the same in every lane, and nothing that the kernel writes.
__device__ __forceinline__ int scalar_at(const int32_t* p, int64_t i) {
  return ((const __attribute__((address_space(4))) int32_t*)p)[i];
}

// A sequence of a step, as far as it can be served: its tokens lie in the packed ones, its request and its length in the
// block table. `fine` false: outputs are NaN, nothing else is touched.
struct PackedSeq {
  int t0, n, len, row;
  bool fine;
  __device__ PackedSeq(const int32_t* cu, const int32_t* rows, const int32_t* lens, int b, int N, int R, int64_t most) {
    t0 = cu[b];
    n = cu[b + 1] - t0;
    len = lens[b];
    row = rows[b];
    fine = t0 >= 0 && n >= 0 && n <= N - t0 && t0 <= N && row >= 0 && row < R && len >= n && len <= most;
  }
};

}  // namespace gsq
