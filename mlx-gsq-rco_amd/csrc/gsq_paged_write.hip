// New tokens of packed sequences into a paged K/V cache: q and k RMS-normalized per head and rotated at their
// positions in one pass, k and v written to their slots (the reference runs these as separate operations of mlx-lm's
// attention, mlx_gsq/models/qwen35.py:114-152).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gsq_common.h"
#include "gsq_seq16.h"

namespace gsq {

// A workgroup per (token, share of its head rows); HD / 8 lanes hold a row, eight values each, so that a wave takes
// 512 / HD rows at once, kRows times before the first is used. The rotary factors of the position are formed once per
// workgroup: turns in double, reduced to half a turn, sine and cosine in float32 (2^-22 of a radian off at any position).
// Everything up to the one rounding of the result is float32.
// Bound by memory: 4445 tokens of 24 + 2 x 4 rows of 256, 146 MB in 40 us (3.7 TB/s; a large copy moves 5.1). Few tokens
// are one latency: 3.6 us for 8 of them.
constexpr int kWholeFrom = 512;  // tokens from which a workgroup takes all rows of its token (us, shares and whole: 128 tokens
                                 // 3.9 and 6.0, 300 5.4 and 7.0, 600 8.7 and 8.5, 2048 22 and 18)

template <bool BF, int HD, int kRows>
__global__ void __launch_bounds__(256) paged_write_kernel(PagedWriteArgs a, bool wide) {
  using E = Half<BF>;
  constexpr int TR = HD / 8, RI = 64 / TR;  // lanes of a row, rows of a wave
  __shared__ __attribute__((aligned(16))) float cs[HD / 2], sn[HD / 2];
  __shared__ __attribute__((aligned(16))) float rot[4][RI][HD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sub = lane / TR, d0 = 8 * (lane % TR);
  const int t = blockIdx.x, hr = a.rd / 2, nh = a.H + 2 * a.Hkv, step = 4 * RI * gridDim.y;
  const bool whole = hr % 8 == 0;
  const int64_t slot = a.slots[t], p = a.pos[t];
  const bool there = slot >= 0 && slot < a.n_slots;
  const uint16_t* const qb = static_cast<const uint16_t*>(a.q) + (int64_t)t * a.q_stride + d0;
  const uint16_t* const kb = static_cast<const uint16_t*>(a.k) + (int64_t)t * a.k_stride + d0;
  const uint16_t* const vb = static_cast<const uint16_t*>(a.v) + (int64_t)t * a.v_stride + d0;
  u32x4 x[kRows];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int h = min(h0 + u * step + sub, nh - 1);
      const uint16_t* const src = h < a.H ? qb + h * a.q_head : h < a.H + a.Hkv ? kb + (h - a.H) * a.k_head : vb + (h - a.H - a.Hkv) * a.v_head;
      if (wide) {
        x[u] = *reinterpret_cast<const u32x4*>(src);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[u][e] = (uint32_t)src[2 * e] | ((uint32_t)src[2 * e + 1] << 16);
      }
    }
  };
  const int first = (blockIdx.y * 4 + wave) * RI;
  load(first);
  float wq[8], wk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    wq[e] = E::ld(static_cast<const uint16_t*>(a.q_norm_w)[d0 + e]);
    wk[e] = E::ld(static_cast<const uint16_t*>(a.k_norm_w)[d0 + e]);
  }
  if (tid < hr) {
    const double turns = (double)p * a.inv_freq[tid] * 0.15915494309189533577;
    sincospif((float)(2. * (turns - rint(turns))), &sn[tid], &cs[tid]);
  }
  __syncthreads();
  const int64_t page = slot / a.P, off = slot - page * a.P;
  for (int h0 = first; h0 < nh; h0 += kRows * step) {
    if (h0 != first) load(h0);
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int h = h0 + u * step + sub;
      const bool isq = h < a.H, isv = h >= a.H + a.Hkv;
      float f[8], ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = E::ld((uint16_t)(x[u][e >> 1] >> (16 * (e & 1))));
        ss += f[e] * f[e];
      }
#pragma unroll
      for (int o = 1; o < TR; o <<= 1) ss += __shfl_xor(ss, o, 64);
      const float rn = 1.f / sqrtf(ss / (float)HD + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= rn * (isq ? wq[e] : wk[e]);
      if (d0 < a.rd) {  // the wave's own rows: its LDS operations complete in order
        float* const mine = &rot[wave][sub][0];
        *reinterpret_cast<f32x4*>(mine + d0) = (f32x4){f[0], f[1], f[2], f[3]};
        *reinterpret_cast<f32x4*>(mine + d0 + 4) = (f32x4){f[4], f[5], f[6], f[7]};
        __builtin_amdgcn_wave_barrier();
        if (whole) {  // all eight on one side of the middle
          const bool low = d0 < hr;
          const int i0 = low ? d0 : d0 - hr;
          const float* const other = mine + (low ? d0 + hr : i0);
          const float sign = low ? -1.f : 1.f;
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const f32x4 y = *reinterpret_cast<const f32x4*>(other + e);
            const f32x4 co = *reinterpret_cast<const f32x4*>(cs + i0 + e), si = *reinterpret_cast<const f32x4*>(sn + i0 + e);
#pragma unroll
            for (int r = 0; r < 4; ++r) f[e + r] = f[e + r] * co[r] + sign * y[r] * si[r];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int d = d0 + e, i = d < hr ? d : d - hr;
            if (d < a.rd) f[e] = f[e] * cs[i] + (d < hr ? -mine[d + hr] : mine[i]) * sn[i];
          }
        }
        __builtin_amdgcn_wave_barrier();
      }
      if (h >= nh) continue;
      u32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = E::pack((f32x2){f[2 * e], f[2 * e + 1]});
      if (isv) o = x[u];
      if (isq) {
        if (!there) o = (u32x4){0, 0, 0, 0};
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.out) + ((int64_t)t * a.H + h) * HD + d0) = o;
      } else if (there) {
        const int kh = isv ? h - a.H - a.Hkv : h - a.H;
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(isv ? a.vp : a.kp) + ((page * a.Hkv + kh) * a.P + off) * HD + d0) = o;
      }
    }
  }
}

template <bool BF>
static hipError_t launch_paged_write_t(const PagedWriteArgs& a, hipStream_t s) {
  auto launch = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) % 16 |
                       (uintptr_t)((a.q_stride | a.q_head | a.k_stride | a.k_head | a.v_stride | a.v_head) % 8)) == 0;
    const int rows = a.H + 2 * a.Hkv, per = 4 * (512 / HD);
    if (a.N < kWholeFrom) {
      hipLaunchKernelGGL((paged_write_kernel<BF, HD, 1>), dim3((unsigned)a.N, (unsigned)((rows + per - 1) / per)), dim3(256), 0, s, a, wide);
    } else {
      hipLaunchKernelGGL((paged_write_kernel<BF, HD, 2>), dim3((unsigned)a.N), dim3(256), 0, s, a, wide);
    }
    return hipGetLastError();
  };
  if (a.hd == 256) return launch(std::integral_constant<int, 256>{});
  if (a.hd == 128) return launch(std::integral_constant<int, 128>{});
  if (a.hd == 64) return launch(std::integral_constant<int, 64>{});
  return hipErrorInvalidValue;
}

hipError_t launch_paged_write(bool bf16, const PagedWriteArgs& a, hipStream_t s) {
  return bf16 ? launch_paged_write_t<true>(a, s) : launch_paged_write_t<false>(a, s);
}

}  // namespace gsq
