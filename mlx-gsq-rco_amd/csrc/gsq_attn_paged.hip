// Attention of packed sequences over a paged K/V cache: single tokens, chunks of prompts and whole prompts in one call
// (the reference runs mlx-lm's attention over one sequence, mlx_gsq/models/qwen35.py:114-152).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gsq_common.h"
#include "gsq_elem.h"
#include "gsq_seq16.h"

namespace gsq {

// A wave per (token, head): one pass over the positions the token sees, the running maximum and sum of the softmax and
// the output in registers.
template <bool BF, int HD>
__global__ void __launch_bounds__(256) attn_paged_wave_kernel(AttnPagedArgs a) {
  using E = Half<BF>;
  constexpr int V = HD / 64;
  const int lane = threadIdx.x & 63, d = V * lane;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= (int64_t)a.N * a.H) return;
  const int t = (int)(i / a.H), h = (int)(i % a.H), b = seq_of(a.cu, a.B, t), kvh = h / (a.H / a.Hkv);
  uint16_t* const out = static_cast<uint16_t*>(a.out) + i * HD + d;
  float o[V], q[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = 0.f;
  if (b >= a.B) {  // behind the last sequence
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = 0;
    return;
  }
  const PackedSeq sq(a.cu, a.rows, a.lens, b, a.N, a.R, a.W * a.P);
  bool bad = !sq.fine || t < sq.t0 || t - sq.t0 >= sq.n;
  float m = -INFINITY, l = 0.f;
  if (!bad) {
    const int last = sq.len - sq.n + (t - sq.t0);
#pragma unroll
    for (int j = 0; j < V; ++j) q[j] = E::ld(static_cast<const uint16_t*>(a.q)[i * HD + d + j]);
    const float scale = 1.44269504088896340736f / sqrtf((float)HD);
    for (int p = 0; p <= last; ++p) {
      const int page = a.table[sq.row * a.W + p / a.P];
      if (page < 0 || page >= a.n_pages) {
        bad = true;
        break;
      }
      const int64_t at = (((int64_t)page * a.Hkv + kvh) * a.P + p % a.P) * HD + d;
      float s = 0.f, v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s += q[j] * E::ld(static_cast<const uint16_t*>(a.kp)[at + j]);
        v[j] = E::ld(static_cast<const uint16_t*>(a.vp)[at + j]);
      }
      s = wave_sum(s) * scale;
      const float mn = fmaxf(m, s), keep = m == mn ? 1.f : exp2_raw(m - mn), w = exp2_raw(s - mn);
      m = mn;
      l = l * keep + w;
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = o[j] * keep + w * v[j];
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float g = 1.f;
    if (a.gate) g = sigmoid_raw(E::ld(static_cast<const uint16_t*>(a.gate)[(int64_t)t * a.gate_stride + h * a.gate_head + d + j]));
    out[j] = E::mk(bad ? __builtin_nanf("") : o[j] / l * g);
  }
}

template <bool BF>
static hipError_t launch_attn_paged_t(const AttnPagedArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)a.N * a.H + 3) / 4));
  auto launch = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    hipLaunchKernelGGL((attn_paged_wave_kernel<BF, HD>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
  };
  if (a.hd == 256) return launch(std::integral_constant<int, 256>{});
  if (a.hd == 128) return launch(std::integral_constant<int, 128>{});
  if (a.hd == 64) return launch(std::integral_constant<int, 64>{});
  return hipErrorInvalidValue;
}

int64_t attn_paged_work(const AttnPagedArgs&) { return 0; }

hipError_t launch_attn_paged(bool bf16, const AttnPagedArgs& a, hipStream_t s) {
  return bf16 ? launch_attn_paged_t<true>(a, s) : launch_attn_paged_t<false>(a, s);
}

}  // namespace gsq
