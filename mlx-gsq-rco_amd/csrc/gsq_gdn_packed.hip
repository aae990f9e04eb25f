// The GatedDeltaNet over packed sequences (gsq_gdn_seq for requests of different lengths in one call, each with states
// of its own; the reference runs one sequence, mlx_gsq/models/qwen35.py:48-111).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gsq_common.h"
#include "gsq_elem.h"
#include "gsq_seq16.h"

namespace gsq {

constexpr int kConvMax = 8;  // inputs of a convolution window at most

// Convolution + SiLU of 128 channels (2 per lane) over the packed tokens TPB blockIdx.y .. + TPB - 1, the window
// sliding in registers from one token of a sequence to the next; q and k channels are RMS-normalized over their head
// (dk / 2 lanes, a power of two) and scaled, so that `work` holds [q | k | v] rows ready for the recurrence. The thread
// that meets a sequence's first token has read its state by then, and writes the new one.
template <bool BF, int TPB>
__global__ void __launch_bounds__(256) gdn_conv_packed_kernel(GdnPackedArgs a, bool pair) {
  using E = Half<BF>;
  const int key_dim = a.Hk * a.dk, conv_dim = 2 * key_dim + a.Hv * a.dv, K = a.K;
  const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int cc = wave * 128 + 2 * lane, c = min(cc, conv_dim - 2);  // conv_dim is even
  const bool on = cc < conv_dim;
  const uint16_t* const q = static_cast<const uint16_t*>(a.qkv) + c;
  auto ld2 = [&](const uint16_t* p, float& x, float& y) {
    const uint32_t w = pair ? *reinterpret_cast<const uint32_t*>(p) : (uint32_t)p[0] | ((uint32_t)p[1] << 16);
    x = E::ld((uint16_t)w);
    y = E::ld((uint16_t)(w >> 16));
  };
  // window and weights right-aligned: slot kConvMax - 1 is the current token
  float w0[kConvMax], w1[kConvMax], in0[kConvMax], in1[kConvMax];
  const uint16_t* const cw = static_cast<const uint16_t*>(a.conv_w) + (int64_t)c * K;
#pragma unroll
  for (int i = 0; i < kConvMax; ++i) {
    const int j = i - (kConvMax - K);
    w0[i] = w1[i] = in0[i] = in1[i] = 0.f;
    if (j >= 0) {
      w0[i] = E::ld(cw[j]);
      w1[i] = E::ld(cw[K + j]);
    }
  }
  const float sc = c < key_dim ? 1.f / (float)a.dk : 1.f / sqrtf((float)a.dk);
  const int half = a.dk >> 1, first = blockIdx.y * TPB;
  int b = -1, t0 = 0, end = 0;  // the sequence of the token before
  bool fine = false;
#pragma unroll
  for (int i = 0; i < TPB; ++i) {
    const int t = first + i;
    if (t >= a.N) break;
    if (b < 0 || t >= end) {  // another sequence: its window before token t
      b = seq_of(a.cu, a.B, t);
      if (b >= a.B) break;
      const PackedSeq sq(a.cu, a.rows, a.lens, b, a.N, a.R, 0x7FFFFFFF);
      t0 = sq.t0;
      end = sq.t0 + sq.n;
      fine = sq.fine && t >= t0 && t < end;
      if (!fine) end = t + 1;
      const bool fresh = sq.len == sq.n;
      uint16_t* const cst = static_cast<uint16_t*>(a.conv) + (int64_t)(fine ? sq.row : 0) * (K - 1) * conv_dim + c;
#pragma unroll
      for (int s = 0; s < kConvMax; ++s) {
        const int j = s - (kConvMax - K);  // the window of token t - 1, oldest 0
        in0[s] = in1[s] = 0.f;
        if (j < 0 || !fine) continue;
        const int u = t - t0 - K + j;
        if (u >= 0) ld2(q + (int64_t)(t0 + u) * a.qkv_stride, in0[s], in1[s]);
        else if (u >= -(K - 1) && !fresh) {
          in0[s] = E::ld(cst[(int64_t)(K - 1 + u) * conv_dim]);
          in1[s] = E::ld(cst[(int64_t)(K - 1 + u) * conv_dim + 1]);
        }
      }
      if (fine && on && t == t0) {  // slots ascending: a shift in place reads before it writes
        for (int j = 0; j < K - 1; ++j) {
          const int u = sq.n - (K - 1) + j;
          uint16_t x = 0, y = 0;
          if (u >= 0) {
            x = q[(int64_t)(t0 + u) * a.qkv_stride];
            y = q[(int64_t)(t0 + u) * a.qkv_stride + 1];
          } else if (!fresh) {
            x = cst[(int64_t)(K - 1 + u) * conv_dim];
            y = cst[(int64_t)(K - 1 + u) * conv_dim + 1];
          }
          cst[(int64_t)j * conv_dim] = x;
          cst[(int64_t)j * conv_dim + 1] = y;
        }
      }
    }
    if (!fine) continue;
#pragma unroll
    for (int s = 0; s + 1 < kConvMax; ++s) {
      in0[s] = in0[s + 1];
      in1[s] = in1[s + 1];
    }
    ld2(q + (int64_t)t * a.qkv_stride, in0[kConvMax - 1], in1[kConvMax - 1]);
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int s = 0; s < kConvMax; ++s)
      if (s >= kConvMax - K) {
        x += in0[s] * w0[s];
        y += in1[s] * w1[s];
      }
    x = silu_f(x);
    y = silu_f(y);
    float ss = x * x + y * y;
    for (int o = 1; o < half; o <<= 1) ss += __shfl_xor(ss, o, 64);
    if (c < 2 * key_dim) {
      const float rn = 1.f / sqrtf(ss / (float)a.dk + 1e-6f);
      x = x * rn * sc;
      y = y * rn * sc;
    }
    if (on) *reinterpret_cast<float2*>(a.work + (int64_t)t * conv_dim + c) = make_float2(x, y);
  }
}

// The recurrence of one (sequence, value head), its state in registers from the first token to the last: a thread
// holds 4 columns of every NG-th row. Per token two sums over the rows, across the workgroup.
template <bool BF, int DK, int DV>
__global__ void __launch_bounds__(256) gdn_rec_packed_kernel(GdnPackedArgs a) {
  using E = Half<BF>;
  constexpr int CG = DV / 4, NG = 256 / CG, NR = DK / NG;  // threads of a row, row groups, rows of a thread
  __shared__ __attribute__((aligned(16))) float red[2][4][DV];
  const int tid = threadIdx.x, wave = tid >> 6, cg = tid % CG, rg = tid / CG, col = 4 * cg;
  const int h = blockIdx.x, kh = h % a.Hk, b = blockIdx.y;
  const int key_dim = a.Hk * DK, conv_dim = 2 * key_dim + a.Hv * DV;
  uint16_t* const out = static_cast<uint16_t*>(a.out) + h * DV + col;
  auto fill = [&](int from, int to, uint16_t v) {
    for (int t = max(from, 0) + rg; t < min(to, a.N); t += NG)
      for (int e = 0; e < 4; ++e) out[(int64_t)t * a.out_stride + e] = v;
  };
  if (b == a.B) {  // rows behind the last sequence
    fill(a.cu[a.B], a.N, 0);
    return;
  }
  const PackedSeq sq(a.cu, a.rows, a.lens, b, a.N, a.R, 0x7FFFFFFF);
  if (!sq.fine) {
    fill(a.cu[b], a.cu[b + 1], E::mk(__builtin_nanf("")));
    return;
  }
  if (sq.n == 0) return;
  float* const Sp = a.rec + (((int64_t)sq.row * a.Hv + h) * DK + rg) * DV + col;
  f32x4 st[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i)
    st[i] = sq.len == sq.n ? (f32x4){0.f, 0.f, 0.f, 0.f} : *reinterpret_cast<const f32x4*>(Sp + (int64_t)i * NG * DV);
  const float dtb = a.dt_bias[h], sa = a.ssm_a[h];
  float w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = E::ld(static_cast<const uint16_t*>(a.norm_w)[col + e]);
  // sum over the row groups: in the wave, then across the waves
  auto sum_rows = [&](f32x4 p, int buf) {
#pragma unroll
    for (int o = CG; o < 64; o <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] += __shfl_xor(p[e], o, 64);
    if ((tid & 63) < CG) *reinterpret_cast<f32x4*>(&red[buf][wave][col]) = p;
    lds_sync();
    f32x4 s = *reinterpret_cast<const f32x4*>(&red[buf][0][col]);
#pragma unroll
    for (int i = 1; i < 4; ++i) s += *reinterpret_cast<const f32x4*>(&red[buf][i][col]);
    return s;
  };
  for (int i = 0; i < sq.n; ++i) {
    const int64_t t = sq.t0 + i;
    const float* const row = a.work + t * conv_dim;
    const uint16_t* const abr = static_cast<const uint16_t*>(a.ab) + t * a.ab_stride;
    float k[NR], q[NR];
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      q[j] = row[kh * DK + rg + j * NG];
      k[j] = row[key_dim + kh * DK + rg + j * NG];
    }
    const f32x4 v = *reinterpret_cast<const f32x4*>(row + 2 * key_dim + h * DV + col);
    const float av = E::ld(abr[h]) + dtb, bv = E::ld(abr[a.Hv + h]);
    const float sp = av > 20.f ? av : log1pf(expf(av));  // softplus (torch's threshold 20)
    const float beta = 1.f / (1.f + expf(-bv)), decay = expf(sa * sp);
    f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      st[j] *= decay;
      p += st[j] * k[j];
    }
    const f32x4 delta = (v - sum_rows(p, 0)) * beta;
    p = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      st[j] += delta * k[j];
      p += st[j] * q[j];
    }
    const f32x4 o = sum_rows(p, 1);
    float ss = o[0] * o[0] + o[1] * o[1] + o[2] * o[2] + o[3] * o[3];
#pragma unroll
    for (int x = 1; x < CG; x <<= 1) ss += __shfl_xor(ss, x, 64);
    const float rn = 1.f / sqrtf(ss / (float)DV + a.eps);
    if (rg == 0) {
      const uint16_t* const z = static_cast<const uint16_t*>(a.z) + t * a.z_stride + h * DV + col;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[t * a.out_stride + e] = E::mk(o[e] * rn * w[e] * silu_f(E::ld(z[e])));
    }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) *reinterpret_cast<f32x4*>(Sp + (int64_t)i * NG * DV) = st[i];
}

int64_t gdn_packed_work(const GdnPackedArgs& a) { return (int64_t)a.N * (2 * a.Hk * a.dk + a.Hv * a.dv); }

template <bool BF>
static hipError_t launch_gdn_packed_t(const GdnPackedArgs& a, hipStream_t s) {
  const int conv_dim = 2 * a.Hk * a.dk + a.Hv * a.dv;
  const bool pair = ((a.qkv_stride & 1) | (reinterpret_cast<uintptr_t>(a.qkv) & 3)) == 0;
  const dim3 cgrid((unsigned)((conv_dim + 511) / 512), (unsigned)((a.N + 7) / 8)), rgrid((unsigned)a.Hv, (unsigned)a.B + 1);
  hipLaunchKernelGGL((gdn_conv_packed_kernel<BF, 8>), cgrid, dim3(256), 0, s, a, pair);
  auto rec = [&](auto dk, auto dv) {
    hipLaunchKernelGGL((gdn_rec_packed_kernel<BF, decltype(dk)::value, decltype(dv)::value>), rgrid, dim3(256), 0, s, a);
    return hipGetLastError();
  };
  auto dims = [&](auto dk) -> hipError_t {
    if (a.dv == 64) return rec(dk, std::integral_constant<int, 64>{});
    if (a.dv == 128) return rec(dk, std::integral_constant<int, 128>{});
    if (a.dv == 256) return rec(dk, std::integral_constant<int, 256>{});
    return hipErrorInvalidValue;
  };
  if (a.dk == 32) return dims(std::integral_constant<int, 32>{});
  if (a.dk == 64) return dims(std::integral_constant<int, 64>{});
  if (a.dk == 128) return dims(std::integral_constant<int, 128>{});
  return hipErrorInvalidValue;
}

hipError_t launch_gdn_packed(bool bf16, const GdnPackedArgs& a, hipStream_t s) {
  return bf16 ? launch_gdn_packed_t<true>(a, s) : launch_gdn_packed_t<false>(a, s);
}

}  // namespace gsq
