// The GatedDeltaNet of a tree of drafted tokens for the Qwen3.5-hybrid decoder (what
// mlx_gsq/models/qwen35.py:48-111 computes token by token along a sequence, along every path of a
// tree): the state S and the convolution's inputs of a token are those of its parent, or the cached ones.
//
// No state is kept for each token. With d_i the decay of token i, G_i the product of the decays on the
// path from the cache to i, S_0 the cached state,
//   S_i = d_i S_parent + k_i u_i^T = G_i S_0 + sum over j on i's path of (G_i / G_j) k_j u_j^T
//   u_i = beta_i (v_i - G_i S_0^T k_i - sum over proper ancestors j of (G_i / G_j) (k_i . k_j) u_j)
//   o_i = G_i S_0^T q_i + sum over j on i's path of (G_i / G_j) (q_i . k_j) u_j
// so S_0 is read once, and the tokens of a head are two products with S_0, two T x T products, and a
// triangular system that lets a token see its ancestors only.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "gsq_common.h"
#include "gsq_elem.h"

namespace gsq {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTreeConv = 8;  // largest convolution kernel

__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

}  // namespace

// One workgroup per (value head, batch row), a wave per 16 state columns, tokens in NI tiles of 16 rows.
// All products are float32 MFMAs (16 x 16 x 4): for A a lane gives row lane % 16, for B and the result
// column lane % 16; a product's step e takes dims 4 (lane / 16) + e, so operands are 16-byte pieces,
// and a result (rows 4 (lane / 16) + e on its registers) is the B operand of the next product as it is.
//  * q and k (convolution, SiLU, norm) go to LDS, a wave per row; v is formed where the system needs it;
//  * tiles of k k^T and q k^T are shared out over the waves, weighted and masked into LDS;
//  * each wave solves for its columns tile by tile: earlier tiles by MFMA, the 16 rows of a tile in turn;
//  * outputs meet in LDS for the gated norm over the head.
// A token whose u is not finite is taken out of the sums and its column's paths through it set to NaN:
// 0 x NaN would reach tokens that do not follow it.
template <int DT, int DKP, int NI>
__global__ void __launch_bounds__(1024) gdn_tree_kernel(GdnTreeArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int QS = DKP + 4, MS = 16 * NI + 4, R = 16 * NI;  // LDS row strides, padded against bank conflicts
  extern __shared__ __attribute__((aligned(16))) float tree_lds[];
  float* const kq = tree_lds;               // k rows, then q rows: [2][R][QS]; outputs [R][dv + 4] afterwards
  const int dv = a.dv, out_s = dv + 4;
  const int kq_size = 2 * R * QS > R * out_s ? 2 * R * QS : R * out_s;
  float* const mk = tree_lds + kq_size;     // weights of u_j in u_i, [j][i] (transposed)
  float* const mk2 = mk + R * MS;           // the same, [i][j]
  float* const mq = mk2 + R * MS;           // weights of u_j in o_i, [i][j]
  float* const grown = mq + R * MS;         // G_i
  float* const betas = grown + R;
  double* const logs = reinterpret_cast<double*>(betas + R);      // log G_i
  uint64_t* const paths = reinterpret_cast<uint64_t*>(logs + R);  // token i and its ancestors
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
  const int g = lane >> 4, c = lane & 15;
  const int h = blockIdx.x, bb = blockIdx.y, Hk = a.Hk, Hv = a.Hv, dk = a.dk, K = a.K, S = a.S, kh = h % Hk;
  const int key_dim = Hk * dk, conv_dim = 2 * key_dim + Hv * dv;
  const int32_t* const parents = a.parents + (int64_t)bb * a.parents_stride;
  const int par = lane < S ? parents[lane] : -1;
  T* const out = static_cast<T*>(a.out) + (int64_t)bb * S * a.out_stride + (int64_t)h * dv;
  if (__any(par < -1 || par >= lane)) {  // uniform
    for (int i = tid; i < S * dv; i += blockDim.x) out[(int64_t)(i / dv) * a.out_stride + i % dv] = E::mk(__builtin_nanf(""));
    return;
  }
  const T* const qkv = static_cast<const T*>(a.qkv) + (int64_t)bb * S * a.qkv_stride;
  const T* const cst = static_cast<const T*>(a.conv) + (int64_t)bb * (K - 1) * conv_dim;

  // this wave's columns of the state: dims 16 s + 4 g + e of column 16 wave + c
  float st[DKP / 4];
  {
    const float* Sp = a.rec + ((int64_t)bb * Hv + h) * dk * dv + 16 * wave + c;
#pragma unroll
    for (int s = 0; s < DKP / 16; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 16 * s + 4 * g + e;
        st[4 * s + e] = d < dk ? Sp[(int64_t)d * dv] : 0.f;
      }
  }
  // paths, decays and beta of the tokens: lane i of the first wave
  if (wave == 0) {
    uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
    double lg = 0.0;
    float beta = 0.f;
    if (lane < S) {
      const T* abr = static_cast<const T*>(a.ab) + ((int64_t)bb * S + lane) * a.ab_stride;
      const float av = E::ld(abr + h) + a.dt_bias[h];
      const float sp = av > 20.f ? av : log1pf(expf(av));  // softplus (torch's threshold 20)
      lg = (double)(a.ssm_a[h] * sp);
      beta = 1.f / (1.f + expf(-E::ld(abr + Hv + h)));
    }
    int p = par;
#pragma unroll
    for (int i = 0; i < 6; ++i) {  // pointer doubling: what p's path so far holds joins
      const int src = p < 0 ? lane : p;
      lo |= __shfl(lo, src, 64);
      hi |= __shfl(hi, src, 64);
      const double up = __shfl(lg, src, 64);
      lg += p < 0 ? 0.0 : up;
      const int pp = __shfl(p, src, 64);  // by every lane: a lane that does not run it gives 0
      p = p < 0 ? -1 : pp;
    }
    if (lane < R) {
      paths[lane] = lane < S ? lo | ((uint64_t)hi << 32) : 0;
      logs[lane] = lg;
      grown[lane] = (float)exp(lg);
      betas[lane] = beta;
    }
  }
  // window of token t (uniform): rows of the inputs, negative ones from the state; newest last
  auto window = [&](int t, int (&at)[kTreeConv]) {
    int p = t;
#pragma unroll
    for (int i = kTreeConv - 1; i >= 0; --i) {
      at[i] = p;
      p = p >= 0 ? parents[p] : p - 1;
    }
  };
  auto input = [&](int p, int ch) {  // input p of a channel
    return p >= 0 ? E::ld(qkv + (int64_t)p * a.qkv_stride + ch) : E::ld(cst + (int64_t)max(K - 1 + p, 0) * conv_dim + ch);
  };
  // q and k rows: half of the waves each, two channels a lane
  {
    const bool isq = wave >= nw / 2;
    const int w0 = isq ? wave - nw / 2 : wave, ws = isq ? nw - nw / 2 : nw / 2, c0 = 2 * lane;
    const bool on = c0 < dk;
    const int ch = (isq ? 0 : key_dim) + kh * dk + min(c0, dk - 2);
    const T* const cw = static_cast<const T*>(a.conv_w) + (int64_t)ch * K;
    float wa[kTreeConv], wb[kTreeConv];
#pragma unroll
    for (int i = 0; i < kTreeConv; ++i) {
      const int j = i - (kTreeConv - K);
      wa[i] = j >= 0 ? E::ld(cw + j) : 0.f;
      wb[i] = j >= 0 ? E::ld(cw + K + j) : 0.f;
    }
    const float sc = isq ? 1.f / (float)dk : 1.f / sqrtf((float)dk);
    float* const dst = kq + (isq ? R * QS : 0);
    for (int t = w0; t < R; t += ws) {
      float x = 0.f, y = 0.f;
      if (t < S) {
        int at[kTreeConv];
        window(t, at);
#pragma unroll
        for (int i = 0; i < kTreeConv; ++i)
          if (i >= kTreeConv - K) {
            x += input(at[i], ch) * wa[i];
            y += input(at[i], ch + 1) * wb[i];
          }
        x = silu_f(x);
        y = silu_f(y);
        const float rn = 1.f / sqrtf(wave_sum(on ? x * x + y * y : 0.f) / (float)dk + 1e-6f) * sc;
        x *= rn;
        y *= rn;
      }
      if (c0 < DKP) *reinterpret_cast<float2*>(dst + t * QS + c0) = on && t < S ? make_float2(x, y) : make_float2(0.f, 0.f);
    }
  }
  // v of rows 16 i + 4 g + e, this lane's column
  f32x4 u[NI];
  {
    const int ch = 2 * key_dim + h * dv + 16 * wave + c;
    const T* const cw = static_cast<const T*>(a.conv_w) + (int64_t)ch * K;
    float w[kTreeConv];
#pragma unroll
    for (int i = 0; i < kTreeConv; ++i) {
      const int j = i - (kTreeConv - K);
      w[i] = j >= 0 ? E::ld(cw + j) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 16 * i + 4 * g + e;
        float x = 0.f;
        if (t < S) {
          int at[kTreeConv];
          window(t, at);
#pragma unroll
          for (int j = 0; j < kTreeConv; ++j)
            if (j >= kTreeConv - K) x += input(at[j], ch) * w[j];
          x = silu_f(x);
        }
        u[i][e] = x;
      }
  }
  __syncthreads();
  // tiles (i, j <= i) of k k^T and q k^T
  for (int n = wave; n < NI * (NI + 1); n += nw) {
    const bool isq = n & 1;
    int i = 0, j = n >> 1;
    while (j > i) j -= ++i;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    const float* const ra = kq + (isq ? R * QS : 0) + (16 * i + c) * QS + 4 * g;
    const float* const rb = kq + (16 * j + c) * QS + 4 * g;
#pragma unroll
    for (int d = 0; d < DKP; d += 16) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(ra + d), y = *reinterpret_cast<const f32x4*>(rb + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = mma4(x[e], y[e], s);
    }
    const int tj = 16 * j + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // row 16 i + 4 g + e, column tj
      const int ti = 16 * i + 4 * g + e;
      const bool see = (paths[ti] >> tj) & 1;
      const float r = see ? s[e] * expf((float)(logs[ti] - logs[tj])) : 0.f;
      if (isq) {
        mq[ti * MS + tj] = r;
      } else {
        const float m = ti == tj ? 0.f : betas[ti] * r;
        mk2[ti * MS + tj] = see ? m : 0.f;
        mk[tj * MS + ti] = see ? m : 0.f;
      }
    }
  }
  // products with the state
  f32x4 o[NI];
  auto with_state = [&](const float* rows) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DKP / 16; ++d) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(rows + c * QS + 4 * g + 16 * d);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = mma4(x[e], st[4 * d + e], s);
    }
    return s;
  };
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const f32x4 ks = with_state(kq + 16 * i * QS), qs = with_state(kq + (R + 16 * i) * QS);
    const f32x4 gr = *reinterpret_cast<const f32x4*>(grown + 16 * i + 4 * g);
    const f32x4 be = *reinterpret_cast<const f32x4*>(betas + 16 * i + 4 * g);
    u[i] = be * (u[i] - gr * ks);
    o[i] = gr * qs;
  }
  __syncthreads();
  uint64_t bad = 0;  // tokens whose u of this column is not finite
#pragma unroll
  for (int i = 0; i < NI; ++i) {
#pragma unroll
    for (int j = 0; j < i; ++j) {
      const f32x4 w = *reinterpret_cast<const f32x4*>(mk2 + (16 * i + c) * MS + 16 * j + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) u[i] = mma4(-w[e], u[j][e], u[i]);
    }
    // the tile's rows in turn: row r is final, its share leaves the rows after it
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int t = 16 * i + r;
      float x = __shfl(u[i][r & 3], 16 * (r >> 2) + c, 64);
      const bool off = !(fabsf(x) <= FLT_MAX) || (paths[t] & bad);
      if (off) {
        bad |= 1ull << t;
        x = 0.f;
      }
      if (g == (r >> 2)) u[i][r & 3] = x;
      const f32x4 w = *reinterpret_cast<const f32x4*>(mk + t * MS + 16 * i + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * g + e > r) u[i][e] -= x == 0.f ? 0.f : w[e] * x;
    }
#pragma unroll
    for (int j = 0; j <= i; ++j) {
      const f32x4 w = *reinterpret_cast<const f32x4*>(mq + (16 * i + c) * MS + 16 * j + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i] = mma4(w[e], u[j][e], o[i]);
    }
  }
  // outputs to LDS (q and k are no longer read), then a wave per row: gated norm over the head
  float* const os = kq;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = 16 * i + 4 * g + e;
      os[t * out_s + 16 * wave + c] = paths[t] & bad ? __builtin_nanf("") : o[i][e];
    }
  __syncthreads();
  const T* const nw_ = static_cast<const T*>(a.norm_w);
  for (int t = wave; t < S; t += nw) {
    const T* z = static_cast<const T*>(a.z) + ((int64_t)bb * S + t) * a.z_stride + (int64_t)h * dv;
    float x[4], ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = 64 * j < dv ? os[t * out_s + 64 * j + lane] : 0.f;
      ss += x[j] * x[j];
    }
    const float rn = 1.f / sqrtf(wave_sum(ss) / (float)dv + a.eps);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (64 * j < dv) {
        const int d = 64 * j + lane;
        out[(int64_t)t * a.out_stride + d] = E::mk(x[j] * rn * E::ld(nw_ + d) * silu_f(E::ld(z + d)));
      }
  }
}

template <int DT, int DKP, int NI>
static hipError_t launch_gdn_tree_t(const GdnTreeArgs& a, hipStream_t s) {
  constexpr int R = 16 * NI;
  const int kq = std::max(2 * R * (DKP + 4), R * (a.dv + 4));
  const int lds = 4 * (kq + 3 * R * (R + 4) + 2 * R) + 16 * R;
  static LdsLimit limit;  // the largest any call of this instance asks for: dv = 256
  constexpr int most = 4 * (2 * R * (DKP + 4) > R * 260 ? 2 * R * (DKP + 4) : R * 260) + 4 * (3 * R * (R + 4) + 2 * R) + 16 * R;
  static_assert(most <= 160 * 1024);
  const hipError_t e = limit.raise((const void*)gdn_tree_kernel<DT, DKP, NI>, most);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((gdn_tree_kernel<DT, DKP, NI>), dim3((unsigned)a.Hv, (unsigned)a.B), dim3((unsigned)(4 * a.dv)), lds, s, a);
  return hipGetLastError();
}

hipError_t launch_gdn_tree(int dt, const GdnTreeArgs& a, hipStream_t s) {
  auto rows = [&](auto t, auto d) -> hipError_t {
    constexpr int DT = decltype(t)::value, DKP = decltype(d)::value;
    if (a.S <= 16) return launch_gdn_tree_t<DT, DKP, 1>(a, s);
    if (a.S <= 32) return launch_gdn_tree_t<DT, DKP, 2>(a, s);
    return launch_gdn_tree_t<DT, DKP, 4>(a, s);
  };
  auto dims = [&](auto t) -> hipError_t {
    return a.dk <= 64 ? rows(t, std::integral_constant<int, 64>{}) : rows(t, std::integral_constant<int, 128>{});
  };
  if (dt == MD_F16) return dims(std::integral_constant<int, MD_F16>{});
  if (dt == MD_BF16) return dims(std::integral_constant<int, MD_BF16>{});
  return dims(std::integral_constant<int, MD_F32>{});
}

}  // namespace gsq
