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
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kTreeConv = 8;  // largest convolution kernel
constexpr int kTreeRows = 4;  // q or k rows of a wave whose inputs are in flight together
constexpr float kTreeUnit = 4096.f;  // q and k rows in fp16 numbers: normalized they are at most sqrt(128) in size

__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// the value of lane 16 Q + lane % 16
template <int Q>
__device__ __forceinline__ float from_row(float v) {
  const uint32_t x = __builtin_bit_cast(uint32_t, v);
  const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);  // rows 0 1 0 1, and 2 3 2 3
  const uint32_t y = h[Q >> 1];
  const auto r = __builtin_amdgcn_permlane16_swap(y, y, false, false);  // the even one four times, and the odd one
  return __builtin_bit_cast(float, (uint32_t)r[Q & 1]);
}

// x / (1 + e^-x) and 1 / sqrt(x) from the hardware's power of two, reciprocal and square root: a few ulps of float32
__device__ __forceinline__ float silu_raw(float x) {
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f));
}
__device__ __forceinline__ float rsqrt_raw(float x) { return __builtin_amdgcn_rsqf(x); }

}  // namespace

// One workgroup per (value head, batch row), a wave per 16 state columns, tokens in NI tiles of 16 rows.
// Products that sum over the key dims take their float32 factors as two fp16 numbers each (hi + lo, 22 bits;
// q and k before their constant factor, state columns over a power of two, so that both are of one size and
// lo x lo, 2^-24 of the product, can go; q and k times 2^12, so that rows far below the norm's epsilon keep their bits too): three MFMAs of 32 dims in 48 cycles where float32 ones take 256. What
// sums over tokens stays in float32 MFMAs (16 x 16 x 4): for A a lane gives row lane % 16, for B and the
// result column lane % 16; step e takes rows 4 (lane / 16) + e, so that operands are 16-byte pieces and a
// result is the B operand of the next product as it is.
//  * q and k (convolution, SiLU, norm) go to LDS, a wave per row; v is formed where the system needs it;
//  * tiles of k k^T and q k^T are shared out over the waves, weighted and masked into LDS;
//  * each wave solves for its columns tile by tile: earlier tiles by MFMA, the 16 rows of a tile in turn;
//  * outputs meet in LDS for the gated norm over the head.
// Bound by the latency of these steps, one workgroup a CU: 64 tokens of 4 rows (48 heads of 128 x 128) take 41 us,
// of them 4 for the windows, 13 for the convolutions, 7 for the products with keys and state, 6 for the system
// and 5 for the norms (float32 products, divisions and LDS shuffles throughout: 87); 13 tokens of one row 16.7.
// A token whose u is not finite is taken out of the products and its column's paths through it set to NaN:
// 0 x NaN would reach tokens that do not follow it.
template <int DT, int DKP, int NI, int TH>
__global__ void __launch_bounds__(TH) gdn_tree_kernel(GdnTreeArgs a, bool pair) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int QS = DKP + 8, MS = 16 * NI + 4, R = 16 * NI;  // LDS row strides, padded against bank conflicts
  extern __shared__ __attribute__((aligned(16))) float tree_lds[];
  // k rows, then q rows, hi then lo: [2][2 R][QS] of fp16; outputs [R][dv + 4] afterwards
  _Float16* const kq = reinterpret_cast<_Float16*>(tree_lds);
  const int dv = a.dv, out_s = dv + 4;
  const int kq_size = 2 * R * QS > R * out_s ? 2 * R * QS : R * out_s;
  float* const mk = tree_lds + kq_size;     // weights of u_j in u_i, [j][i] (transposed)
  float* const mk2 = mk + R * MS;           // the same, [i][j]
  float* const mq = mk2 + R * MS;           // weights of u_j in o_i, [i][j]
  float* const grown = mq + R * MS;         // G_i
  float* const betas = grown + R;
  double* const logs = reinterpret_cast<double*>(betas + R);      // log G_i
  uint64_t* const paths = reinterpret_cast<uint64_t*>(logs + R);  // token i and its ancestors
  const T** const where = reinterpret_cast<const T**>(paths + R);  // input i of token t's window: [kTreeConv][R], newest first
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

  // this wave's columns of the state: dims 32 s + 8 g + j of column 16 wave + c
  float sf[DKP / 32][8];
  {
    const float* Sp = a.rec + ((int64_t)bb * Hv + h) * dk * dv + 16 * wave + c;
#pragma unroll
    for (int s = 0; s < DKP / 32; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = 32 * s + 8 * g + j;
        sf[s][j] = d < dk ? Sp[(int64_t)d * dv] : 0.f;
      }
  }
  // a and b of the tokens: lane i of the first wave
  float av = 0.f, bv = 0.f;
  if (wave == 0 && lane < S) {
    const T* abr = static_cast<const T*>(a.ab) + ((int64_t)bb * S + lane) * a.ab_stride;
    av = E::ld(abr + h) + a.dt_bias[h];
    bv = E::ld(abr + Hv + h);
  }
  // windows: lane t finds the rows that hold the inputs of token t, newest first (tokens past the last: the last's);
  // negative: the state's rows, -1 its last
  const T* in_at[kTreeConv];
  {
    int p = min(lane, S - 1);
#pragma unroll
    for (int i = 0; i < kTreeConv; ++i) {
      in_at[i] = p >= 0 ? qkv + (int64_t)p * a.qkv_stride : cst + (int64_t)max(K - 1 + p, 0) * conv_dim;
      if (i % nw == wave && lane < R) where[i * R + lane] = in_at[i];
      const int up = __shfl(par, max(p, 0), 64);
      p = p >= 0 ? up : p - 1;
    }
  }
  auto row_of = [&](const T* p, int t) {  // lane t's
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const T*>((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, t) |
                                      ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), t) << 32));
  };
  __syncthreads();  // the windows
  // v of rows 16 i + 4 g + e, this lane's column; the first tile's inputs come while q and k are formed
  const int vch = 2 * key_dim + h * dv + 16 * wave + c;
  float vw[kTreeConv];
  T vin[4][kTreeConv];
  auto load_v = [&](int i) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < kTreeConv; ++j)
        if (j < K) vin[e][j] = where[j * R + 16 * i + 4 * g + e][vch];
  };
#pragma unroll
  for (int i = 0; i < kTreeConv; ++i) vw[i] = i < K ? E::ld(static_cast<const T*>(a.conv_w) + (int64_t)vch * K + K - 1 - i) : 0.f;
  load_v(0);
  // q and k rows: half of the waves each, two channels a lane, kTreeRows rows' inputs in flight
  {
    const bool isq = wave >= nw / 2;
    const int w0 = isq ? wave - nw / 2 : wave, ws = isq ? nw - nw / 2 : nw / 2, c0 = 2 * lane;
    const bool on = c0 < dk;
    const int ch = (isq ? 0 : key_dim) + kh * dk + min(c0, dk - 2);
    const T* const cw = static_cast<const T*>(a.conv_w) + (int64_t)ch * K;
    float wa[kTreeConv], wb[kTreeConv];
#pragma unroll
    for (int i = 0; i < kTreeConv; ++i) {
      wa[i] = i < K ? E::ld(cw + K - 1 - i) : 0.f;
      wb[i] = i < K ? E::ld(cw + 2 * K - 1 - i) : 0.f;
    }
    const float dki = 1.f / (float)dk;
    _Float16* const dst = kq + (isq ? R * QS : 0);
    for (int t0 = w0; t0 < R; t0 += kTreeRows * ws) {
      struct alignas(2 * sizeof(T)) P { T e[2]; } in[kTreeRows][kTreeConv];
#pragma unroll
      for (int u = 0; u < kTreeRows; ++u)
#pragma unroll
        for (int i = 0; i < kTreeConv; ++i)
          if (i < K) {
            const T* const p = row_of(in_at[i], min(t0 + u * ws, S - 1)) + ch;
            if (pair) {
              in[u][i] = *reinterpret_cast<const P*>(p);
            } else {
              in[u][i].e[0] = p[0];
              in[u][i].e[1] = p[1];
            }
          }
#pragma unroll
      for (int u = 0; u < kTreeRows; ++u) {
        const int t = t0 + u * ws;
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int i = kTreeConv - 1; i >= 0; --i)
          if (i < K) {
            x += E::ld(&in[u][i].e[0]) * wa[i];
            y += E::ld(&in[u][i].e[1]) * wb[i];
          }
        x = silu_raw(x);
        y = silu_raw(y);
        const float rn = rsqrt_raw(lanes_sum(on ? x * x + y * y : 0.f) * dki + 1e-6f) * kTreeUnit;
        x = on && t < S ? x * rn : 0.f;
        y = on && t < S ? y * rn : 0.f;
        if (c0 < DKP && t < R) {
          const struct alignas(4) H { _Float16 e[2]; } hi = {{(_Float16)x, (_Float16)y}},
              lo = {{(_Float16)(x - (float)hi.e[0]), (_Float16)(y - (float)hi.e[1])}};
          *reinterpret_cast<H*>(dst + t * QS + c0) = hi;
          *reinterpret_cast<H*>(dst + (2 * R + t) * QS + c0) = lo;
        }
      }
    }
  }
  f32x4 u[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if (i) load_v(i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = 0.f;
#pragma unroll
      for (int j = kTreeConv - 1; j >= 0; --j)
        if (j < K) x += E::ld(&vin[e][j]) * vw[j];
      u[i][e] = 16 * i + 4 * g + e < S ? silu_raw(x) : 0.f;
    }
  }
  // paths, decays and beta of the tokens
  if (wave == 0) {
    uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
    const float sp = av > 20.f ? av : log1pf(expf(av));  // softplus (torch's threshold 20)
    double lg = lane < S ? (double)(a.ssm_a[h] * sp) : 0.0;
    // a decay below e^-1000 is 0 for any use of it; its logarithm would take the others' bits from the sums along the path
    lg = lg < -1000.0 ? -1000.0 : lg;
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
      betas[lane] = lane < S ? 1.f / (1.f + expf(-bv)) : 0.f;
    }
  }
  __syncthreads();
  const float qscale = 1.f / (kTreeUnit * (float)dk), kscale = 1.f / (kTreeUnit * sqrtf((float)dk));
  // tiles (i, j <= i) of k k^T and q k^T
  for (int n = wave; n < NI * (NI + 1); n += nw) {
    const bool isq = n & 1;
    int i = 0, j = n >> 1;
    while (j > i) j -= ++i;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    const _Float16* const ra = kq + ((isq ? R : 0) + 16 * i + c) * QS + 8 * g;
    const _Float16* const rb = kq + (16 * j + c) * QS + 8 * g;
#pragma unroll
    for (int d = 0; d < DKP; d += 32) {
      const f16x8 xh = *reinterpret_cast<const f16x8*>(ra + d), xl = *reinterpret_cast<const f16x8*>(ra + 2 * R * QS + d);
      const f16x8 yh = *reinterpret_cast<const f16x8*>(rb + d), yl = *reinterpret_cast<const f16x8*>(rb + 2 * R * QS + d);
      s = mma16(xh, yh, s);
      s = mma16(xh, yl, s);
      s = mma16(xl, yh, s);
    }
    s *= isq ? qscale * kscale : kscale * kscale;
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
  f16x8 sh[DKP / 32], sl[DKP / 32];
  float mx = 0.f;
#pragma unroll
  for (int s = 0; s < DKP / 32; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(sf[s][j]));
  mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
  const int ex = mx > 0.f && mx <= FLT_MAX ? -ilogbf(mx) : 0;  // the column's largest: 1 .. 2
#pragma unroll
  for (int s = 0; s < DKP / 32; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = ldexpf(sf[s][j], ex);
      sh[s][j] = (_Float16)x;
      sl[s][j] = (_Float16)(x - (float)sh[s][j]);
    }
  const float ks_ = ldexpf(kscale, -ex), qs_ = ldexpf(qscale, -ex);
  f32x4 o[NI];
  auto with_state = [&](const _Float16* rows) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DKP / 32; ++d) {
      const f16x8 xh = *reinterpret_cast<const f16x8*>(rows + c * QS + 8 * g + 32 * d);
      const f16x8 xl = *reinterpret_cast<const f16x8*>(rows + (2 * R + c) * QS + 8 * g + 32 * d);
      s = mma16(xh, sh[d], s);
      s = mma16(xh, sl[d], s);
      s = mma16(xl, sh[d], s);
    }
    return s;
  };
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const f32x4 ks = with_state(kq + 16 * i * QS) * ks_, qs = with_state(kq + (R + 16 * i) * QS) * qs_;
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
    if (i && __any(bad != 0))
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (paths[16 * i + 4 * g + e] & bad) u[i][e] = __builtin_nanf("");
    // the tile's rows in turn: row r is final, its share leaves the rows that follow it (the others' weight is 0)
    f32x4 w[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = *reinterpret_cast<const f32x4*>(mk + (16 * i + r) * MS + 16 * i + 4 * g);
#pragma unroll
    for (int r = 0; r < 15; ++r) {
      const float ur = u[i][r & 3];
      const float x = r < 4 ? from_row<0>(ur) : (r < 8 ? from_row<1>(ur) : (r < 12 ? from_row<2>(ur) : from_row<3>(ur)));
#pragma unroll
      for (int e = 0; e < 4; ++e) u[i][e] = w[r][e] == 0.f ? u[i][e] : __builtin_fmaf(-w[r][e], x, u[i][e]);
    }
    // what is not finite stays out of the products, and marks the tokens that follow it
    uint32_t off = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(fabsf(u[i][e]) <= FLT_MAX)) {
        off |= 1u << (4 * g + e);
        u[i][e] = 0.f;
      }
    if (__any(off != 0)) {
      off |= __shfl_xor(off, 16, 64);
      off |= __shfl_xor(off, 32, 64);
      bad |= (uint64_t)off << (16 * i);
    }
#pragma unroll
    for (int j = 0; j <= i; ++j) {
      const f32x4 wq = *reinterpret_cast<const f32x4*>(mq + (16 * i + c) * MS + 16 * j + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i] = mma4(wq[e], u[j][e], o[i]);
    }
  }
  // outputs to LDS (q and k are no longer read), then a wave per row: gated norm over the head
  float* const os = tree_lds;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = 16 * i + 4 * g + e;
      os[t * out_s + 16 * wave + c] = paths[t] & bad ? __builtin_nanf("") : o[i][e];
    }
  __syncthreads();
  const float dvi = 1.f / (float)dv;
  float nm[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) nm[j] = 64 * j < dv ? E::ld(static_cast<const T*>(a.norm_w) + 64 * j + lane) : 0.f;
  for (int t0 = wave; t0 < S; t0 += kTreeRows * nw) {
    T z[kTreeRows][4];
#pragma unroll
    for (int v = 0; v < kTreeRows; ++v)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (64 * j < dv)
          z[v][j] = static_cast<const T*>(a.z)[((int64_t)bb * S + min(t0 + v * nw, S - 1)) * a.z_stride + (int64_t)h * dv + 64 * j + lane];
#pragma unroll
    for (int v = 0; v < kTreeRows; ++v) {
      const int t = t0 + v * nw;
      if (t >= S) break;
      float x[4], ss = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = 64 * j < dv ? os[t * out_s + 64 * j + lane] : 0.f;
        ss += x[j] * x[j];
      }
      const float rn = rsqrt_raw(lanes_sum(ss) * dvi + a.eps);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (64 * j < dv) out[(int64_t)t * a.out_stride + 64 * j + lane] = E::mk(x[j] * rn * nm[j] * silu_raw(E::ld(&z[v][j])));
    }
  }
}

template <int DT, int DKP, int NI, int TH>
static hipError_t launch_gdn_tree_t(const GdnTreeArgs& a, hipStream_t s) {
  using T = typename Elem<DT>::T;
  constexpr int R = 16 * NI;
  constexpr auto bytes = [](int dv) { return 4 * (std::max(2 * R * (DKP + 8), R * (dv + 4)) + 3 * R * (R + 4) + 2 * R) + (16 + 8 * kTreeConv) * R; };
  static_assert(bytes(256) <= 160 * 1024);
  static LdsLimit limit;
  const hipError_t e = limit.raise((const void*)gdn_tree_kernel<DT, DKP, NI, TH>, bytes(TH / 4));
  if (e != hipSuccess) return e;
  // pairs of channels in one load: every row of inputs and states starts at a multiple of them
  const bool pair = ((a.qkv_stride & 1) | ((reinterpret_cast<uintptr_t>(a.qkv) | reinterpret_cast<uintptr_t>(a.conv)) & (2 * sizeof(T) - 1))) == 0;
  hipLaunchKernelGGL((gdn_tree_kernel<DT, DKP, NI, TH>), dim3((unsigned)a.Hv, (unsigned)a.B), dim3((unsigned)(4 * a.dv)),
                     bytes(a.dv), s, a, pair);
  return hipGetLastError();
}

hipError_t launch_gdn_tree(int dt, const GdnTreeArgs& a, hipStream_t s) {
  auto rows = [&](auto t, auto d) -> hipError_t {
    constexpr int DT = decltype(t)::value, DKP = decltype(d)::value;
    auto threads = [&](auto n) -> hipError_t {
      constexpr int NI = decltype(n)::value;
      return a.dv <= 128 ? launch_gdn_tree_t<DT, DKP, NI, 512>(a, s) : launch_gdn_tree_t<DT, DKP, NI, 1024>(a, s);
    };
    if (a.S <= 16) return threads(std::integral_constant<int, 1>{});
    if (a.S <= 32) return threads(std::integral_constant<int, 2>{});
    return threads(std::integral_constant<int, 4>{});
  };
  auto dims = [&](auto t) -> hipError_t {
    return a.dk <= 64 ? rows(t, std::integral_constant<int, 64>{}) : rows(t, std::integral_constant<int, 128>{});
  };
  if (dt == MD_F16) return dims(std::integral_constant<int, MD_F16>{});
  if (dt == MD_BF16) return dims(std::integral_constant<int, MD_BF16>{});
  return dims(std::integral_constant<int, MD_F32>{});
}

}  // namespace gsq
