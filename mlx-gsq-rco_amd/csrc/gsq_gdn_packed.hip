// The GatedDeltaNet over packed sequences (gsq_gdn_seq for requests of different lengths in one call, each with states
// of its own; the reference runs one sequence, mlx_gsq/models/qwen35.py:48-111).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gsq_common.h"
#include "gsq_elem.h"
#include "gsq_seq16.h"

namespace gsq {

// Eight float32 values as three bf16 numbers each, cut off one after the other: exactly their 24 bits, from 2^-102 on (terms
// below 2^-126 are 0 to the matrix instructions).
struct Three {
  u32x4 h, m, l;
};
__device__ __forceinline__ float cut16(float x) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t upper16(float x, float y) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
}
// a pair of values
__device__ __forceinline__ void split3(float x, float y, uint32_t& h, uint32_t& m, uint32_t& l) {
  h = upper16(x, y);
  x -= cut16(x);
  y -= cut16(y);
  m = upper16(x, y);
  l = upper16(x - cut16(x), y - cut16(y));
}
__device__ __forceinline__ Three split3(f32x4 a, f32x4 b) {
  Three r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f32x4 v = j < 2 ? a : b;
    uint32_t h, m, l;
    split3(v[2 * (j & 1)], v[2 * (j & 1) + 1], h, m, l);
    r.h[j] = h;
    r.m[j] = m;
    r.l[j] = l;
  }
  return r;
}
// their product; left out: what is 2^-24 of it and less
__device__ __forceinline__ f32x4 mma_three(const Three& a, const Three& b, f32x4 c) {
  c = Half<true>::mma(a.l, b.h, c);
  c = Half<true>::mma(a.h, b.l, c);
  c = Half<true>::mma(a.m, b.m, c);
  c = Half<true>::mma(a.m, b.h, c);
  c = Half<true>::mma(a.h, b.m, c);
  return Half<true>::mma(a.h, b.h, c);
}

constexpr int kConvMax = 8;  // inputs of a convolution window at most

// Convolution + SiLU of 128 channels (2 per lane) over the packed tokens TPB blockIdx.y .. + TPB - 1, whose inputs are all
// asked for at once; the window slides in registers from one token of a sequence to the next. q and k channels are
// RMS-normalized over their head (dk / 2 lanes, a power of two) and scaled, so that `work` holds [q | k | v] rows ready
// for the recurrence, in float32. The states are
// read only: tokens of one window lie in different workgroups, so the launch behind this one advances them.
// KW: window of the convolution (kConvMax: any up to it). Bound by its bytes where tokens are many (5118 of 10240 channels:
// 314 MB in 72 us, 4.4 TB/s), by its latencies where they are few (32: 4 us).
template <bool BF, int TPB, int KW>
__global__ void __launch_bounds__(256) gdn_conv_packed_kernel(GdnPackedArgs a, bool pair) {
  using E = Half<BF>;
  const int key_dim = a.Hk * a.dk, conv_dim = 2 * key_dim + a.Hv * a.dv, K = KW < kConvMax ? KW : a.K;
  const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int cc = wave * 128 + 2 * lane, c = min(cc, conv_dim - 2);  // conv_dim is even
  const bool on = cc < conv_dim;
  const uint16_t* const q = static_cast<const uint16_t*>(a.qkv) + c;
  auto ld2 = [&](const uint16_t* p) { return pair ? *reinterpret_cast<const uint32_t*>(p) : (uint32_t)p[0] | ((uint32_t)p[1] << 16); };
  const int half = a.dk >> 1, first = blockIdx.y * TPB;
  uint32_t x[TPB];
#pragma unroll
  for (int i = 0; i < TPB; ++i) x[i] = ld2(q + (int64_t)min(first + i, a.N - 1) * a.qkv_stride);
  // window and weights right-aligned: slot KW - 1 is the current token
  float w0[KW], w1[KW], in0[KW], in1[KW];
  const uint16_t* const cw = static_cast<const uint16_t*>(a.conv_w) + (int64_t)c * K;
#pragma unroll
  for (int i = 0; i < KW; ++i) {
    const int j = i - (KW - K);
    w0[i] = w1[i] = in0[i] = in1[i] = 0.f;
    if (j >= 0) {
      w0[i] = E::ld(cw[j]);
      w1[i] = E::ld(cw[K + j]);
    }
  }
  const float sc = c < key_dim ? 1.f / (float)a.dk : 1.f / sqrtf((float)a.dk);
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
      const uint16_t* const cst = static_cast<const uint16_t*>(a.conv) + (int64_t)(fine ? sq.row : 0) * (K - 1) * conv_dim + c;  // conv_dim is even
      uint32_t old[KW];  // the window of token t - 1, oldest first; slot KW - K is shifted out
#pragma unroll
      for (int s = 0; s < KW; ++s) {
        const int j = s - (KW - K), u = t - t0 - K + j;
        old[s] = 0;
        if (j < 1 || !fine) continue;
        if (u >= 0) old[s] = ld2(q + (int64_t)(t0 + u) * a.qkv_stride);
        else if (!fresh) old[s] = (uint32_t)cst[(int64_t)(K - 1 + u) * conv_dim] | ((uint32_t)cst[(int64_t)(K - 1 + u) * conv_dim + 1] << 16);
      }
#pragma unroll
      for (int s = 0; s < KW; ++s) {
        in0[s] = E::ld((uint16_t)old[s]);
        in1[s] = E::ld((uint16_t)(old[s] >> 16));
      }
    }
    if (!fine) continue;
#pragma unroll
    for (int s = 0; s + 1 < KW; ++s) {
      in0[s] = in0[s + 1];
      in1[s] = in1[s + 1];
    }
    in0[KW - 1] = E::ld((uint16_t)x[i]);
    in1[KW - 1] = E::ld((uint16_t)(x[i] >> 16));
    float y0 = 0.f, y1 = 0.f;
#pragma unroll
    for (int s = 0; s < KW; ++s) {
      if (KW == kConvMax && s < KW - K) continue;  // weights of 0 times anything
      y0 += in0[s] * w0[s];
      y1 += in1[s] * w1[s];
    }
    y0 *= sigmoid_raw(y0);
    y1 *= sigmoid_raw(y1);
    if (wave * 128 < 2 * key_dim) {  // a wave with q or k channels
      float ss = y0 * y0 + y1 * y1;
      for (int o = 1; o < half; o <<= 1) ss += __shfl_xor(ss, o, 64);
      if (c < 2 * key_dim) {
        const float rn = 1.f / sqrtf(ss / (float)a.dk + 1e-6f);
        y0 = y0 * rn * sc;
        y1 = y1 * rn * sc;
      }
    }
    if (on) *reinterpret_cast<float2*>(a.work + (int64_t)t * conv_dim + c) = make_float2(y0, y1);
  }
}

// The recurrence of one (sequence, value head), its state in registers from the first token to the last: a thread
// holds 4 columns of every NG-th row. Per token two sums over the rows, across the workgroup. Bound by the states' bytes (32
// single tokens of 48 heads of 128 x 128: 201 MB in 31 us, part of it warm in the last-level cache), 2.7 us for each further token.
template <bool BF, int DK, int DV>
__global__ void __launch_bounds__(256) gdn_rec_packed_kernel(GdnPackedArgs a, int long_from) {
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
  {  // this head's share of the convolution state: every input of the step's windows has been read
    const int K = a.K;
    const uint16_t* const q = static_cast<const uint16_t*>(a.qkv) + (int64_t)sq.t0 * a.qkv_stride;
    uint16_t* const cst = static_cast<uint16_t*>(a.conv) + (int64_t)sq.row * (K - 1) * conv_dim;
    for (int c = h * 256 + tid; c < conv_dim; c += a.Hv * 256) {
      uint16_t y[kConvMax - 1];
#pragma unroll
      for (int j = 0; j < kConvMax - 1; ++j) {
        const int u = sq.n - (K - 1) + j;
        y[j] = j >= K - 1 ? 0 : u >= 0 ? q[(int64_t)u * a.qkv_stride + c] : sq.len == sq.n ? 0 : cst[(int64_t)(K - 1 + u) * conv_dim + c];
      }
#pragma unroll
      for (int j = 0; j < kConvMax - 1; ++j)
        if (j < K - 1) cst[(int64_t)j * conv_dim + c] = y[j];
    }
  }
  if (sq.n >= long_from) return;
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

// ---- long sequences: chunks of 64 tokens ----------------------------------------------------------
// With G the running sum of a chunk's logarithms of decays, S the state before it, and row vectors q_t, k_t, v_t:
//   u_t = beta_t (v_t - e^(G_t) k_t S - sum_(s<t) e^(G_t - G_s) (k_t . k_s) u_s)          u = T r, T = (1 + M)^-1
//   o_t = e^(G_t) q_t S + sum_(s<=t) e^(G_t - G_s) (q_t . k_s) u_s                        o = e^G (q S) + P u
//   S' = e^(G_C) S + sum_s e^(G_C - G_s) k_s^T u_s
// T and P depend on no state: gdn_chunk_kernel forms them for all chunks at once. What is left is a chain of products
// over the chunks (gdn_scan_kernel), split over the state's columns, which do not meet. Products are float32 matrix
// instructions, those of the state as Three; G is summed in float64, as e^(G_t - G_s) would lose bits behind tokens that forget
// nearly everything, and a token's logarithm is at least -1000.
//
// Matrix instruction j of four takes element j of 16-byte pieces: lane (g, c) = (lane / 16, lane % 16) holds A[c][4 g + j] and
// B[4 g + j][c], and C[4 g + r][c] in register r, so that a product's result is the next one's B operand as it lies.
constexpr int kChunk = 64;
constexpr int kChunkFloats = 2 * kChunk * kChunk + 3 * kChunk;  // T, P, e^G, e^(G_C - G), beta of a chunk and head

__device__ __forceinline__ f32x4 mma4(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// lane t: token t of a chunk of n
struct ChunkGate {
  float beta;
  double sum;  // G
  __device__ ChunkGate(const uint16_t* ab, int64_t stride, int n, int h, int Hv, float dtb, float sa, bool bf) {
    const int lane = threadIdx.x & 63;
    const uint16_t* const p = ab + (int64_t)min(lane, n - 1) * stride;
    const float av = (bf ? Half<true>::ld(p[h]) : Half<false>::ld(p[h])) + dtb;
    const float bv = bf ? Half<true>::ld(p[Hv + h]) : Half<false>::ld(p[Hv + h]);
    const float sp = av > 20.f ? av : log1pf(expf(av));  // softplus (torch's threshold 20)
    const float g = sa * sp;
    beta = lane < n ? 1.f / (1.f + expf(-bv)) : 0.f;
    sum = lane < n ? (g < -1000.f ? -1000.0 : (double)g) : 0.0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double u = __shfl_up(sum, o, 64);
      if (lane >= o) sum += u;
    }
  }
};

// Slots of the workspaces that hold T, P and gates of a chunk: those of a long sequence begin at slot (its first token / 64)
// + (long sequences before it), of which there are at most one for every long_from tokens.
__host__ __device__ __forceinline__ int64_t gdn_slots(int64_t N, int64_t B, int long_from) {
  const int64_t most = N / long_from;
  return N / 64 + (B < most ? B : most) + 1;
}
// whether sequences base + lane are long, and below n
__device__ __forceinline__ uint64_t long_ones(const GdnPackedArgs& a, int base, int n, int long_from) {
  const int i = base + (threadIdx.x & 63), at = min(i, a.B - 1);
  return __ballot(i < n && a.cu[at + 1] - a.cu[at] >= long_from);
}
__device__ __forceinline__ int first_slot(const GdnPackedArgs& a, int b, int long_from) {
  int n = max(a.cu[b], 0) >> 6;
  for (int base = 0; base < b; base += 64) n += __popcll(long_ones(a, base, b, long_from));
  return n;
}
// The chunk that a slot belongs to.
struct ChunkAt {
  int b = -1, c = -1;
  __device__ ChunkAt(const GdnPackedArgs& a, int slot, int long_from) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.B; base += 64) {
      const uint64_t those = long_ones(a, base, a.B, long_from);
      const int first = (max(a.cu[min(base + lane, a.B - 1)], 0) >> 6) + before + __popcll(those & ((1ull << lane) - 1));
      const uint64_t here = __ballot(first <= slot) & those;
      if (here) {  // the last of them
        const int at = 63 - __builtin_clzll(here);
        b = base + at;
        c = slot - __builtin_amdgcn_readlane(first, at);
      }
      before += __popcll(those);
    }
  }
};

// T and P of one chunk, for the value heads of one key head. The ten 16 x 16 blocks of the lower triangles of k k^T and q k^T
// are shared out over the waves; T by blocks: forward substitution in the diagonal ones, then T_ij = -T_ii (sum over
// i > l >= j of M_il T_lj), three levels of them. Bound by the stages' latencies, two workgroups to a CU: 24 us for one chunk of
// 48 heads, 104 us for 81.
template <bool BF, int DK>
__global__ void __launch_bounds__(256) gdn_chunk_kernel(GdnPackedArgs a, float* tp, int long_from) {
  constexpr int LD = kChunk + 4;
  __shared__ __attribute__((aligned(16))) float M[kChunk * LD], T[kChunk * LD], beta_s[kChunk];
  __shared__ double sum_s[kChunk];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
  const ChunkAt at(a, blockIdx.x, long_from);
  if (at.b < 0 || at.c < 0) return;
  const PackedSeq sq(a.cu, a.rows, a.lens, at.b, a.N, a.R, 0x7FFFFFFF);
  if (!sq.fine || sq.n < long_from || at.c * kChunk >= sq.n) return;
  const int n = min(kChunk, sq.n - at.c * kChunk), kh = blockIdx.y, key_dim = a.Hk * DK, conv_dim = 2 * key_dim + a.Hv * a.dv;
  const int64_t t0 = sq.t0 + at.c * kChunk;
  // block (bi, bj) p of this wave: (3,0) (3,1) (3,2) | (3,3) (2,0) (2,1) | (2,2) (1,0) | (1,1) (0,0)
  constexpr int BI[4][3] = {{3, 3, 3}, {3, 2, 2}, {2, 1, -1}, {1, 0, -1}}, BJ[4][3] = {{0, 1, 2}, {3, 0, 1}, {2, 0, -1}, {1, 0, -1}};
  int bi[3], bj[3];
  f32x4 kk[3], qk[3];
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    bi[p] = wave == 0 ? BI[0][p] : wave == 1 ? BI[1][p] : wave == 2 ? BI[2][p] : BI[3][p];
    bj[p] = wave == 0 ? BJ[0][p] : wave == 1 ? BJ[1][p] : wave == 2 ? BJ[2][p] : BJ[3][p];
    kk[p] = qk[p] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (bi[p] < 0) continue;
    const float* const qi = a.work + (t0 + min(16 * bi[p] + c, n - 1)) * conv_dim + kh * DK + 4 * g;
    const float* const kj = a.work + (t0 + min(16 * bj[p] + c, n - 1)) * conv_dim + key_dim + kh * DK + 4 * g;
#pragma unroll
    for (int s = 0; s < DK / 16; ++s) {
      const f32x4 b = *reinterpret_cast<const f32x4*>(kj + 16 * s);
      qk[p] = mma4(*reinterpret_cast<const f32x4*>(qi + 16 * s), b, qk[p]);
      kk[p] = mma4(*reinterpret_cast<const f32x4*>(qi + key_dim + 16 * s), b, kk[p]);
    }
  }
  for (int h = kh; h < a.Hv; h += a.Hk) {
    if (wave == 0) {
      const ChunkGate gate(static_cast<const uint16_t*>(a.ab) + t0 * a.ab_stride, a.ab_stride, n, h, a.Hv, a.dt_bias[h], a.ssm_a[h], BF);
      beta_s[lane] = gate.beta;
      sum_s[lane] = gate.sum;
    }
    __syncthreads();
    float* const Tg = tp + ((int64_t)blockIdx.x * a.Hv + h) * kChunkFloats;
    float* const Pg = Tg + kChunk * kChunk;
    if (wave == 1) {
      const double sum = sum_s[lane];
      float* const gates = Pg + kChunk * kChunk + lane;
      gates[0] = expf((float)sum);
      gates[kChunk] = expf((float)(sum_s[kChunk - 1] - sum));
      gates[2 * kChunk] = beta_s[lane];
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      if (bi[p] < 0) continue;
      const int s = 16 * bj[p] + c;
      const double gs = sum_s[s];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * bi[p] + 4 * g + r;
        const float ratio = s <= t ? expf((float)(sum_s[t] - gs)) : 0.f;
        M[t * LD + s] = s < t ? beta_s[t] * ratio * kk[p][r] : 0.f;
        Pg[t * kChunk + s] = s <= t ? ratio * qk[p][r] : 0.f;
      }
    }
    __syncthreads();
    {  // column c of the inverse of diagonal block `wave`, in every lane group
      const float* const D = M + 16 * wave * LD + 16 * wave;
      float x[16];
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        float v = t == c ? 1.f : 0.f;
#pragma unroll
        for (int s = 0; s < t; ++s) v -= D[t * LD + s] * x[s];
        x[t] = v;
      }
#pragma unroll
      for (int t = 0; t < 16; ++t)
        if ((t >> 2) == g) T[(16 * wave + t) * LD + 16 * wave + c] = x[t];
    }
#pragma unroll
    for (int level = 1; level < 4; ++level) {
      __syncthreads();
      const int i = level + wave, j = wave;  // block (i, j)
      if (i < 4) {
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        for (int l = j; l < i; ++l) {
          f32x4 b;
#pragma unroll
          for (int r = 0; r < 4; ++r) b[r] = T[(16 * l + 4 * g + r) * LD + 16 * j + c];
          y = mma4(*reinterpret_cast<const f32x4*>(M + (16 * i + c) * LD + 16 * l + 4 * g), b, y);
        }
        const f32x4 z = mma4(*reinterpret_cast<const f32x4*>(T + (16 * i + c) * LD + 16 * i + 4 * g), y, (f32x4){0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int r = 0; r < 4; ++r) T[(16 * i + 4 * g + r) * LD + 16 * j + c] = -z[r];
      }
    }
    __syncthreads();
    for (int i = tid; i < kChunk * kChunk / 4; i += 256) {
      const int t = i / 16, s = 4 * (i % 16);
      if (s < (t | 15)) *reinterpret_cast<f32x4*>(Tg + t * kChunk + s) = *reinterpret_cast<const f32x4*>(T + t * LD + s);
    }
    __syncthreads();
  }
}

// The chain over a sequence's chunks, for 32 columns of a value head's state: its tiles stay in registers (32 rows to each
// of the first waves), a copy in LDS is the products' operand. Wave w holds tokens 16 w .. of a chunk. The products with
// the state, and those that advance it, take their operands as three bf16 numbers (Three): float32's bits for every row and
// column whatever its neighbours are, in six 16-bit matrix instructions, 96 cycles where float32 ones would take 256; u and
// the outputs inside the chunk are float32 products. Bound by the chain: a chunk's operands come from L2 a chunk ahead, two
// workgroups to a CU.
// Columns: 64 read q, k, T and P half as often but leave one workgroup to a CU (3 prompts of 2047, 48 heads, operands of two
// fp16 numbers: 691 against 635 us for the whole call).

constexpr int kScanColumns = 32;

template <bool BF, int DK>
__global__ void __launch_bounds__(256, 2) gdn_scan_kernel(GdnPackedArgs a, const float* tp, float* ow, int long_from) {
  static_assert(kScanColumns == 32);
  constexpr int LS = DK + 8, LT = kChunk + 4, LU = kChunk + 8, COLS = kScanColumns, CT = COLS / 16;
  __shared__ __attribute__((aligned(16))) uint16_t Sh[3][COLS * LS], uh[3][COLS * LU];  // the state's copy and left u, by column
  __shared__ __attribute__((aligned(16))) float rl[COLS * LT], ul[COLS * LT];
  __shared__ int odd_s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
  const int ns = a.dv / COLS, h = blockIdx.x / ns, col0 = blockIdx.x % ns * COLS, kh = h % a.Hk, b = blockIdx.y;
  const PackedSeq sq(a.cu, a.rows, a.lens, b, a.N, a.R, 0x7FFFFFFF);
  if (!sq.fine || sq.n < long_from) return;
  const int key_dim = a.Hk * DK, conv_dim = 2 * key_dim + a.Hv * a.dv, vdim = a.Hv * a.dv, n = sq.n;
  const float* const wq = a.work + (int64_t)sq.t0 * conv_dim + kh * DK;
  const float* const wk = wq + key_dim;
  const float* const wv = a.work + (int64_t)sq.t0 * conv_dim + 2 * key_dim + h * a.dv + col0;
  float* const o_at = ow + (int64_t)sq.t0 * vdim + h * a.dv + col0;
  const uint16_t* const ab = static_cast<const uint16_t*>(a.ab) + (int64_t)sq.t0 * a.ab_stride;
  const int slot = first_slot(a, b, long_from);
  if (slot + (n + kChunk - 1) / kChunk > gdn_slots(a.N, a.B, long_from)) {  // sequences that lie over one another
    for (int i = tid; i < n * COLS; i += 256) o_at[(int64_t)(i / COLS) * vdim + i % COLS] = NAN;
    return;
  }
  const float* tg = tp + ((int64_t)slot * a.Hv + h) * kChunkFloats;
  const int64_t next = (int64_t)a.Hv * kChunkFloats;
  float* const Sg = a.rec + (((int64_t)sq.row * a.Hv + h) * DK) * a.dv + col0;
  const bool fresh = sq.len == n;
  if (tid == 0) odd_s = 0;
  // four values of a column, and where the other terms of them are
  auto put_split = [&](uint16_t* to, int term, f32x4 v) {
    uint32_t w[3][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) split3(v[2 * j], v[2 * j + 1], w[0][j], w[1][j], w[2][j]);
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<uint2*>(to + i * term) = make_uint2(w[i][0], w[i][1]);
  };
  const bool owner = 32 * wave < DK;  // of rows 32 wave .. + 31 of the state
  f32x4 st[2][CT];
  auto copy_state = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < CT; ++t) put_split(&Sh[0][(16 * t + c) * LS + 32 * wave + 16 * i + 4 * g], COLS * LS, st[i][t]);
  };
  if (owner) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        st[i][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (!fresh)
#pragma unroll
          for (int r = 0; r < 4; ++r) st[i][t][r] = Sg[(int64_t)(32 * wave + 16 * i + 4 * g + r) * a.dv + 16 * t + c];
      }
    copy_state();
  }
  // what a chunk reads from memory is asked for a chunk before it is used, when its registers have been read
  constexpr int KQ = DK / 32;
  f32x4 q4[KQ][2], k4[KQ][2], kt[2][4], v4[CT], t4[4], p4[4], grown, left, beta;
  float all;
  auto load_rows = [&](int t0) {  // tokens behind the last repeat it
    const int m = min(kChunk, n - t0);
    const int64_t row = t0 + min(16 * wave + c, m - 1);
#pragma unroll
    for (int s = 0; s < KQ; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        q4[s][e] = *reinterpret_cast<const f32x4*>(wq + row * conv_dim + 32 * s + 8 * g + 4 * e);
        k4[s][e] = *reinterpret_cast<const f32x4*>(wk + row * conv_dim + 32 * s + 8 * g + 4 * e);
      }
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) v4[t][r] = wv[(int64_t)(t0 + min(16 * wave + 4 * g + r, m - 1)) * conv_dim + 16 * t + c];
  };
  auto load_block = [&](f32x4 (&x)[4], const float* at) {
#pragma unroll
    for (int l = 0; l < 4; ++l)
      x[l] = *reinterpret_cast<const f32x4*>(at + (16 * wave + c) * kChunk + 16 * min(l, wave) + 4 * g);
  };
  auto load_columns = [&](int t0) {
    const int m = min(kChunk, n - t0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int l = 0; l < 4; ++l)
#pragma unroll
        for (int r = 0; r < 4; ++r) kt[i][l][r] = wk[(int64_t)(t0 + min(16 * l + 4 * g + r, m - 1)) * conv_dim + min(32 * wave, DK - 32) + 16 * i + c];
  };
  auto load_gates = [&](const float* at) {
    at += 2 * kChunk * kChunk;
    grown = *reinterpret_cast<const f32x4*>(at + 16 * wave + 4 * g);
    left = *reinterpret_cast<const f32x4*>(at + kChunk + 16 * wave + 4 * g);
    beta = *reinterpret_cast<const f32x4*>(at + 2 * kChunk + 16 * wave + 4 * g);
    all = at[kChunk - 1];
  };
  load_rows(0);
  load_gates(tg);
  load_block(t4, tg);
  load_block(p4, tg + kChunk * kChunk);
  load_columns(0);
  __syncthreads();
  for (int t0 = 0; t0 < n; t0 += kChunk, tg += next) {
    const int m = min(kChunk, n - t0);
    // the last chunk asks for its own again: a load that some turn of the loop leaves out would be waited for at once
    const bool more = t0 + kChunk < n;
    const int tn = more ? t0 + kChunk : t0;
    const float* const tgn = more ? tg + next : tg;
    f32x4 qs[CT], ks[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) qs[t] = ks[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KQ; ++s) {
      const Three q = split3(q4[s][0], q4[s][1]), k = split3(k4[s][0], k4[s][1]);
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        const uint16_t* const at = &Sh[0][(16 * t + c) * LS + 32 * s + 8 * g];
        const Three x = {*reinterpret_cast<const u32x4*>(at), *reinterpret_cast<const u32x4*>(at + COLS * LS),
                         *reinterpret_cast<const u32x4*>(at + 2 * COLS * LS)};
        ks[t] = mma_three(k, x, ks[t]);
        qs[t] = mma_three(q, x, qs[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < CT; ++t)
      *reinterpret_cast<f32x4*>(rl + (16 * t + c) * LT + 16 * wave + 4 * g) = beta * (v4[t] - grown * ks[t]);
    load_rows(tn);
    lds_sync();
    f32x4 u[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) u[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      if (l > wave) break;
#pragma unroll
      for (int t = 0; t < CT; ++t) u[t] = mma4(t4[l], *reinterpret_cast<const f32x4*>(rl + (16 * t + c) * LT + 16 * l + 4 * g), u[t]);
    }
    load_block(t4, tgn);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      *reinterpret_cast<f32x4*>(ul + (16 * t + c) * LT + 16 * wave + 4 * g) = u[t];
      put_split(&uh[0][(16 * t + c) * LU + 16 * wave + 4 * g], COLS * LU, u[t] * left);
    }
    lds_sync();
    f32x4 o[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) o[t] = qs[t] * grown;
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      if (l > wave) break;
#pragma unroll
      for (int t = 0; t < CT; ++t) o[t] = mma4(p4[l], *reinterpret_cast<const f32x4*>(ul + (16 * t + c) * LT + 16 * l + 4 * g), o[t]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (16 * wave + 4 * g + r < m)
#pragma unroll
        for (int t = 0; t < CT; ++t) o_at[(int64_t)(t0 + 16 * wave + 4 * g + r) * vdim + 16 * t + c] = o[t][r];
    load_block(p4, tgn + kChunk * kChunk);
    if (owner) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < CT; ++t) st[i][t] *= all;
#pragma unroll
      for (int l = 0; l < 4; l += 2) {  // tokens 16 l + 4 g .. + 3 and 16 more on, of both operands
        Three x[CT];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          auto both = [&](int term) {
            const uint16_t* const at = &uh[term][(16 * t + c) * LU + 16 * l + 4 * g];
            const uint2 lo = *reinterpret_cast<const uint2*>(at), hi = *reinterpret_cast<const uint2*>(at + 16);
            return (u32x4){lo.x, lo.y, hi.x, hi.y};
          };
          x[t] = {both(0), both(1), both(2)};
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const Three k = split3(kt[i][l], kt[i][l + 1]);
#pragma unroll
          for (int t = 0; t < CT; ++t) st[i][t] = mma_three(k, x[t], st[i][t]);
        }
      }
      copy_state();
    }
    load_columns(tn);
    load_gates(tgn);
    lds_sync();
  }
  // a u that is not finite leaves a state that is not
  bool odd = false;
  if (owner)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) odd |= !(fabsf(st[i][t][r]) <= 3.4028235e38f);
  if (odd) odd_s = 1;
  __syncthreads();
  if (!odd_s) {
    if (owner)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) Sg[(int64_t)(32 * wave + 16 * i + 4 * g + r) * a.dv + 16 * t + c] = st[i][t][r];
    return;
  }
  // A value that is not finite has reached tokens before its own through the products: once more, token by token. Thread
  // (x, y) = (tid / 32, tid % 32) holds rows x, x + 8, .. of column y.
  {
    constexpr int NR = DK / 8;
    const int x = tid >> 5, y = tid & 31;
    float s[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) s[i] = fresh ? 0.f : Sg[(int64_t)(x + 8 * i) * a.dv + y];
    auto total = [&](float v) {  // over x
      __syncthreads();
      rl[x * 32 + y] = v;
      __syncthreads();
      float r = 0.f;
      for (int i = 0; i < 8; ++i) r += rl[i * 32 + y];
      return r;
    };
    for (int t = 0; t < n; ++t) {
      const float av = Half<BF>::ld(ab[(int64_t)t * a.ab_stride + h]) + a.dt_bias[h], bv = Half<BF>::ld(ab[(int64_t)t * a.ab_stride + a.Hv + h]);
      const float sp = av > 20.f ? av : log1pf(expf(av)), decay = expf(a.ssm_a[h] * sp), beta = 1.f / (1.f + expf(-bv));
      float p = 0.f;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        s[i] *= decay;
        p += s[i] * wk[(int64_t)t * conv_dim + x + 8 * i];
      }
      const float d = (wv[(int64_t)t * conv_dim + y] - total(p)) * beta;
      p = 0.f;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        s[i] += d * wk[(int64_t)t * conv_dim + x + 8 * i];
        p += s[i] * wq[(int64_t)t * conv_dim + x + 8 * i];
      }
      const float o = total(p);
      if (x == 0) o_at[(int64_t)t * vdim + y] = o;
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) Sg[(int64_t)(x + 8 * i) * a.dv + y] = s[i];
  }
}

// Gated RMSNorm of the long sequences' outputs: a workgroup per token, dv / 8 lanes to a head, eight values each. Bound by its
// bytes: 5118 tokens of 48 heads of 128, 252 MB in 44 us (5.7 TB/s, the scan's outputs being partly in the last-level cache).
template <bool BF>
__global__ void __launch_bounds__(256) gdn_out_packed_kernel(GdnPackedArgs a, const float* ow, int long_from, bool wide) {
  using E = Half<BF>;
  const int t = blockIdx.x, b = seq_of(a.cu, a.B, t), vdim = a.Hv * a.dv, lanes = a.dv >> 3;
  if (b >= a.B) return;
  const PackedSeq sq(a.cu, a.rows, a.lens, b, a.N, a.R, 0x7FFFFFFF);
  if (!sq.fine || sq.n < long_from || t < sq.t0 || t - sq.t0 >= sq.n) return;
  const float* const o = ow + (int64_t)t * vdim;
  const uint16_t* const z = static_cast<const uint16_t*>(a.z) + (int64_t)t * a.z_stride;
  uint16_t* const out = static_cast<uint16_t*>(a.out) + (int64_t)t * a.out_stride;
  const int d = 8 * (threadIdx.x & (lanes - 1));
  float w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = E::ld(static_cast<const uint16_t*>(a.norm_w)[d + e]);
  for (int i = 8 * threadIdx.x; i < vdim; i += 2048) {  // whole heads to a wave: dv divides 512
    const f32x4 lo = *reinterpret_cast<const f32x4*>(o + i), hi = *reinterpret_cast<const f32x4*>(o + i + 4);
    u32x4 zw;
    if (wide) {
      zw = *reinterpret_cast<const u32x4*>(z + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) zw[e] = (uint32_t)z[i + 2 * e] | ((uint32_t)z[i + 2 * e + 1] << 16);
    }
    const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
    for (int m = 1; m < lanes; m <<= 1) ss += __shfl_xor(ss, m, 64);
    const float rn = 1.f / sqrtf(ss / (float)a.dv + a.eps);
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float z0 = E::ld((uint16_t)zw[e]), z1 = E::ld((uint16_t)(zw[e] >> 16));
      r[e] = E::pack((f32x2){x[2 * e] * rn * w[2 * e] * (z0 * sigmoid_raw(z0)), x[2 * e + 1] * rn * w[2 * e + 1] * (z1 * sigmoid_raw(z1))});
    }
    if (wide) {
      *reinterpret_cast<u32x4*>(out + i) = r;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) out[i + e] = (uint16_t)(r[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// Sequences from kLongFrom tokens on go by chunks (us for the whole call, one sequence of 48 heads of 128, token by token
// and by chunks: 16 tokens 47 and 44, 24 tokens 66 and 46, 64 tokens 176 and 48; 15 tokens token by token 45. Several short
// ones beside each other would be quicker token by token: eight of 16 53 and 88, eight of 24 75 and 116).
constexpr int kLongFrom = 16;

// whether a step may have long sequences, which take launches and memory of their own
static bool gdn_may_chunk(const GdnPackedArgs& a) { return a.max_new >= kLongFrom && a.B > 0; }

// convolution outputs; if there may be long sequences, T and P of their chunks and the recurrence's outputs
int64_t gdn_packed_work(const GdnPackedArgs& a) {
  const int64_t rows = (int64_t)a.N * (2 * a.Hk * a.dk + a.Hv * a.dv);
  return !gdn_may_chunk(a) ? rows : rows + gdn_slots(a.N, a.B, kLongFrom) * a.Hv * kChunkFloats + (int64_t)a.N * a.Hv * a.dv;
}

template <bool BF>
static hipError_t launch_gdn_packed_t(const GdnPackedArgs& a, hipStream_t s) {
  const int conv_dim = 2 * a.Hk * a.dk + a.Hv * a.dv;
  const bool pair = ((a.qkv_stride & 1) | (reinterpret_cast<uintptr_t>(a.qkv) & 3)) == 0;
  const dim3 rgrid((unsigned)a.Hv, (unsigned)a.B + 1);
  auto conv = [&](auto tpb, auto kw) {
    constexpr int TPB = decltype(tpb)::value;
    hipLaunchKernelGGL((gdn_conv_packed_kernel<BF, TPB, decltype(kw)::value>), dim3((unsigned)((conv_dim + 511) / 512), (unsigned)((a.N + TPB - 1) / TPB)),
                       dim3(256), 0, s, a, pair);
  };
  auto width = [&](auto tpb) {
    if (a.K == 4) conv(tpb, std::integral_constant<int, 4>{});
    else conv(tpb, std::integral_constant<int, kConvMax>{});
  };
  // tokens of a thread (us for the whole call, 1 and 8: 64 tokens 50 and 54, 256 77 and 79, 512 104 and 102, 2048 294 and 275)
  if (a.N <= 512) width(std::integral_constant<int, 1>{});
  else width(std::integral_constant<int, 8>{});
  const bool chunks = gdn_may_chunk(a);
  const int long_from = chunks ? kLongFrom : 0x7FFFFFFF;
  auto rec = [&](auto dk, auto dv) {
    if (chunks) {
      float* const tp = a.work + (int64_t)a.N * conv_dim;
      const int64_t slots = gdn_slots(a.N, a.B, kLongFrom);
      float* const ow = tp + slots * a.Hv * kChunkFloats;
      hipLaunchKernelGGL((gdn_chunk_kernel<BF, decltype(dk)::value>), dim3((unsigned)slots, (unsigned)a.Hk), dim3(256), 0, s, a, tp, long_from);
      hipLaunchKernelGGL((gdn_scan_kernel<BF, decltype(dk)::value>), dim3((unsigned)(a.Hv * (a.dv / kScanColumns)), (unsigned)a.B), dim3(256), 0, s, a,
                         (const float*)tp, ow, long_from);
      const bool wide = ((reinterpret_cast<uintptr_t>(a.z) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0 && ((a.z_stride | a.out_stride) & 7) == 0;
      hipLaunchKernelGGL(gdn_out_packed_kernel<BF>, dim3((unsigned)a.N), dim3(256), 0, s, a, (const float*)ow, long_from, wide);
    }
    hipLaunchKernelGGL((gdn_rec_packed_kernel<BF, decltype(dk)::value, decltype(dv)::value>), rgrid, dim3(256), 0, s, a, long_from);
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
