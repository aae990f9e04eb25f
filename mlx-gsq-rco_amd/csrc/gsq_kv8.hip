// An 8-bit K/V cache for the gated attention layers of the Qwen3.5-hybrid decoder: quantised as it is
// written, read back, and attended to by single tokens, prompts and trees of drafted tokens (the
// 16-bit cache of gsq_attn_decode / gsq_attn_seq holds twice the bytes; the reference runs mlx-lm's
// attention over a 16-bit cache, mlx_gsq/models/qwen35.py:114-152).
//
// A cached row of hd values x (one token, one KV head) is held as bytes u and a float32 scale s:
//   s = max |x| / 127 (rounded to float32), u = 128 + rint(x / s), x ~ (u - 128) s;
// s = 0: every u is 128; a row with a value that is not finite has s = NaN. k is quantised from its
// normalized and rotated values before any rounding to 16 bits.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "gsq_common.h"
#include "gsq_elem.h"

namespace gsq {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// the two 16-bit activation types
template <bool BF>
struct E16 {
  __device__ static float ld(uint16_t b) {
    if constexpr (BF) return __builtin_bit_cast(float, (uint32_t)b << 16);
    else return (float)__builtin_bit_cast(_Float16, b);
  }
  __device__ static uint16_t mk(float v) {
    if constexpr (BF) return (uint16_t)f32_to_bf16_bits(v);
    else return __builtin_bit_cast(uint16_t, (_Float16)v);
  }
};

// v_exp_f32: 2^x to one ulp (results below the normal range are 0)
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// 1 / (1 + e^-x) from the hardware's power of two and reciprocal, to a few ulps of float32
__device__ __forceinline__ float sigmoid_raw(float x) {
  return __builtin_amdgcn_rcpf(1.f + exp2_raw(x * -1.44269504088896340736f));
}

// True (uniformly) if row bb's new tokens do not all lie inside the cache, or its tree names a parent
// that is not an earlier token: its outputs are then NaN and its cache rows are left alone.
// Called by whole waves.
__device__ __forceinline__ bool row_invalid(const int64_t* pos, int64_t L, int S, const int32_t* parents) {
  if (pos[0] < 0 || pos[0] > L - S) return true;
  if (!parents) return false;
  const int lane = threadIdx.x & 63, p = lane < S ? parents[lane] : -1;
  return __any(p < -1 || p >= lane);
}

// The tree's paths (S <= 64 tokens, a token's parent before it, -1: the cache): in lane t the set of
// t and its ancestors as bits, by pointer doubling. Called by whole waves.
__device__ __forceinline__ uint64_t tree_path(const int32_t* parents, int S) {
  const int lane = threadIdx.x & 63;
  int p = lane < S ? parents[lane] : -1;
  uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const int src = p < 0 ? lane : p;  // a root adds itself
    lo |= __shfl(lo, src, 64);
    hi |= __shfl(hi, src, 64);
    const int pp = __shfl(p, src, 64);  // by every lane: a lane that does not run it gives 0
    p = p < 0 ? -1 : pp;
  }
  return lo | ((uint64_t)hi << 32);
}

}  // namespace

// ---- writing -----------------------------------------------------------------------------------
// One workgroup per (token, share of the heads): a wave per head row, kWriteRows rows loaded before
// the first is used. The rotary factors of the token's position are formed once per workgroup, angles
// in double. Rounding to 8 bits jumps at values next to a border, so k is formed in double and a row that has
// a quotient within 1e-4 of a border (five times what float32 can be off) divides in double too:
// the bytes are those of the definition. Bound by the arithmetic of a row (2047 tokens of 24 + 2 x 4 heads
// of 256: 60 MB in 22 us; one token of 8 rows 5.1 us).
constexpr int kWriteRows = 2;

template <bool BF, int HD>
__global__ void __launch_bounds__(256) kv8_write_kernel(Kv8WriteArgs a, bool wide) {
  using E = E16<BF>;
  constexpr int V = HD / 64;  // consecutive values per lane
  typedef uint16_t vec_t __attribute__((ext_vector_type(V)));
  typedef uint8_t bytes_t __attribute__((ext_vector_type(V)));
  __shared__ double row[4][HD], cs[HD / 2], sn[HD / 2];
  __shared__ float csf[HD / 2], snf[HD / 2];
  __shared__ int depth;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, d0 = V * lane;
  const int t = blockIdx.x, bb = blockIdx.y, hr = a.rd / 2, nh = a.H + 2 * a.Hkv, step = 4 * gridDim.z;
  const int64_t* const pos = a.pos + (int64_t)bb * a.pos_stride;
  const int32_t* const parents = a.parents ? a.parents + (int64_t)bb * a.parents_stride : nullptr;
  const int64_t r = (int64_t)bb * a.S + t;
  uint16_t* const qo = static_cast<uint16_t*>(a.q) + r * a.H * HD + d0;
  const uint16_t* const qg = static_cast<const uint16_t*>(a.qg) + r * a.qg_stride + d0;
  const uint16_t* const kn = static_cast<const uint16_t*>(a.k) + r * a.k_stride + d0;
  const uint16_t* const vn = static_cast<const uint16_t*>(a.v) + r * a.v_stride + d0;
  vec_t x[kWriteRows];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < kWriteRows; ++u) {
      const int h = min(h0 + u * step, nh - 1);
      const uint16_t* src = h < a.H ? qg + (int64_t)h * 2 * HD
                                    : (h < a.H + a.Hkv ? kn + (int64_t)(h - a.H) * HD : vn + (int64_t)(h - a.H - a.Hkv) * HD);
      if (wide) {
        x[u] = *reinterpret_cast<const vec_t*>(src);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[u][j] = src[j];
      }
    }
  };
  int h0 = blockIdx.z * 4 + wave;
  load(h0);
  if (row_invalid(pos, a.L, a.S, parents)) {
    for (int h = blockIdx.z * 4 + wave; h < a.H; h += step)
      for (int j = 0; j < V; ++j) qo[(int64_t)h * HD + j] = E::mk(__builtin_nanf(""));
    return;
  }
  if (parents) {  // rotary position: the token's depth in the tree behind the cache
    if (wave == 0) {
      const uint64_t path = tree_path(parents, a.S);
      if (lane == t) depth = __popcll(path) - 1;
    }
    __syncthreads();
  }
  const int64_t rp = pos[0] + (parents ? depth : t), slot = pos[0] + t;
  if (tid < hr) {
    double si, co;
    sincos((double)rp * a.inv_freq[tid], &si, &co);
    csf[tid] = (float)(cs[tid] = co);
    snf[tid] = (float)(sn[tid] = si);
  }
  float wq[V], wk[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    wq[j] = E::ld(static_cast<const uint16_t*>(a.q_norm_w)[d0 + j]);
    wk[j] = E::ld(static_cast<const uint16_t*>(a.k_norm_w)[d0 + j]);
  }
  __syncthreads();
  // x / rms(x) * w, rotated on its first rd dims, in T; through the wave's own row area, whose LDS
  // operations complete in order
  auto norm_rope = [&](auto zero, const vec_t& in, const float (&w)[V], auto* cs, auto* sn, auto (&f)[V]) {
    using T = decltype(zero);
    T* const rw = reinterpret_cast<T*>(row[wave]);
    T ss = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f[j] = E::ld(in[j]);
      ss += f[j] * f[j];
    }
    ss = lanes_sum(ss) * (T)(1.0 / HD) + (T)a.eps;
    T rn;
    if constexpr (sizeof(T) == 4) rn = __builtin_amdgcn_rsqf(ss);
    else rn = rsqrt(ss);
#pragma unroll
    for (int j = 0; j < V; ++j) rw[d0 + j] = f[j] = f[j] * rn * (T)w[j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int d = d0 + j;
      if (d < a.rd) {
        const int i = d < hr ? d : d - hr;
        const T other = d < hr ? -rw[d + hr] : rw[i];
        f[j] = f[j] * cs[i] + other * sn[i];
      }
    }
    __builtin_amdgcn_wave_barrier();
  };
  for (; h0 < nh; h0 += step * kWriteRows) {
    vec_t cur[kWriteRows];
#pragma unroll
    for (int u = 0; u < kWriteRows; ++u) cur[u] = x[u];
    if (h0 + step * kWriteRows < nh) load(h0 + step * kWriteRows);
#pragma unroll
    for (int u = 0; u < kWriteRows; ++u) {
      const int h = h0 + u * step;
      if (h >= nh) break;
      if (h < a.H) {
        float f[V];
        norm_rope(0.f, cur[u], wq, csf, snf, f);
        vec_t o;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = E::mk(f[j]);
        *reinterpret_cast<vec_t*>(qo + (int64_t)h * HD) = o;
        continue;
      }
      const bool isk = h < a.H + a.Hkv;
      double f[V];
      float x32[V];
      float s;
      bool bad = false;
      if (isk) {
        norm_rope(0.0, cur[u], wk, cs, sn, f);
        double mx = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          bad |= !(fabs(f[j]) <= DBL_MAX);
          mx = fmax(mx, fabs(f[j]));
          x32[j] = (float)f[j];
        }
        s = (float)(lanes_reduce(mx, [](double x, double y) { return fmax(x, y); }) / 127.0);
      } else {
        float mx = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          f[j] = x32[j] = E::ld(cur[u][j]);
          bad |= !(fabsf(x32[j]) <= FLT_MAX);
          mx = fmaxf(mx, fabsf(x32[j]));
        }
        s = (float)((double)lanes_reduce(mx, [](float x, float y) { return fmaxf(x, y); }) / 127.0);
      }
      if (__any(bad) || !(s <= FLT_MAX)) s = __builtin_nanf("");
      bytes_t o;
      if (s > 0.f) {
        const float inv = 1.f / s;  // infinite for the smallest scales: their quotients are not finite, and divided in double
        float n[V];
        bool close = false;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float t = x32[j] * inv;
          n[j] = rintf(t);
          close |= !(fabsf(t - n[j]) < 0.4999f);
        }
        if (__any(close)) {
#pragma unroll
          for (int j = 0; j < V; ++j) n[j] = (float)fmin(fmax(rint(f[j] / (double)s), -127.0), 127.0);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = (uint8_t)(128 + (int)n[j]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = 128;
      }
      const int64_t at = ((int64_t)bb * a.Hkv + (isk ? h - a.H : h - a.H - a.Hkv)) * a.L + slot;
      *reinterpret_cast<bytes_t*>((isk ? a.kc : a.vc) + at * HD + d0) = o;
      if (lane == 0) (isk ? a.ks : a.vs)[at] = s;
    }
  }
}

// ---- reading back --------------------------------------------------------------------------------
// out[b, h, j, :] = round((u - 128) s), the product in float32, of rows start .. start + n - 1 of both caches: a thread per 16
// values, K's rows first. Bound by memory: hd + 4 bytes read and hd values written per row (8 rows of 4 x 512
// positions, 25 MB, 7.8 us).
template <int DT>  // 0 float32, 1 fp16, 2 bf16
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8ReadArgs a) {
  const int per = a.hd >> 4;  // threads per row
  const int64_t half = (int64_t)a.heads * a.n * per, total = 2 * half;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const bool v = i >= half;
    const int64_t k = v ? i - half : i, r = k / per, c = 16 * (k - r * per), head = r / a.n;
    const int64_t src = head * a.L + a.start + (r - head * a.n);
    const uint4 q = *reinterpret_cast<const uint4*>((v ? a.vc : a.kc) + src * a.hd + c);
    const float s = (v ? a.vs : a.ks)[src];
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    float f[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      f[e] = (float)((int)((w[e >> 2] >> (8 * (e & 3))) & 255) - 128) * s;
      asm volatile("" : "+v"(f[e]));  // the float32 product, rounded to fp16 on its own (not in one instruction)
    }
    if constexpr (DT == 0) {
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(v ? a.v : a.k) + r * a.hd + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
    } else {
      uint32_t p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        p[e] = (uint32_t)E16<DT == 2>::mk(f[2 * e]) | ((uint32_t)E16<DT == 2>::mk(f[2 * e + 1]) << 16);
      uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(v ? a.v : a.k) + r * a.hd + c);
      o[0] = make_uint4(p[0], p[1], p[2], p[3]);
      o[1] = make_uint4(p[4], p[5], p[6], p[7]);
    }
  }
}

// ---- attention -----------------------------------------------------------------------------------
// Rows of a KV head: its rep = heads / kv_heads query heads of every token, row t rep + r for head r of
// token t. Two kernels share the arithmetic: attn_kv8_rows_kernel for few rows, attn_kv8_tile_kernel for
// many.
//
//  * Products on fp16 MFMAs, transposed: S^T = K Q^T puts a row (query) on each lane column, lane % 16,
//    and positions 16 b + 4 (lane / 16) + e of a block of 32 on its registers, which is the layout of the B
//    operand of O^T = V^T P^T: probabilities never leave their lane.
//  * A byte u with a zero byte above it is the fp16 (subnormal) number u 2^-24, which the matrix cores
//    take as it is: one v_perm expands two bytes, and K and V cost no rounding. What the 128 in u adds to a
//    score is known: -128 sum(q) starts its accumulator (queries of one sign, 4 to 16 times their spread,
//    leave fp16 outputs 0.4 per cent more error than their rounding; without the offset none, for 5 per cent of
//    the time). V's bytes lose their 128 as pairs, before the product: sums over u, with 128 times the weights'
//    sum taken off, end 1.4 to 2.8 x 2^-24 of the rows' largest values low in all dims alike, as the matrix
//    cores truncate (over u - 128: 0.3 to 0.7), which an average over 131072 positions shows (4.5e-5 of the
//    output against 1.7e-5; cost: prompt of 4096 320 -> 329 us, none where the cache's bytes bound it).
//  * The scale of a K row multiplies its scores, that of a V row its probabilities. bf16 queries are
//    scaled to fp16 by a power of two for each row: their 8 bits fit, and what falls below 2^-38 of the
//    row's largest cannot be seen in float32 sums.
//  * K's dims may be taken in any order (the sum is the same): those of a product's step are what a lane's
//    16 bytes hold. V's are spread so that a lane's piece of a row is PW neighbouring dims, each of
//    another output tile, and two rows give a pair of one tile's operand by one v_perm.
//  * The reference of the exponent moves only when a score passes it by 2^kLazy, for all rows of the
//    wave at once: mostly no rescaling and no exchange between lanes in the loop. It is a row's largest score,
//    or lower where that position's V row is small against the largest one met: then what the row's largest
//    weight is decides, as V rows that it does not see, or hardly, are not to take its weights' bits.
//  * A weight (probability times V scale, 2^kPScale over the largest V scale met) is at most 2^(kLazy + 3 +
//    kPScale) = 2^15 and held in two fp16 values (22 bits, down to 2^-25 of the unit). With one (11 bits) fp16
//    outputs would be off by 1.4 times their rounding and 3 to 9 of 100 bf16 outputs would take the other neighbour
//    (0.01 of 100 with two); it would save a third of the matrix instructions (700 bf16 tokens behind 5000: 267
//    against 310 us, a tree of 64 tokens of 4 rows 152 against 175; few rows the same).
constexpr float kLazy = 6.f;
constexpr float kPScale = 6.f;
constexpr float kLeast = 2.f;  // a row's largest weight stays above 2^kLeast
constexpr float kFar = 60.f;   // as long as its scores pass the reference by less than that

__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// v, as a value that nothing is known about: what is formed from it is formed there, not kept in a register
// through the loop around it
__device__ __forceinline__ int anew(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// A selector of v_perm in a scalar register: the compiler would keep a vector register for each.
__device__ __forceinline__ uint32_t scalar(uint32_t v) {
  asm("" : "+s"(v));
  return v;
}

// a value that is the same in every lane, in a scalar register
__device__ __forceinline__ float uniform(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

// eight bytes as an operand of u 2^-24
__device__ __forceinline__ u32x4 bytes8(uint32_t w0, uint32_t w1) {
  const uint32_t lo = scalar(0x0C010C00u), hi = scalar(0x0C030C02u);
  return (u32x4){__builtin_amdgcn_perm(0, w0, lo), __builtin_amdgcn_perm(0, w0, hi), __builtin_amdgcn_perm(0, w1, lo),
                 __builtin_amdgcn_perm(0, w1, hi)};
}
// byte i of two dwords as a pair of (u - 128) 2^-24 (fp16 sums of subnormal numbers are exact)
__device__ __forceinline__ uint32_t byte_pair(uint32_t second, uint32_t first, int i) {
  const uint32_t u = __builtin_amdgcn_perm(second, first, scalar(0x0C000C00u | (uint32_t)((4 + i) << 16) | (uint32_t)i));
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, u) + (f16x2){(_Float16)-0x1p-17f, (_Float16)-0x1p-17f});
}

// blocks of 32 positions that rows up to token t see
__device__ __forceinline__ int kv8_blocks(int64_t pos, int t) { return (int)((pos + t) / 32) + 1; }
// blocks of a split, for workgroups of rt rows: whole tiles of two where those are what the kernel takes
__device__ __forceinline__ int kv8_per_split(int nblk, int nsplit, int rt) {
  const int per = (nblk + nsplit - 1) / nsplit;
  return rt > 16 ? (per + 1) & ~1 : per;
}

// What a workgroup is asked to do: 16 NT rows of one (batch row, KV head), positions of one split.
template <int RT>
struct Kv8Task {
  const int64_t* posp;
  const int32_t* parents;
  int rep, R, kvh, z, bb, r0, tfirst, tlast, blk0, blk1;
  int64_t pos, base;
  __device__ explicit Kv8Task(const Kv8AttnArgs& a) {
    rep = a.H / a.Hkv;
    R = a.S * rep;
    const int ntile = (R + RT - 1) / RT;
    kvh = blockIdx.x % a.Hkv;  // consecutive workgroups: other KV heads, then other splits of the same rows
    const int rest = blockIdx.x / a.Hkv;
    z = rest % a.nsplit;
    r0 = (ntile - 1 - rest / a.nsplit) * RT;  // the last rows see most: first
    bb = blockIdx.y;
    posp = a.pos + (int64_t)bb * a.pos_stride;
    parents = a.parents ? a.parents + (int64_t)bb * a.parents_stride : nullptr;
    base = ((int64_t)bb * a.Hkv + kvh) * a.L;
    tfirst = r0 / rep;
    tlast = min(r0 + RT - 1, R - 1) / rep;
  }
  // the blocks of this split; false if there are none
  __device__ bool blocks(const Kv8AttnArgs& a) {
    pos = posp[0];
    const int nblk = kv8_blocks(pos, tlast), per = kv8_per_split(nblk, a.nsplit, RT);
    blk0 = z * per;
    blk1 = min(nblk, blk0 + per);
    return blk0 < blk1;
  }
  // row r of this KV head in q, qg and out
  __device__ int64_t row_at(const Kv8AttnArgs& a, int r, int64_t stride, int width) const {
    const int t = r / rep;
    return ((int64_t)bb * a.S + t) * stride + (int64_t)(kvh * rep + r - t * rep) * width;
  }
};

// NaN outputs of a batch row that is not served
template <bool BF, int HD, int RT>
__device__ __forceinline__ void kv8_nan_rows(const Kv8AttnArgs& a, const Kv8Task<RT>& w) {
  if (a.nsplit == 1)  // else the merge writes them
    for (int i = threadIdx.x; i < RT * HD; i += blockDim.x)
      if (w.r0 + i / HD < w.R)
        static_cast<uint16_t*>(a.out)[w.row_at(a, w.r0 + i / HD, a.out_stride, HD) + i % HD] = E16<BF>::mk(__builtin_nanf(""));
}

// Queries of the task to LDS in operand order (16 bytes per lane, step and 16-row tile), with each row's
// factor (2^24 over its power of two) and bias; HD / 8 threads a row. All threads of the workgroup.
template <bool BF, int HD, int RT>
__device__ __forceinline__ void kv8_stage_q(const Kv8AttnArgs& a, const Kv8Task<RT>& k, u32x4* qs, float* rowc_s, float* bias_s) {
  using E = E16<BF>;
  constexpr int TR = HD / 8, KS = HD / 32;
#pragma unroll 1
  for (int i = threadIdx.x; i < RT * TR; i += blockDim.x) {
    const int r = i / TR, o = i % TR;  // octet o: dims 8 o .. + 7
    u32x4 w = {0, 0, 0, 0};
    if (k.r0 + r < k.R)
      w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + k.row_at(a, k.r0 + r, a.q_stride, HD) + 8 * o);
    float v[8], sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = E::ld((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
    int ex = 0;
    if constexpr (BF) {
      float mx = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(v[e]));
#pragma unroll
      for (int x = 1; x < TR; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
      if (mx > 0.f && mx <= FLT_MAX) ex = 14 - ilogbf(mx);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], ex);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pack_h2(v[2 * e], v[2 * e + 1]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += v[e];
#pragma unroll
    for (int x = 1; x < TR; x <<= 1) sum += __shfl_xor(sum, x, 64);
    // dims 64 s + 16 g + 8 h: step 2 s + h of lane group g
    const int ks = 2 * (o >> 3) + (o & 1);
    qs[((r >> 4) * KS + ks) * 64 + 16 * ((o >> 1) & 3) + (r & 15)] = w;
    if (o == 0) {
      rowc_s[r] = ldexpf(1.f, 24 - ex);
      bias_s[r] = -sum * 0x1p-17f;
    }
  }
}

// The softmax and the sums of a wave's 16 NT rows over the blocks it has seen.
template <bool BF, int HD, int NT>
struct Kv8Rows {
  static constexpr int VB = HD / 16, TERMS = 2;  // output tiles; fp16 values that hold a weight
  float rowc[NT], m[NT], l[NT];
  float* tops;  // LDS, row 16 n + c: power of two of the row's largest weight, as of the last move of its reference
  bool unset[NT];  // the row has seen no position yet: m is 0
  bool pending;    // some row of the wave is unset
  float vref, vunit;  // power of two below the largest V scale met (the weights' unit), and 2^kPScale over it
  f32x4 acc[NT][VB];

  __device__ void init(const float* rowc_s) {
    pending = true;
    vref = 0x1p-120f;
    vunit = 0x1p126f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      rowc[n] = rowc_s[16 * n];
      m[n] = l[n] = 0.f;
      unset[n] = true;
#pragma unroll
      for (int i = 0; i < VB; ++i) acc[n][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
  }
  __device__ void init_tops(float* p) {
    tops = p;
#pragma unroll
    for (int n = 0; n < NT; ++n) tops[16 * n + (threadIdx.x & 15)] = -INFINITY;
  }
  // factor of K's scales: fp16 queries need none of their own
  __device__ static float key_factor() { return 1.44269504088896340736f / sqrtf((float)HD) * (BF ? 1.f : 0x1p24f); }

  // Scales (ks, vs) of one position a lane, as the sums take them. A V row that is not finite makes the scores of
  // its position NaN and has no weight, so that it does not reach the rows that do not see it (0 x NaN
  // would).
  __device__ void scales(float& ks, float& vs) {
    const bool fine = fabsf(vs) <= FLT_MAX;
    ks = fine ? ks * key_factor() : __builtin_nanf("");
    vs = fine ? vs : 0.f;
    if (__any(vs > vref * 8.f)) {
      float x = vs;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
      const int ex = ilogbf(uniform(x)), c = anew(threadIdx.x) & 15;
      const float d = (float)(ex - ilogbf(vref));
      vref = uniform(ldexpf(1.f, ex));
      vunit = uniform(ldexpf(exp2_raw(kPScale), -ex));
      // the new unit comes off a row's reference, its weights stay as they are; off the weights only where
      // the row's sum would leave float32
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float down = unset[n] ? 0.f : fminf(fmaxf(floorf(kFar + 20.f - __builtin_amdgcn_logf(sum(n))), 0.f), d);
        const float f = exp2_raw(down - d);
        m[n] -= down;
        l[n] *= exp2_raw(down);
        tops[16 * n + c] = tops[16 * n + c] + (down - d);
#pragma unroll
        for (int i = 0; i < VB; ++i) acc[n][i] *= f;
      }
    }
    vs *= vunit;
  }

  // scores s of a block from position j0 on to weights pf; ks4, vs4: scales() of this lane's positions; rows
  // r0 + lane % 16 + 16 n; masked: some position may lie behind a row's token, or off its path
  template <int RT, int NB>  // NB: groups of 16 positions
  __device__ void weights(const Kv8AttnArgs& a, const Kv8Task<RT>& k, int r0, int64_t j0, bool masked, const uint64_t* paths,
                          f32x4 (&s)[NT][NB], const f32x4 (&ks4)[NB], const f32x4 (&vs4)[NB], u32x4 (&pf)[NB / 2][TERMS][NT]) {
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[n][b][e] = __builtin_fmaf(BF ? s[n][b][e] * rowc[n] : s[n][b][e], ks4[b][e], -m[n]);
    if (masked) {
      const int node0 = (int)max(min(j0 - k.pos, (int64_t)1 << 30), -((int64_t)1 << 30)) + 4 * g;  // negative: cached positions
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int tok = min(r0 + 16 * n + c, k.R - 1) / k.rep;
        uint64_t path = 0;
        if (k.parents) path = paths[tok];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int node = node0 + 16 * b + e;
            const bool see = node <= tok && (!k.parents || node < 0 || ((path >> (node & 63)) & 1));
            s[n][b][e] = see ? s[n][b][e] : -INFINITY;
          }
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < NT; ++n) mx = fmaxf(mx, s[n][b][e]);
    if (pending || __any(mx > kLazy)) {
      bool left = false;
      const int row = anew(threadIdx.x) & 15;
      float xs[NT], ys[NT];  // largest scores and weights of the rows
#pragma unroll
      for (int n = 0; n < NT; ++n) xs[n] = ys[n] = -INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = __builtin_amdgcn_logf(vs4[b][e]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            xs[n] = fmaxf(xs[n], s[n][b][e]);
            ys[n] = fmaxf(ys[n], s[n][b][e] + v);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x = xs[n], y = ys[n];
        x = fmaxf(x, __shfl_xor(x, 16, 64));
        x = fmaxf(x, __shfl_xor(x, 32, 64));
        y = fmaxf(y, __shfl_xor(y, 16, 64));
        y = fmaxf(y, __shfl_xor(y, 32, 64));
        y = fmaxf(y, tops[16 * n + row]);
        // to the largest score, as far as weights of 2^kLeast remain (they are at most 2^(x + 3 + kPScale))
        const float to = fmaxf(fminf(x, y - kLeast), x - kFar);
        const float up = unset[n] ? (x == -INFINITY ? 0.f : to) : fmaxf(to, 0.f);
        const float alpha = unset[n] ? 1.f : exp2_raw(-up);
        tops[16 * n + row] = y - up;
        unset[n] = unset[n] && x == -INFINITY;
        left |= unset[n];
        m[n] += up;
        l[n] *= alpha;
#pragma unroll
        for (int i = 0; i < VB; ++i) acc[n][i] *= alpha;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][b][e] -= up;
      }
      pending = __any(left);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = exp2_raw(s[n][b][e]);
          l[n] += p;
          w[e] = p * vs4[b][e];
        }
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const f16x2 hi = __builtin_convertvector((f32x2){w[e], w[e + 1]}, f16x2);
            pf[b / 2][t][n][2 * (b & 1) + e / 2] = __builtin_bit_cast(uint32_t, hi);
            w[e] -= (float)hi.x;  // what the term leaves, for the next one
            w[e + 1] -= (float)hi.y;
          }
      }
  }
  // output tile i += V's operand times the weights
  __device__ void add(int i, u32x4 vf, const u32x4 (&pf)[TERMS][NT]) {
#pragma unroll
    for (int t = 0; t < TERMS; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n][i] = mma16(vf, pf[t][n], acc[n][i]);
  }
  // what leaves the kernel are averages of V rows, which float32 holds whatever the rows' size; sums of rows near its
  // largest number it would not: acc over a row's sum l (0: no position), then vref
  __device__ static float over(float l) { return l == 0.f ? 0.f : exp2_raw(24.f - kPScale) / l; }
  __device__ float top(int n) const { return unset[n] ? -FLT_MAX : m[n]; }
  __device__ float sum(int n) const {  // over the lanes of a row
    const float x = l[n] + __shfl_xor(l[n], 16, 64);
    return x + __shfl_xor(x, 32, 64);
  }
};

// N (4 or 8) gated outputs of a row, from dim d on
template <bool BF, int N>
__device__ __forceinline__ void kv8_out(const uint16_t* gate, uint16_t* out, const float (&o)[N]) {
  using E = E16<BF>;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const uint2 gw = *reinterpret_cast<const uint2*>(gate + i);
    const uint16_t gv[4] = {(uint16_t)gw.x, (uint16_t)(gw.x >> 16), (uint16_t)gw.y, (uint16_t)(gw.y >> 16)};
    uint32_t q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = E::mk(o[i + e] * sigmoid_raw(E::ld(gv[e])));
    *reinterpret_cast<uint2*>(out + i) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
  }
}

// Few rows (16 a workgroup): the cache goes by once, and its bytes bound the kernel. Four waves take the
// blocks in turn, each with a softmax of its own; K and V go from memory to registers in 16-byte pieces,
// a block ahead, and are expanded there: no LDS and no barrier in the loop. The waves are merged at the end.
// One token of 24 heads over 131071 positions (4 KV heads of 256, 272 MB): 44 us, 6.2 TB/s with part of it in
// the last-level cache; 32 rows of 4096 to 8191 positions (414 MB) 76 us. Over 300 positions 11 us, all of it
// latency: position, queries and first blocks, two more blocks, gates.
template <bool BF, int HD>
__global__ void __launch_bounds__(256, 2) attn_kv8_rows_kernel(Kv8AttnArgs a) {
  constexpr int KS = HD / 32, KL = HD / 64, VB = HD / 16, RT = 16;  // VB: bytes of a lane's V piece
  typedef uint32_t vpiece __attribute__((ext_vector_type(VB / 4)));
  extern __shared__ __attribute__((aligned(16))) uint8_t kv8_lds[];
  // queries, row factors and biases, scales of a wave's block, largest weights; the merge of the waves takes the same memory
  u32x4* const qs = reinterpret_cast<u32x4*>(kv8_lds);
  float* const rowc_s = reinterpret_cast<float*>(kv8_lds + RT * HD * 2);
  float* const bias_s = rowc_s + RT;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  float* const sc = bias_s + RT + wave * 64;
  const int g = lane >> 4, c = lane & 15;
  Kv8Task<RT> k(a);
  if (row_invalid(k.posp, a.L, a.S, k.parents)) {
    kv8_nan_rows<BF, HD>(a, k);
    return;
  }
  if (!k.blocks(a)) return;  // the merge knows
  const int64_t klast = k.pos + k.tlast;  // last position any row sees; later ones of a block repeat it
  u32x4 kr[2][KL];
  vpiece vr[8];
  float scv = 0.f;  // lane l < 32: K scale of position l of the block; else V scale of l - 32
  auto load_k = [&](int blk) {
    const int64_t j0 = (int64_t)blk * 32;
    const int left = (int)min(klast - j0, (int64_t)31);
    const uint8_t* p = a.kc + (k.base + j0) * HD + 16 * g;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int s = 0; s < KL; ++s) kr[b][s] = *reinterpret_cast<const u32x4*>(p + min(16 * b + c, left) * HD + 64 * s);
  };
  auto load_v = [&](int blk) {
    const int64_t j0 = (int64_t)blk * 32;
    const int left = (int)min(klast - j0, (int64_t)31);
    const uint8_t* p = a.vc + (k.base + j0) * HD + VB * c;
#pragma unroll
    for (int i = 0; i < 8; ++i) vr[i] = *reinterpret_cast<const vpiece*>(p + min(16 * (i >> 2) + 4 * g + (i & 3), left) * HD);
  };
  auto load_s = [&](int blk) {
    const int64_t j0 = (int64_t)blk * 32;
    const int left = (int)min(klast - j0, (int64_t)31);
    scv = (lane < 32 ? a.ks : a.vs)[k.base + j0 + min(lane & 31, left)];
  };
  int blk = k.blk0 + wave;
  if (blk < k.blk1) {
    load_k(blk);
    load_v(blk);
    load_s(blk);
  }
  __shared__ uint64_t paths[64];
  if (k.parents && wave == 0) paths[lane] = tree_path(k.parents, a.S);
  kv8_stage_q<BF, HD>(a, k, qs, rowc_s, bias_s);
  __syncthreads();
  u32x4 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = qs[s * 64 + lane];
  Kv8Rows<BF, HD, 1> rows;
  rows.init(rowc_s + c);
  rows.init_tops(bias_s + RT + 256 + wave * 16);
  const float bias = bias_s[c];
  for (; blk < k.blk1; blk += 4) {
    const bool more = blk + 4 < k.blk1;
    // scales of the block's positions to the lanes that hold them (the wave's LDS operations are in order)
    {
      const float other = __shfl_xor(scv, 32, 64);
      float x = lane < 32 ? scv : 0.f, y = lane < 32 ? other : scv;
      rows.scales(x, y);
      sc[lane] = lane < 32 ? x : y;
    }
    __builtin_amdgcn_wave_barrier();
    f32x4 ks4[2], vs4[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      ks4[b] = *reinterpret_cast<const f32x4*>(sc + 16 * b + 4 * g);
      vs4[b] = *reinterpret_cast<const f32x4*>(sc + 32 + 16 * b + 4 * g);
    }
    __builtin_amdgcn_wave_barrier();
    if (more) load_s(blk + 4);
    f32x4 s[1][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[0][b] = (f32x4){bias, bias, bias, bias};
#pragma unroll
      for (int st = 0; st < KS; ++st)
        s[0][b] = mma16(bytes8(kr[b][st >> 1][2 * (st & 1)], kr[b][st >> 1][2 * (st & 1) + 1]), qf[st], s[0][b]);
    }
    if (more) load_k(blk + 4);
    const int64_t j0 = (int64_t)blk * 32;
    u32x4 pf[1][Kv8Rows<BF, HD, 1>::TERMS][1];
    rows.weights(a, k, k.r0, j0, k.parents ? j0 + 31 >= k.pos : j0 + 31 > k.pos + k.tfirst, paths, s, ks4, vs4, pf);
#pragma unroll
    for (int i = 0; i < VB; ++i)  // dim VB c + i of the 8 positions: byte i & 3 of dword i / 4 of each row
      rows.add(i, (u32x4){byte_pair(vr[1][i >> 2], vr[0][i >> 2], i & 3), byte_pair(vr[3][i >> 2], vr[2][i >> 2], i & 3),
                          byte_pair(vr[5][i >> 2], vr[4][i >> 2], i & 3), byte_pair(vr[7][i >> 2], vr[6][i >> 2], i & 3)}, pf[0]);
    if (more) load_v(blk + 4);
  }
  // merge of the waves: every wave's maximum, sum and outputs over its own sum
  constexpr int OS = HD + 4;
  float* const mo = reinterpret_cast<float*>(kv8_lds);             // [4][16][OS]
  float2* const ml = reinterpret_cast<float2*>(mo + 4 * 16 * OS);  // [4][16]
  const float ls = rows.sum(0), over = rows.over(ls), vref = rows.vref;
  __syncthreads();  // queries and scales are no longer read
  float* const mine = mo + (wave * 16 + c) * OS;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int i = 0; i < VB; i += 4)
      *reinterpret_cast<f32x4*>(mine + VB * (4 * g + e) + i) =
          (f32x4){rows.acc[0][i][e], rows.acc[0][i + 1][e], rows.acc[0][i + 2][e], rows.acc[0][i + 3][e]} * over * vref;
  if (g == 0) ml[wave * 16 + c] = make_float2(rows.top(0), ls);
  __syncthreads();
  for (int i = tid; i < 16 * HD / 4; i += 256) {
    const int rr = i / (HD / 4), d = 4 * (i % (HD / 4)), r = k.r0 + rr;
    if (r >= k.R) continue;
    float mm = -FLT_MAX, ll = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[w * 16 + rr].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 x = ml[w * 16 + rr];
      f[w] = x.y * exp2_raw(x.x - mm);
      ll += f[w];
    }
    const float inv = ll == 0.f && a.nsplit > 1 ? 0.f : 1.f / ll;  // no weight at all: NaN, unless another split has one
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) o += *reinterpret_cast<const f32x4*>(mo + (w * 16 + rr) * OS + d) * (f[w] * inv);
    if (a.nsplit > 1) {
      const int64_t all = (int64_t)a.B * a.Hkv * k.R, at = (((int64_t)k.bb * a.Hkv + k.kvh) * k.R + r) * a.nsplit + k.z;
      *reinterpret_cast<f32x4*>(a.part + at * HD + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(a.part + all * a.nsplit * HD + 2 * at) = make_float2(mm, ll);
    } else {
      const float v[4] = {o[0], o[1], o[2], o[3]};
      kv8_out<BF, 4>(static_cast<const uint16_t*>(a.qg) + k.row_at(a, r, a.qg_stride, 2 * HD) + HD + d,
                     static_cast<uint16_t*>(a.out) + k.row_at(a, r, a.out_stride, HD) + d, v);
    }
  }
}

// steps of a wave's queries that attn_kv8_tile_kernel reads from LDS
constexpr int kv8_lds_steps(int hd) { return hd == 256 ? 1 : 0; }

// Many rows: 16 NT a wave, four waves to a workgroup, over tiles of 64 positions whose bytes come to LDS by
// DMA, a tile ahead (two buffers, one barrier a tile), and are read by every wave: 16 bytes of K or PW of V a
// lane at a time, expanded in registers.
//  * K's 16-byte pieces are XOR-swizzled by position, V's pieces (or rows) by bits 2 and 3 of it, so that the
//    lanes of a read fall on different banks; the DMA's source address does it.
//  * What bounds it are vector instructions and matrix cores: at head dim 256 a wave's 32 rows and a block of 32
//    positions take 96 MFMAs (1536 cycles) and about 390 vector instructions (192 of them
//    expand bytes), two waves a SIMD overlapping them in part. Matrix instructions go at raised priority
//    (353 -> 346 us). The accumulators and queries of two waves a SIMD fill the 512 registers: what the loop
//    does not need in them lies in LDS (a step of the queries, biases, scales, paths, largest weights), as spills would wait for the
//    DMA in flight (413 -> 370).
//  * 4096 tokens of 24 heads of 256 in fp16 350 us (0.59 PFLOP/s without the second term of the weights; a large
//    library product 1.31), of which a fifth is the triangle's tail; 700 bf16 tokens of 2 x 32 heads of 128 behind
//    5000 positions 322 (352 workgroups on 256 CUs); a tree of 64 tokens of 4 rows behind 8000 to 16000 162 + 16.
template <bool BF, int HD, int NT>
__global__ void __launch_bounds__(256, 2) attn_kv8_tile_kernel(Kv8AttnArgs a) {
  constexpr int KS = HD / 32, VB = HD / 16, RT = 64 * NT, NC = HD / 16;  // NC: 16-byte pieces of a row
  constexpr int PW = VB < 8 ? VB : 8, NP = VB / PW;                      // dims of a V piece, pieces of a lane
  constexpr int SH = HD == 256 ? 0 : (HD == 128 ? 1 : 2);                // 2^SH rows to the 64 banks
  constexpr int KB = HD == 256 || NT == 4 ? 1 : 2;  // blocks of 32 positions in one step, as the registers allow
  constexpr int TB = 64 * HD;                                           // bytes of a tile of K or V
  typedef uint32_t vpiece __attribute__((ext_vector_type(PW / 4)));
  extern __shared__ __attribute__((aligned(16))) uint8_t kv8_lds[];
  // two buffers of [K tile | V tile | K scales | V scales], then QL steps of the queries, for which there are
  // not enough registers; all queries pass through before the first tile
  constexpr int BUF = 2 * TB + 512, QL = kv8_lds_steps(HD);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  Kv8Task<RT> k(a);
  if (row_invalid(k.posp, a.L, a.S, k.parents)) {
    kv8_nan_rows<BF, HD>(a, k);
    return;
  }
  if (!k.blocks(a)) return;  // the merge knows
  const int64_t klast = k.pos + k.tlast;
  u32x4 qf[NT][KS];
  u32x4* const ql = reinterpret_cast<u32x4*>(kv8_lds + 2 * BUF) + wave * NT * QL * 64 + lane;
  float* const sw = reinterpret_cast<float*>(kv8_lds + 2 * BUF + 4096 * NT * QL) + wave * 128;  // the wave's scales
  // the rows' biases as the first accumulator of their scores
  f32x4* const bl = reinterpret_cast<f32x4*>(kv8_lds + 2 * BUF + 4096 * NT * QL + 2048) + wave * NT * 16;
  uint64_t* const paths = reinterpret_cast<uint64_t*>(kv8_lds + 2 * BUF + 4096 * NT * QL + 2048 + 1024 * NT);  // of a tree
  Kv8Rows<BF, HD, NT> rows;
  {
    u32x4* const qs = reinterpret_cast<u32x4*>(kv8_lds);
    float* const rowc_s = reinterpret_cast<float*>(kv8_lds + RT * HD * 2);
    float* const bias_s = rowc_s + RT;
    kv8_stage_q<BF, HD>(a, k, qs, rowc_s, bias_s);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[n][s] = qs[((wave * NT + n) * KS + s) * 64 + lane];
    rows.init(rowc_s + 16 * NT * wave + c);
    float bias[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) bias[n] = bias_s[16 * (NT * wave + n) + c];
    __syncthreads();  // the buffers, and what lies behind them, may be written
    rows.init_tops(reinterpret_cast<float*>(paths + 64) + wave * 16 * NT);
    if (k.parents && wave == 0) paths[lane] = tree_path(k.parents, a.S);
#pragma unroll
    for (int n = 0; n < NT; ++n)
      if (g == 0) bl[16 * n + c] = (f32x4){bias[n], bias[n], bias[n], bias[n]};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int s = 0; s < QL; ++s) ql[(n * QL + s) * 64] = qf[n][s];
  }
  // tile of blocks blk, blk + 1; positions past the last repeat it. Piece i of a wave: 64 / NC rows from
  // 16 wave + i 64 / NC on, NC lanes a row.
  auto issue = [&](int blk, uint8_t* buf) {
    const int64_t j0 = (int64_t)blk * 32;
    const int left = (int)min(klast - j0, (int64_t)63);
    const uint8_t* const kp = a.kc + (k.base + j0) * HD;
    const uint8_t* const vp = a.vc + (k.base + j0) * HD;
    const int ln = anew(lane), first = 16 * wave + ln / NC;
#pragma unroll
    for (int i = 0; i < NC / 4; ++i) {
      const int row = first + i * (64 / NC), o = (ln ^ (4 * i + (ln >> 4))) & (NC - 1);
      // V: rows of 128 and 64 bytes change places, 16-byte pieces of longer ones
      const int vrow = row ^ (HD == 128 ? (ln >> 5) & 1 : (HD == 64 ? ln >> 4 : 0)), vo = (ln ^ (HD == 256 ? 8 * (i & 1) : 0)) & (NC - 1);
      uint8_t* const dst = buf + (wave * (NC / 4) + i) * 1024;
      __builtin_amdgcn_global_load_lds(kp + (uint32_t)(min(row, left) * HD + 16 * o), (lds_ptr_t)dst, 16, 0, 0);
      __builtin_amdgcn_global_load_lds(vp + (uint32_t)(min(vrow, left) * HD + 16 * vo), (lds_ptr_t)(dst + TB), 16, 0, 0);
    }
    if (wave < 2)
      __builtin_amdgcn_global_load_lds((wave ? a.vs : a.ks) + k.base + j0 + (uint32_t)min(ln, left),
                                       (lds_ptr_t)(buf + 2 * TB + wave * 256), 4, 0, 0);
  };
  const int r0 = k.r0 + 16 * NT * wave;
  const int64_t pfirst = k.pos + min(r0, k.R - 1) / k.rep, plast = k.pos + min(r0 + 16 * NT - 1, k.R - 1) / k.rep;
  const bool on = r0 < k.R;
  issue(k.blk0, kv8_lds);
  int cur = 0;
  for (int blk = k.blk0; blk < k.blk1; blk += 2, cur ^= 1) {
    // the tile has landed; every wave is done with the other buffer
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (blk + 2 < k.blk1) issue(blk + 2, kv8_lds + (cur ^ 1) * BUF);
    const uint8_t* const kt = kv8_lds + cur * BUF;
    if (on && (int64_t)blk * 32 <= plast) {
      float x = reinterpret_cast<const float*>(kt + 2 * TB)[lane], y = reinterpret_cast<const float*>(kt + 2 * TB)[64 + lane];
      rows.scales(x, y);
      sw[lane] = x;
      sw[64 + lane] = y;
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll 1
    for (int sb = 0; sb < 2; sb += KB) {
      const int64_t j0 = (int64_t)(blk + sb) * 32;
      if (!on || blk + sb >= k.blk1 || j0 > plast) continue;
      const int ln = anew(lane), g = ln >> 4, c = ln & 15;
      const uint8_t* const kb = kt + (32 * sb + c) * HD;
      const uint8_t* const vb = kt + TB;
      const float* const sc = sw + 32 * sb + 4 * g;
      f32x4 s[NT][2 * KB];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n][0] = bl[16 * n + c];
#pragma unroll
        for (int b = 1; b < 2 * KB; ++b) s[n][b] = s[n][0];
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int st = 0; st < KS / 2; ++st) {
        u32x4 w[2 * KB];
#pragma unroll
        for (int b = 0; b < 2 * KB; ++b)  // position 32 sb + 16 b + c: its swizzle does not depend on sb and b
          w[b] = *reinterpret_cast<const u32x4*>(kb + 16 * b * HD + 16 * ((4 * st + g) ^ ((c >> SH) & (NC - 1))));
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int b = 0; b < 2 * KB; ++b) {
            const u32x4 kf = bytes8(w[b][2 * h], w[b][2 * h + 1]);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              s[n][b] = mma16(kf, 2 * st + h < QL ? ql[(n * QL + 2 * st + h) * 64] : qf[n][2 * st + h], s[n][b]);
          }
      }
      __builtin_amdgcn_s_setprio(0);
      if constexpr (HD == 256) __builtin_amdgcn_sched_barrier(0);  // what follows needs the registers of K's pieces
      f32x4 ks4[2 * KB], vs4[2 * KB];
#pragma unroll
      for (int b = 0; b < 2 * KB; ++b) {
        ks4[b] = *reinterpret_cast<const f32x4*>(sc + 16 * b);
        vs4[b] = *reinterpret_cast<const f32x4*>(sc + 64 + 16 * b);
      }
      u32x4 pf[KB][Kv8Rows<BF, HD, NT>::TERMS][NT];
      const int64_t end = j0 + 32 * KB - 1;
      rows.weights(a, k, r0, j0, k.parents ? end >= k.pos : end > pfirst, paths, s, ks4, vs4, pf);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int q = 0; q < KB; ++q)
#pragma unroll
        for (int h = 0; h < NP; ++h) {
          vpiece v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = 32 * (sb + q) + 16 * (i >> 2) + 4 * g + (i & 3);
            const int row = HD == 256 ? key : key ^ (g & ((1 << SH) - 1));
            const int at = HD == 256 ? ((128 * h + PW * c) ^ ((g & 1) << 7)) : PW * c;
            v[i] = *reinterpret_cast<const vpiece*>(vb + row * HD + at);
          }
#pragma unroll
          for (int i = 0; i < PW; ++i)  // dim (HD / NP) h + PW c + i of the 8 positions
            rows.add(PW * h + i,
                     (u32x4){byte_pair(v[1][i >> 2], v[0][i >> 2], i & 3), byte_pair(v[3][i >> 2], v[2][i >> 2], i & 3),
                             byte_pair(v[5][i >> 2], v[4][i >> 2], i & 3), byte_pair(v[7][i >> 2], v[6][i >> 2], i & 3)},
                     pf[q]);
        }
    }
    __builtin_amdgcn_s_setprio(0);
  }
  // a lane's outputs: row r0 + 16 n + c, dims (HD / NP) h + PW (4 g + e) + i
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + 16 * n + c;
    const float ls = rows.sum(n), vref = rows.vref;
    const float over = ls == 0.f && a.nsplit == 1 ? __builtin_nanf("") : rows.over(ls);
    if (r >= k.R) continue;
    const int64_t all = (int64_t)a.B * a.Hkv * k.R, at = (((int64_t)k.bb * a.Hkv + k.kvh) * k.R + r) * a.nsplit + k.z;
    if (a.nsplit > 1 && g == 0) *reinterpret_cast<float2*>(a.part + all * a.nsplit * HD + 2 * at) = make_float2(rows.top(n), ls);
    const uint16_t* const gate = static_cast<const uint16_t*>(a.qg) + k.row_at(a, r, a.qg_stride, 2 * HD) + HD;
    uint16_t* const out = static_cast<uint16_t*>(a.out) + k.row_at(a, r, a.out_stride, HD);
#pragma unroll
    for (int h = 0; h < NP; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = HD / NP * h + PW * (4 * g + e);
        float o[PW];
#pragma unroll
        for (int i = 0; i < PW; ++i) o[i] = rows.acc[n][PW * h + i][e] * over * vref;
        if (a.nsplit > 1) {
#pragma unroll
          for (int i = 0; i < PW; i += 4)
            *reinterpret_cast<f32x4*>(a.part + at * HD + d + i) = (f32x4){o[i], o[i + 1], o[i + 2], o[i + 3]};
        } else {
          kv8_out<BF, PW>(gate + d, out + d, o);
        }
      }
  }
}

// Outputs of split positions: a workgroup per row, a wave to every eight splits (up to 16 waves); each wave weighs
// those of its splits that hold positions of the row's tile by their share of its sum, and the waves meet
// in LDS. Bound by the latency of one read of the partial outputs, all in flight at once (128 splits of 24 rows
// 7 us, with one wave a row 49).
constexpr int kMergeWaves = 16, kMergeSplits = 8;

template <bool BF, int HD>
__global__ void __launch_bounds__(64 * kMergeWaves) attn_kv8_merge_kernel(Kv8AttnArgs a, int rt) {
  using E = E16<BF>;
  constexpr int V = HD / 64;
  typedef float vec_t __attribute__((ext_vector_type(V)));
  extern __shared__ __attribute__((aligned(16))) float merge_lds[];  // [waves][HD], then (maximum, sum) of each
  const int rep = a.H / a.Hkv, R = a.S * rep, nw = blockDim.x >> 6;
  float2* const mls = reinterpret_cast<float2*>(merge_lds + nw * HD);
  const int64_t rows = (int64_t)a.B * a.Hkv * R, i = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = (int)(i % R), kvh = (int)(i / R % a.Hkv), d = V * lane, t = r / rep;
  const int64_t bb = i / R / a.Hkv;
  const int64_t* const posp = a.pos + bb * a.pos_stride;
  const int32_t* const parents = a.parents ? a.parents + bb * a.parents_stride : nullptr;
  const int64_t head = kvh * rep + r - t * rep, tok = bb * a.S + t;
  uint16_t* const out = static_cast<uint16_t*>(a.out) + tok * a.out_stride + head * HD + d;
  const uint16_t* const gate = static_cast<const uint16_t*>(a.qg) + tok * a.qg_stride + head * 2 * HD + HD + d;
  if (row_invalid(posp, a.L, a.S, parents)) {
    if (wave == 0)
      for (int j = 0; j < V; ++j) out[j] = E::mk(__builtin_nanf(""));
    return;
  }
  const int nblk = kv8_blocks(posp[0], min(r / rt * rt + rt - 1, R - 1) / rep), per = kv8_per_split(nblk, a.nsplit, rt);
  const int nz = (nblk + per - 1) / per;
  const float2* const ml = reinterpret_cast<const float2*>(a.part + rows * a.nsplit * HD) + i * a.nsplit;
  const float* const po = a.part + i * a.nsplit * HD + d;
  float m = -FLT_MAX, l = 0.f;
  vec_t o = 0.f;
  for (int z0 = wave * kMergeSplits; z0 < nz; z0 += nw * kMergeSplits) {
    vec_t x[kMergeSplits];
    float2 s[kMergeSplits];
#pragma unroll
    for (int u = 0; u < kMergeSplits; ++u) {
      const int z = min(z0 + u, nz - 1);
      x[u] = *reinterpret_cast<const vec_t*>(po + (int64_t)z * HD);
      s[u] = ml[z];
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < kMergeSplits; ++u) mn = fmaxf(mn, s[u].x);
    float w[kMergeSplits];
    const float before = l * exp2_raw(m - mn);
    l = before;
#pragma unroll
    for (int u = 0; u < kMergeSplits; ++u) {
      w[u] = z0 + u < nz ? s[u].y * exp2_raw(s[u].x - mn) : 0.f;
      l += w[u];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    o *= before * inv;
    m = mn;
#pragma unroll
    for (int u = 0; u < kMergeSplits; ++u)
      if (z0 + u < nz) o += x[u] * (w[u] * inv);
  }
  *reinterpret_cast<vec_t*>(merge_lds + wave * HD + d) = o;
  if (lane == 0) mls[wave] = make_float2(m, l);
  __syncthreads();
  if (wave) return;
  float mm = -FLT_MAX;
  for (int w = 0; w < nw; ++w) mm = fmaxf(mm, mls[w].x);
  l = 0.f;
  for (int w = 0; w < nw; ++w) l += mls[w].y * exp2_raw(mls[w].x - mm);
  const float inv = 1.f / l;
  o = 0.f;
  for (int w = 0; w < nw; ++w)
    o += *reinterpret_cast<const vec_t*>(merge_lds + w * HD + d) * (mls[w].y * exp2_raw(mls[w].x - mm) * inv);
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = E::mk(o[j] * sigmoid_raw(E::ld(gate[j])));
}

// ---- launches ------------------------------------------------------------------------------------

template <bool BF>
static hipError_t launch_kv8_write_t(const Kv8WriteArgs& a, hipStream_t s) {
  // few tokens: the heads of one are shared out over several workgroups (24 + 2 x 4 heads of 256, shared or not: one token
  // 3.8 / 7.6 us, 512 tokens 8.1 / 9.5, 768 11.0 / 10.6, 1024 13.9 / 12.1, 2047 24.7 / 20.6)
  const int64_t tokens = (int64_t)a.B * a.S;
  const int rows = a.H + 2 * a.Hkv, most = (rows + 4 * kWriteRows - 1) / (4 * kWriteRows);
  if (a.S >= 1 << 24) return hipErrorInvalidValue;  // a launch counts its threads along x in 32 bits
  const dim3 grid((unsigned)a.S, (unsigned)a.B, (unsigned)(tokens >= 1024 ? 1 : most));
  auto launch = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    // a lane's values in one load: every head row starts at a multiple of them
    const bool wide = ((reinterpret_cast<uintptr_t>(a.qg) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) % (HD / 32) |
                       (uintptr_t)((a.qg_stride | a.k_stride | a.v_stride) % (HD / 64))) == 0;
    hipLaunchKernelGGL((kv8_write_kernel<BF, HD>), grid, dim3(256), 0, s, a, wide);
    return hipGetLastError();
  };
  if (a.hd == 256) return launch(std::integral_constant<int, 256>{});
  if (a.hd == 128) return launch(std::integral_constant<int, 128>{});
  if (a.hd == 64) return launch(std::integral_constant<int, 64>{});
  return hipErrorInvalidValue;
}

hipError_t launch_kv8_write(bool bf16, const Kv8WriteArgs& a, hipStream_t s) {
  return bf16 ? launch_kv8_write_t<true>(a, s) : launch_kv8_write_t<false>(a, s);
}

hipError_t launch_kv8_read(int dt, const Kv8ReadArgs& a, hipStream_t s) {
  const int64_t threads = 2ll * a.heads * a.n * (a.hd >> 4), blocks = (threads + 255) / 256;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
  if (dt == 0) hipLaunchKernelGGL(kv8_read_kernel<0>, grid, dim3(256), 0, s, a);
  else if (dt == 1) hipLaunchKernelGGL(kv8_read_kernel<1>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(kv8_read_kernel<2>, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

// Workgroups of rt rows, and the merge of their splits; `launch` starts the kernel over a grid.
template <bool BF, int HD, typename F>
static hipError_t launch_attn_kv8_t(const Kv8AttnArgs& a, hipStream_t s, int rt, F launch) {
  const int64_t rows = (int64_t)a.S * (a.H / a.Hkv), all = rows * a.Hkv * a.B;
  const int64_t wgs = (rows + rt - 1) / rt * a.Hkv * a.nsplit;
  const int waves = std::min((a.nsplit + kMergeSplits - 1) / kMergeSplits, kMergeWaves);
  // a launch counts its threads along x in 32 bits
  if (wgs >= (1ll << 24) || (a.nsplit > 1 && all >= (1ll << 26) / waves)) return hipErrorInvalidValue;
  const hipError_t e = launch(dim3((unsigned)wgs, (unsigned)a.B));
  if (e != hipSuccess) return e;
  if (a.nsplit > 1) {
    hipLaunchKernelGGL((attn_kv8_merge_kernel<BF, HD>), dim3((unsigned)all), dim3(64 * waves), waves * (HD * 4 + 8), s, a, rt);
  }
  return hipGetLastError();
}

template <bool BF, int HD>
static hipError_t launch_attn_kv8_rows(const Kv8AttnArgs& a, hipStream_t s) {
  constexpr int q = 16 * HD * 2 + 2 * 16 * 4 + 4 * 64 * 4 + 4 * 16 * 4, merge = 4 * 16 * (HD + 4) * 4 + 4 * 16 * 8;
  constexpr int lds = q > merge ? q : merge;
  return launch_attn_kv8_t<BF, HD>(a, s, 16, [&](dim3 grid) {
    static LdsLimit limit;
    const hipError_t e = limit.raise((const void*)attn_kv8_rows_kernel<BF, HD>, lds);
    if (e == hipSuccess) hipLaunchKernelGGL((attn_kv8_rows_kernel<BF, HD>), grid, dim3(256), lds, s, a);
    return e;
  });
}

template <bool BF, int HD, int NT>
static hipError_t launch_attn_kv8_tile(const Kv8AttnArgs& a, hipStream_t s) {
  constexpr int q = 64 * NT * (HD * 2 + 8), tiles = 2 * (2 * 64 * HD + 512) + 4096 * NT * kv8_lds_steps(HD) + 2560 + (1024 + 256) * NT;
  constexpr int lds = q > tiles ? q : tiles;
  return launch_attn_kv8_t<BF, HD>(a, s, 64 * NT, [&](dim3 grid) {
    static LdsLimit limit;
    const hipError_t e = limit.raise((const void*)attn_kv8_tile_kernel<BF, HD, NT>, lds);
    if (e == hipSuccess) hipLaunchKernelGGL((attn_kv8_tile_kernel<BF, HD, NT>), grid, dim3(256), lds, s, a);
    return e;
  });
}

// Rows of a workgroup. attn_kv8_rows_kernel (16) has the shorter chain, attn_kv8_tile_kernel reads the cache once
// for 128 rows. The tiles are for kTileBlocks tiles of 16 rows by 32 positions and more, where the two meet: by rows
// and by tiles, in us, in caches as long as their content,
//                                      at half of it   at it         twice         four times
//   24 heads of 256   13 drafted         57 /  64      102 /  89     199 / 149     399 / 250
//   (4 KV heads)      64 drafted         48 /  66       79 /  82     139 / 114     261 / 180
//                     400 tokens         54 /  66       97 /  82     182 / 115     342 / 184
//   32 heads of 128   13 drafted         32 /  44       51 /  61      88 /  98     183 / 173
//   (8)               64 drafted         33 /  44       50 /  52      84 /  73     151 / 112
//                     400 tokens         33 /  48       54 /  59      97 /  81     184 / 127
//   64 heads of 64    13 drafted         25 /  34       38 /  38      62 /  55     111 /  87
//   (8)               64 drafted         26 /  33       38 /  40      62 /  55     110 /  79
//                     400 tokens         22 /  44       32 /  53      52 /  71      91 / 106
// in fp16; in bf16 both are up to 8 per cent slower and meet at the same places. Prompts of 333, 1100 and 1600 without a
// cache: 16 / 44, 68 / 83, 112 / 127 at head dim 256; 13 / 27, 45 / 55, 78 / 78 at 128; 14 / 20, 49 / 44, 87 / 73 at 64.
// What the host knows is the capacity (max_len), not the positions in use: in a cache with room left fewer
// tokens take the tiles (333 behind none in 4096 positions: 51 us).
// Head dim 64 takes 256 rows instead of 128 where that makes two workgroups a CU (4096 tokens of 2 x 32 heads: over 4 KV
// heads 302 against 325 us, over 32 336 against 340); at 128 the registers do not hold them (with sums over u, 521 against 481).
constexpr int64_t kTileBlocks = 49152;

int attn_kv8_plan(int64_t batch, int64_t seq, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_len) {
  const int64_t rows = seq * (heads / kv_heads), groups = batch * kv_heads;
  // a row sees all but half of the new tokens on average
  if (rows <= 32 || (rows + 15) / 16 * groups * ((max_len - seq / 2 + 31) / 32) < kTileBlocks) return 16;
  return head_dim == 64 && (rows + 255) / 256 * groups >= 512 ? 256 : 128;
}

// Splits that give each of `cus` CUs two workgroups, of at least 256 positions each: below that a split's
// share of the merge costs more than it saves.
int64_t attn_kv8_splits(int64_t batch, int64_t seq, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_len,
                        int cus) {
  const int rt = attn_kv8_plan(batch, seq, heads, kv_heads, head_dim, max_len);
  const int64_t wgs = (seq * (heads / kv_heads) + rt - 1) / rt * kv_heads * batch;
  return std::max<int64_t>(1, std::min<int64_t>({2 * cus / std::max<int64_t>(wgs, 1), max_len / 256, 65535}));
}

hipError_t launch_attn_kv8(bool bf16, const Kv8AttnArgs& a, hipStream_t s) {
  const int rt = attn_kv8_plan(a.B, a.S, a.H, a.Hkv, a.hd, a.L);
  auto tiles = [&](auto bf, auto hd) -> hipError_t {
    constexpr bool BF = decltype(bf)::value;
    constexpr int HD = decltype(hd)::value;
    if (rt == 16) return launch_attn_kv8_rows<BF, HD>(a, s);
    if constexpr (HD == 64) {
      if (rt == 256) return launch_attn_kv8_tile<BF, HD, 4>(a, s);
    }
    return launch_attn_kv8_tile<BF, HD, 2>(a, s);
  };
  auto dims = [&](auto bf) -> hipError_t {
    if (a.hd == 256) return tiles(bf, std::integral_constant<int, 256>{});
    if (a.hd == 128) return tiles(bf, std::integral_constant<int, 128>{});
    if (a.hd == 64) return tiles(bf, std::integral_constant<int, 64>{});
    return hipErrorInvalidValue;
  };
  return bf16 ? dims(std::true_type{}) : dims(std::false_type{});
}

}  // namespace gsq
