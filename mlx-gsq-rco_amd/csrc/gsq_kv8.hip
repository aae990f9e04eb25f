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

#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "gsq_common.h"

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
// in double. k and v rows are handled in double: rounding to 8 bits jumps at values next to a border,
// and so the bytes are those of the definition. Bound by memory latency (each row read and written
// once).
constexpr int kWriteRows = 4;

template <bool BF, int HD>
__global__ void __launch_bounds__(256) kv8_write_kernel(Kv8WriteArgs a) {
  using E = E16<BF>;
  constexpr int V = HD / 64;  // consecutive values per lane
  typedef uint16_t vec_t __attribute__((ext_vector_type(V)));
  typedef uint8_t bytes_t __attribute__((ext_vector_type(V)));
  __shared__ double row[4][HD], cs[HD / 2], sn[HD / 2];
  __shared__ int depth;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, d0 = V * lane;
  const int t = blockIdx.x, bb = blockIdx.y, hr = a.rd / 2, nh = a.H + 2 * a.Hkv, step = 4 * gridDim.z;
  const int64_t* const pos = a.pos + (int64_t)bb * a.pos_stride;
  const int32_t* const parents = a.parents ? a.parents + (int64_t)bb * a.parents_stride : nullptr;
  const int64_t r = (int64_t)bb * a.S + t;
  uint16_t* const qo = static_cast<uint16_t*>(a.q) + r * a.H * HD + d0;
  const bool invalid = row_invalid(pos, a.L, a.S, parents);
  if (invalid) {
    for (int h = blockIdx.z * 4 + wave; h < a.H; h += step)
      for (int j = 0; j < V; ++j) qo[(int64_t)h * HD + j] = E::mk(__builtin_nanf(""));
    return;
  }
  const uint16_t* const qg = static_cast<const uint16_t*>(a.qg) + r * a.qg_stride + d0;
  const uint16_t* const kn = static_cast<const uint16_t*>(a.k) + r * a.k_stride + d0;
  const uint16_t* const vn = static_cast<const uint16_t*>(a.v) + r * a.v_stride + d0;
  uint16_t x[kWriteRows][V];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < kWriteRows; ++u) {
      const int h = min(h0 + u * step, nh - 1);
      const uint16_t* src = h < a.H ? qg + (int64_t)h * 2 * HD
                                    : (h < a.H + a.Hkv ? kn + (int64_t)(h - a.H) * HD : vn + (int64_t)(h - a.H - a.Hkv) * HD);
#pragma unroll
      for (int j = 0; j < V; ++j) x[u][j] = src[j];
    }
  };
  int h0 = blockIdx.z * 4 + wave;
  load(h0);
  if (parents) {  // rotary position: the token's depth in the tree behind the cache
    if (wave == 0) {
      const uint64_t path = tree_path(parents, a.S);
      if (lane == t) depth = __popcll(path) - 1;
    }
    __syncthreads();
  }
  const int64_t rp = pos[0] + (parents ? depth : t), slot = pos[0] + t;
  if (tid < hr) {
    const double ang = (double)rp * a.inv_freq[tid];
    cs[tid] = cos(ang);
    sn[tid] = sin(ang);
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
  auto norm_rope = [&](auto zero, const uint16_t (&in)[V], const float (&w)[V], auto (&f)[V]) {
    using T = decltype(zero);
    T* const rw = reinterpret_cast<T*>(row[wave]);
    T ss = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f[j] = E::ld(in[j]);
      ss += f[j] * f[j];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    const T rn = (T)1 / sqrt(ss / (T)HD + (T)a.eps);
#pragma unroll
    for (int j = 0; j < V; ++j) rw[d0 + j] = f[j] = f[j] * rn * (T)w[j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int d = d0 + j;
      if (d < a.rd) {
        const int i = d < hr ? d : d - hr;
        const T other = d < hr ? -rw[d + hr] : rw[i];
        f[j] = f[j] * (T)cs[i] + other * (T)sn[i];
      }
    }
    __builtin_amdgcn_wave_barrier();
  };
  for (; h0 < nh; h0 += step * kWriteRows) {
    uint16_t cur[kWriteRows][V];
#pragma unroll
    for (int u = 0; u < kWriteRows; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) cur[u][j] = x[u][j];
    if (h0 + step * kWriteRows < nh) load(h0 + step * kWriteRows);
#pragma unroll
    for (int u = 0; u < kWriteRows; ++u) {
      const int h = h0 + u * step;
      if (h >= nh) break;
      if (h < a.H) {
        float f[V];
        norm_rope(0.f, cur[u], wq, f);
        vec_t o;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = E::mk(f[j]);
        *reinterpret_cast<vec_t*>(qo + (int64_t)h * HD) = o;
        continue;
      }
      const bool isk = h < a.H + a.Hkv;
      double f[V], mx = 0;
      if (isk) {
        norm_rope(0.0, cur[u], wk, f);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = E::ld(cur[u][j]);
      }
      bool bad = false;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        bad |= !(fabs(f[j]) <= DBL_MAX);
        mx = fmax(mx, fabs(f[j]));
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor(mx, o, 64));
      float s = (float)(mx / 127.0);
      if (__any(bad) || !(s <= FLT_MAX)) s = __builtin_nanf("");
      bytes_t o;
#pragma unroll
      for (int j = 0; j < V; ++j)
        o[j] = (uint8_t)(s > 0.f ? 128 + (int)fmin(fmax(rint(f[j] / (double)s), -127.0), 127.0) : 128);
      const int64_t at = ((int64_t)bb * a.Hkv + (isk ? h - a.H : h - a.H - a.Hkv)) * a.L + slot;
      *reinterpret_cast<bytes_t*>((isk ? a.kc : a.vc) + at * HD + d0) = o;
      if (lane == 0) (isk ? a.ks : a.vs)[at] = s;
    }
  }
}

// ---- reading back --------------------------------------------------------------------------------
// out[b, h, j, :] = round((u - 128) s), the product in float32, of rows start .. start + n - 1 of both caches: a thread per 16
// values, K's rows first. Bound by memory: hd + 4 bytes read and hd values written per row.
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
// token t. A workgroup takes 16 NT rows of one (batch row, KV head) and a run of 32-position blocks;
// its four waves take the blocks in turn, each with a softmax of its own, and are merged at the end.
//
//  * Products on fp16 MFMAs, transposed: S^T = K Q^T puts a row (query) on each lane column, lane % 16,
//    and positions 16 b + 4 (lane / 16) + e of the block on its registers, which is the layout of the B
//    operand of O^T = V^T P^T: probabilities never leave their lane.
//  * Bytes are exact in fp16, so K and V cost no rounding; the scale of a K row multiplies its scores, that
//    of a V row its probabilities. bf16 queries are scaled to fp16 by a power of two for each row:
//    their 8 bits fit, and what falls below 2^-38 of the row's largest cannot be seen in float32 sums.
//  * K and V go from memory to registers in 16-byte pieces and are expanded there: no LDS, no barrier
//    in the loop. For K the dims of a product's step are those a lane's piece holds (any order of dims
//    gives the same sum); for V a lane holds hd / 16 neighbouring dims of 8 positions, and dim d of a
//    lane's run belongs to output tile d.
//  * The reference of the exponent moves only when a score passes it by 2^kLazy, for all rows of the
//    wave at once: mostly no rescaling and no exchange between lanes in the loop.
//  * A weight (probability times V scale, 2^kPScale over the largest V scale met) is at most 2^(2 kLazy +
//    kPScale) = 2^15 and held in fp16: for bf16 outputs in one value (11 bits, eight times finer than the
//    output's own rounding), for fp16 outputs in two (22 bits, down to 2^-25 of the unit), as one would
//    add an error as large as the output's rounding.
constexpr int kLazy = 3;
constexpr float kPScale = 9.f;

// bytes of a dword pair as fp16 (u - 128): v_perm puts 0x64 above a byte, which is 1024 + u in fp16
__device__ __forceinline__ uint32_t bytes_f16(uint32_t hi, uint32_t lo, uint32_t sel) {
  const uint32_t w = __builtin_amdgcn_perm(hi, lo, sel) | 0x64006400u;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w) + (f16x2){(_Float16)-1152.f, (_Float16)-1152.f});
}

__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// blocks of 32 positions that rows up to token t see, and those of a split
__device__ __forceinline__ int kv8_blocks(int64_t pos, int t) { return (int)((pos + t) / 32) + 1; }

template <bool BF, int HD, int NT>
__global__ void __launch_bounds__(256, NT == 1 ? 2 : 1) attn_kv8_kernel(Kv8AttnArgs a) {
  using E = E16<BF>;
  constexpr int KS = HD / 32, KL = HD / 64, VB = HD / 16, RT = 16 * NT;  // VB: dims (bytes) of a lane, output tiles
  constexpr bool QREG = NT <= 2;
  constexpr int TERMS = BF ? 1 : 2;  // fp16 values that hold a weight
  constexpr int VW = VB / 4;  // dwords of a lane's V piece
  typedef uint32_t vpiece __attribute__((ext_vector_type(VW)));
  extern __shared__ __attribute__((aligned(16))) uint8_t kv8_lds[];
  // queries in operand order (16 bytes per lane, step and tile), row factors, scales of a wave's block;
  // the merge of the waves takes the same memory afterwards
  u32x4* const qs = reinterpret_cast<u32x4*>(kv8_lds);
  float* const rowc_s = reinterpret_cast<float*>(kv8_lds + RT * HD * 2);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  float* const sc = rowc_s + RT + wave * 64;
  const int g = lane >> 4, c = lane & 15;
  const int rep = a.H / a.Hkv, R = a.S * rep, ntile = (R + RT - 1) / RT;
  const int kvh = blockIdx.x % a.Hkv, rest = blockIdx.x / a.Hkv, z = rest % a.nsplit, tile = ntile - 1 - rest / a.nsplit;
  const int bb = blockIdx.y, r0 = tile * RT;
  const int64_t* const posp = a.pos + (int64_t)bb * a.pos_stride;
  const int32_t* const parents = a.parents ? a.parents + (int64_t)bb * a.parents_stride : nullptr;
  // rows r0 .. of this KV head in q, qg and out
  auto row_at = [&](int r, int64_t stride, int width) {
    const int t = r / rep;
    return ((int64_t)bb * a.S + t) * stride + (int64_t)(kvh * rep + r - t * rep) * width;
  };
  if (row_invalid(posp, a.L, a.S, parents)) {
    if (a.nsplit == 1)
      for (int i = tid; i < RT * HD; i += 256)
        if (r0 + i / HD < R)
          static_cast<uint16_t*>(a.out)[row_at(r0 + i / HD, a.out_stride, HD) + i % HD] = E::mk(__builtin_nanf(""));
    return;
  }
  const int64_t pos = posp[0];
  const int tfirst = r0 / rep, tlast = min(r0 + RT - 1, R - 1) / rep;
  const int nblk = kv8_blocks(pos, tlast), per = (nblk + a.nsplit - 1) / a.nsplit;
  const int blk0 = z * per, blk1 = min(nblk, blk0 + per);
  if (blk0 >= blk1) return;  // the merge knows
  const int64_t base = ((int64_t)bb * a.Hkv + kvh) * a.L;
  const int64_t klast = pos + tlast;  // last position any row sees

  u32x4 kr[2][KL];
  vpiece vr[8];
  auto load_k = [&](int blk) {  // positions past the last repeat it
    const int64_t j0 = (int64_t)blk * 32;
    const int left = (int)min(klast - j0, (int64_t)31);
    const uint8_t* p = a.kc + (base + j0) * HD + 16 * g;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int s = 0; s < KL; ++s)
        kr[b][s] = *reinterpret_cast<const u32x4*>(p + min(16 * b + c, left) * HD + 64 * s);
  };
  auto load_v = [&](int blk) {
    const int64_t j0 = (int64_t)blk * 32;
    const int left = (int)min(klast - j0, (int64_t)31);
    const uint8_t* p = a.vc + (base + j0) * HD + VB * c;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      vr[i] = *reinterpret_cast<const vpiece*>(p + min(16 * (i >> 2) + 4 * g + (i & 3), left) * HD);
  };
  float scv = 0.f;  // lane l < 32: K scale of position l of the block; else V scale of l - 32
  auto load_s = [&](int blk) {
    const int64_t j0 = (int64_t)blk * 32;
    const int left = (int)min(klast - j0, (int64_t)31);
    scv = (lane < 32 ? a.ks : a.vs)[base + j0 + min(lane & 31, left)];
  };
  int blk = blk0 + wave;
  if (blk < blk1) {
    load_k(blk);
    load_v(blk);
    load_s(blk);
  }
  // queries to LDS in operand order: HD / 8 threads a row, 8 values each
  {
    constexpr int TR = HD / 8;  // threads a row: 8, 16 or 32
#pragma unroll 1
    for (int i = tid; i < RT * TR; i += 256) {
      const int r = i / TR, o = i % TR;  // octet o: dims 8 o .. + 7
      u32x4 w = {0, 0, 0, 0};
      if (r0 + r < R)
        w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + row_at(r0 + r, a.q_stride, HD) + 8 * o);
      float cr = 1.f;
      if constexpr (BF) {
        float v[8], mx = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = E::ld((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
          mx = fmaxf(mx, fabsf(v[e]));
        }
#pragma unroll
        for (int x = 1; x < TR; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
        int ex = 0;
        if (mx > 0.f && mx <= FLT_MAX) ex = 14 - ilogbf(mx);
        cr = ldexpf(1.f, -ex);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = pack_h2(ldexpf(v[2 * e], ex), ldexpf(v[2 * e + 1], ex));
      }
      // dims 64 s + 16 g + 8 h: step 2 s + h of lane group g
      const int s = o >> 3, gg = (o >> 1) & 3, ks = 2 * s + (o & 1);
      qs[((r >> 4) * KS + ks) * 64 + 16 * gg + (r & 15)] = w;
      if (o == 0) rowc_s[r] = cr;
    }
  }
  __syncthreads();
  u32x4 qf[QREG ? NT : 1][QREG ? KS : 1];
  if constexpr (QREG) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[n][s] = qs[(n * KS + s) * 64 + lane];
  }
  float rowc[NT], m[NT], l[NT];
  int tok[NT];
  uint64_t path[NT];
  const uint64_t paths = parents ? tree_path(parents, a.S) : 0;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    rowc[n] = rowc_s[16 * n + c];
    m[n] = -FLT_MAX;
    l[n] = 0.f;
    tok[n] = min(r0 + 16 * n + c, R - 1) / rep;
    path[n] = __shfl((uint32_t)paths, tok[n], 64) | ((uint64_t)__shfl((uint32_t)(paths >> 32), tok[n], 64) << 32);
  }
  f32x4 acc[NT][VB];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < VB; ++i) acc[n][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float vref = 0x1p-100f;  // largest V scale met (the probabilities' unit)
  const float c_ = 1.44269504088896340736f / sqrtf((float)HD);

  for (; blk < blk1; blk += 4) {
    const bool more = blk + 4 < blk1;
    // scales of the block's positions to the lanes that hold them
    sc[lane] = lane < 32 ? scv * c_ : scv;
    __builtin_amdgcn_wave_barrier();
    f32x4 ks4[2], vs4[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      ks4[b] = *reinterpret_cast<const f32x4*>(sc + 16 * b + 4 * g);
      vs4[b] = *reinterpret_cast<const f32x4*>(sc + 32 + 16 * b + 4 * g);
    }
    __builtin_amdgcn_wave_barrier();
    if (more) load_s(blk + 4);
    f32x4 s[NT][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        const uint32_t w0 = kr[b][st >> 1][2 * (st & 1)], w1 = kr[b][st >> 1][2 * (st & 1) + 1];
        const u32x4 kf = {bytes_f16(0, w0, 0x0C010C00), bytes_f16(0, w0, 0x0C030C02), bytes_f16(0, w1, 0x0C010C00),
                          bytes_f16(0, w1, 0x0C030C02)};
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][b] = mma16(kf, QREG ? qf[QREG ? n : 0][QREG ? st : 0] : qs[(n * KS + st) * 64 + lane], s[n][b]);
      }
    }
    if (more) load_k(blk + 4);
    // positions behind a row's token, or off its path
    const int64_t j0 = (int64_t)blk * 32;
    if (parents ? j0 + 31 >= pos : j0 + 31 > pos + tfirst) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t node = j0 + 16 * b + 4 * g + e - pos;  // negative: a cached position
            const bool see = parents ? node < 0 || (node < 64 && ((path[n] >> (node & 63)) & 1)) : node <= tok[n];
            s[n][b][e] = see ? s[n][b][e] * ks4[b][e] * (BF ? rowc[n] : 1.f) : -INFINITY;
          }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][b][e] = s[n][b][e] * ks4[b][e] * (BF ? rowc[n] : 1.f);
    }
    float vmax = 0.f;
    bool move = false;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) vmax = fmaxf(vmax, vs4[b][e]);
    move |= vmax > vref * (float)(1 << kLazy);
    float mx[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mx[n] = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[n] = fmaxf(mx[n], s[n][b][e]);
      move |= mx[n] > m[n] + (float)kLazy;
    }
    if (__any(move)) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) vmax = fmaxf(vmax, __shfl_xor(vmax, o, 64));
      const float vnew = fmaxf(vref, vmax), vr_ = vref / vnew;
      vref = vnew;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x = fmaxf(mx[n], __shfl_xor(mx[n], 16, 64));
        x = fmaxf(x, __shfl_xor(x, 32, 64));
        const float mn = fmaxf(m[n], x), alpha = exp2_raw(m[n] - mn);
        m[n] = mn;
        l[n] *= alpha;
#pragma unroll
        for (int i = 0; i < VB; ++i) acc[n][i] *= alpha * vr_;
      }
    }
    // weights of V: probability x scale / vref, 0 for what a row does not see whatever the scale is
    const float vinv = 1.f / vref;
#pragma unroll
    for (int b = 0; b < 2; ++b) vs4[b] *= vinv * exp2_raw(kPScale);
    u32x4 pf[TERMS][NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = exp2_raw(s[n][b][e] - m[n]);
          l[n] += p;
          w[e] = s[n][b][e] == -INFINITY ? 0.f : p * vs4[b][e];
        }
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const f16x2 hi = __builtin_convertvector((f32x2){w[e], w[e + 1]}, f16x2);
            pf[t][n][2 * b + e / 2] = __builtin_bit_cast(uint32_t, hi);
            w[e] -= (float)hi.x;  // what the term leaves, for the next one
            w[e + 1] -= (float)hi.y;
          }
      }
#pragma unroll
    for (int i = 0; i < VB; ++i) {
      // dim VB c + i of the 8 positions: byte i & 3 of dword i / 4 of each row
      const uint32_t sel = 0x0C000C00u | (uint32_t)((4 + (i & 3)) << 16) | (uint32_t)(i & 3);
      const u32x4 vf = {bytes_f16(vr[1][i >> 2], vr[0][i >> 2], sel), bytes_f16(vr[3][i >> 2], vr[2][i >> 2], sel),
                        bytes_f16(vr[5][i >> 2], vr[4][i >> 2], sel), bytes_f16(vr[7][i >> 2], vr[6][i >> 2], sel)};
#pragma unroll
      for (int t = 0; t < TERMS; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][i] = mma16(vf, pf[t][n], acc[n][i]);
    }
    if (more) load_v(blk + 4);
  }
  // merge of the waves, 16 rows at a time: every wave's maximum, sum and outputs (in V's own unit)
  constexpr int OS = HD + 4;
  float* const mo = reinterpret_cast<float*>(kv8_lds);             // [4][16][OS]
  float2* const ml = reinterpret_cast<float2*>(mo + 4 * 16 * OS);  // [4][16]
  const float unit = vref * exp2_raw(-kPScale);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    __syncthreads();  // queries, or the tile before, are no longer read
    float* const mine = mo + (wave * 16 + c) * OS;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < VB; i += 4)
        *reinterpret_cast<f32x4*>(mine + VB * (4 * g + e) + i) =
            (f32x4){acc[n][i][e], acc[n][i + 1][e], acc[n][i + 2][e], acc[n][i + 3][e]} * unit;
    float ls = l[n] + __shfl_xor(l[n], 16, 64);
    ls += __shfl_xor(ls, 32, 64);
    if (g == 0) ml[wave * 16 + c] = make_float2(m[n], ls);
    __syncthreads();
    for (int i = tid; i < 16 * HD / 4; i += 256) {
      const int rr = i / (HD / 4), d = 4 * (i % (HD / 4)), r = r0 + 16 * n + rr;
      if (r >= R) continue;
      float mm = -FLT_MAX, ll = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[w * 16 + rr].x);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 x = ml[w * 16 + rr];
        const float f = exp2_raw(x.x - mm);
        ll += x.y * f;
        o += *reinterpret_cast<const f32x4*>(mo + (w * 16 + rr) * OS + d) * f;
      }
      if (a.nsplit > 1) {
        const int64_t rows = (int64_t)a.B * a.Hkv * R, at = (((int64_t)bb * a.Hkv + kvh) * R + r) * a.nsplit + z;
        *reinterpret_cast<f32x4*>(a.part + at * HD + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(a.part + rows * a.nsplit * HD + 2 * at) = make_float2(mm, ll);
      } else {
        const uint16_t* gate = static_cast<const uint16_t*>(a.qg) + row_at(r, a.qg_stride, 2 * HD) + HD + d;
        const uint2 gw = *reinterpret_cast<const uint2*>(gate);
        const uint16_t gv[4] = {(uint16_t)gw.x, (uint16_t)(gw.x >> 16), (uint16_t)gw.y, (uint16_t)(gw.y >> 16)};
        const float inv = 1.f / ll;
        uint32_t q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = E::mk(o[e] * inv * (1.f / (1.f + expf(-E::ld(gv[e])))));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row_at(r, a.out_stride, HD) + d) =
            make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
      }
    }
  }
}

// Outputs of split positions: a wave per row weighs the splits that hold positions of the row's tile by
// their maxima, normalizes and gates. Bound by reading the partial outputs once.
template <bool BF, int HD>
__global__ void __launch_bounds__(256) attn_kv8_merge_kernel(Kv8AttnArgs a, int rt) {
  using E = E16<BF>;
  constexpr int V = HD / 64;
  typedef float vec_t __attribute__((ext_vector_type(V)));
  const int rep = a.H / a.Hkv, R = a.S * rep;
  const int64_t rows = (int64_t)a.B * a.Hkv * R, i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= rows) return;
  const int r = (int)(i % R), kvh = (int)(i / R % a.Hkv), d = V * (threadIdx.x & 63), t = r / rep;
  const int64_t bb = i / R / a.Hkv;
  const int64_t* const posp = a.pos + bb * a.pos_stride;
  const int32_t* const parents = a.parents ? a.parents + bb * a.parents_stride : nullptr;
  const int64_t head = kvh * rep + r - t * rep, tok = bb * a.S + t;
  uint16_t* const out = static_cast<uint16_t*>(a.out) + tok * a.out_stride + head * HD + d;
  const uint16_t* const gate = static_cast<const uint16_t*>(a.qg) + tok * a.qg_stride + head * 2 * HD + HD + d;
  if (row_invalid(posp, a.L, a.S, parents)) {
    for (int j = 0; j < V; ++j) out[j] = E::mk(__builtin_nanf(""));
    return;
  }
  const int nblk = kv8_blocks(posp[0], min(r / rt * rt + rt - 1, R - 1) / rep), per = (nblk + a.nsplit - 1) / a.nsplit;
  const int nz = (nblk + per - 1) / per;
  const float2* const ml = reinterpret_cast<const float2*>(a.part + rows * a.nsplit * HD) + i * a.nsplit;
  const float* const po = a.part + i * a.nsplit * HD + d;
  float m = -FLT_MAX, l = 0.f;
  vec_t o = 0.f;
  for (int z = 0; z < nz; ++z) m = fmaxf(m, ml[z].x);
  for (int z = 0; z < nz; ++z) {
    const float w = exp2_raw(ml[z].x - m);
    l += ml[z].y * w;
    o += *reinterpret_cast<const vec_t*>(po + (int64_t)z * HD) * w;
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = E::mk(o[j] * inv * (1.f / (1.f + expf(-E::ld(gate[j])))));
}

// ---- launches ------------------------------------------------------------------------------------

template <bool BF>
static hipError_t launch_kv8_write_t(const Kv8WriteArgs& a, hipStream_t s) {
  // few tokens: the heads of one are shared out over several workgroups
  const int64_t tokens = (int64_t)a.B * a.S;
  const int rows = a.H + 2 * a.Hkv, most = (rows + 4 * kWriteRows - 1) / (4 * kWriteRows);
  const dim3 grid((unsigned)a.S, (unsigned)a.B, (unsigned)(tokens >= 1024 ? 1 : most));
  auto launch = [&](auto hd) {
    hipLaunchKernelGGL((kv8_write_kernel<BF, decltype(hd)::value>), grid, dim3(256), 0, s, a);
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

template <bool BF, int HD, int NT>
static hipError_t launch_attn_kv8_t(const Kv8AttnArgs& a, hipStream_t s) {
  constexpr int RT = 16 * NT;
  constexpr int lds_q = RT * HD * 2 + RT * 4 + 4 * 64 * 4, lds_m = 4 * 16 * (HD + 4) * 4 + 4 * 16 * 8;
  constexpr int lds = lds_q > lds_m ? lds_q : lds_m;
  const int64_t rows = (int64_t)a.S * (a.H / a.Hkv), all = rows * a.Hkv * a.B;
  const int64_t wgs = (rows + RT - 1) / RT * a.Hkv * a.nsplit;
  if (wgs >= (1ll << 31) || (a.nsplit > 1 && (all + 3) / 4 >= (1ll << 31))) return hipErrorInvalidValue;
  static LdsLimit limit;
  const hipError_t e = limit.raise((const void*)attn_kv8_kernel<BF, HD, NT>, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((attn_kv8_kernel<BF, HD, NT>), dim3((unsigned)wgs, (unsigned)a.B), dim3(256), lds, s, a);
  if (a.nsplit > 1)
    hipLaunchKernelGGL((attn_kv8_merge_kernel<BF, HD>), dim3((unsigned)((all + 3) / 4)), dim3(256), 0, s, a, RT);
  return hipGetLastError();
}

hipError_t launch_attn_kv8(bool bf16, const Kv8AttnArgs& a, hipStream_t s) {
  auto tiles = [&](auto bf, auto hd) -> hipError_t {
    return launch_attn_kv8_t<decltype(bf)::value, decltype(hd)::value, 1>(a, s);
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
