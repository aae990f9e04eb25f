// Attention of packed sequences over a paged K/V cache: single tokens, chunks of prompts and whole prompts in one call
// (the reference runs mlx-lm's attention over one sequence, mlx_gsq/models/qwen35.py:114-152).
//
// The rows of a (sequence, KV head) are its rep = heads / kv_heads query heads of every new token, row t rep + r for
// head r of token t. Two kinds of workgroups share the arithmetic and a launch: paged_rows for few rows, whose waves share a
// tile of 16 rows and take its positions in turn, paged_tile for many, whose waves share tiles of K and V in LDS.
// Both products run on the 16-bit matrix cores, transposed: S^T = K Q^T puts a row on each lane column, lane % 16, and
// positions 16 b + 4 (lane / 16) + e of a block of 32 on its registers, which is the layout of the B operand of
// O^T = V^T P^T: weights never leave their lane.
//
// What a workgroup does follows from the lengths on the device (PagedTask): no host knows them, and a captured call
// follows them. Positions are split over workgroups so that the step's work fills the device, in pieces of one length
// for all its sequences; what pieces of one row leave meets in attn_paged_merge_kernel.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "gsq_common.h"
#include "gsq_elem.h"
#include "gsq_seq16.h"

namespace gsq {

// Which sequences a launch serves: all, or those of few or of many rows.
enum { kAll = 0, kFew = 1, kMany = 2 };

struct PagedSched {
  int lrt;        // log2 of the rows of a workgroup
  int which;      // kAll, kFew or kMany
  int target;     // workgroups that fill the device
  int least;      // fewest blocks of 32 positions to a piece
  int64_t parts;    // pieces whose partial outputs `part` holds
  int64_t part_at;  // the first of them, in floats
  __device__ __host__ int rt() const { return 1 << lrt; }
};

namespace {

// Transposing LDS read: 16 lanes read 4 rows of 16 values (lane j: values 4 (j % 4) .. + 3 of row
// j / 4, 8 bytes); lane j gets column j of the four rows.
__device__ __forceinline__ s16x4 tr_read(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// v, as a value that nothing is known about: what is formed from it is formed there, not kept in a register
// through the loop around it
__device__ __forceinline__ int anew(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// 16 bytes a lane from base + off to LDS, 64 times 16 from `dst` on. As assembly: the compiler makes every transposing read
// wait for all DMA that it knows of, the next tile's too. Whoever reads what it brings waits for vmcnt.
__device__ __forceinline__ void dma16(const uint16_t* base, uint32_t off, const uint8_t* dst) {
  const uint32_t lds = uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)dst);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}

constexpr int kRowsTile = 16;   // rows of a workgroup of paged_rows: 2^4
constexpr int kTileRows = 128;  // of paged_tile: 2^7
// Rows up to which a sequence takes the first (us, six heads to a KV head of 256, first and second: 36 rows behind 30000 62
// and 55, 96 rows 91 and 62; 36 rows of 16 sequences behind 3000 74 and 68; one sequence of 36 behind 2000 20 and 30, a
// latency that steps of few tokens and short contexts pay).
constexpr int kFewRows = 32;

// Lane's view of a sequence.
struct SeqLane {
  int n, tiles, blocks;
  __device__ SeqLane(const AttnPagedArgs& a, const PagedSched& p, int b) {
    n = tiles = blocks = 0;
    if (b >= a.B) return;
    const int t0 = min(max(a.cu[b], 0), a.N), t1 = min(max(a.cu[b + 1], t0), a.N);
    const PackedSeq s(a.cu, a.rows, a.lens, b, a.N, a.R, a.W * a.P);
    n = t1 - t0;
    const bool few = n * a.rep <= kFewRows;
    if (p.which != kAll && few != (p.which == kFew)) n = 0;
    tiles = (n * a.rep + p.rt() - 1) >> p.lrt;
    blocks = s.fine ? (s.len + 31) / 32 : 1;  // one that is not served: its rows are NaN, in one piece
  }
  // pieces of `per` blocks (1 / per given), or one more: what counts is that all workgroups get the same
  __device__ int splits(float over) const { return max((int)ceilf((float)blocks * over), 1); }
};

template <typename T>
__device__ __forceinline__ T wave_scan(T v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

// One over the blocks of a piece. Few rows: the step's work (tiles of rows times blocks) over as many workgroups as
// fill the device. Many rows: the longest sequence in 1 .. 64 pieces, whichever ends first when workgroups of one piece each
// fill the device in turn (kPieceCost blocks for what a piece costs besides: its partial outputs, written and merged); of more
// than kSearched sequences, which the search would take too long for, in proportion to the work as few rows; with
// enough tiles of rows none is split. Only sequences of many rows count here: what runs beside them is another kind's (fp16,
// 24 heads of 256 over 4 KV heads, us, in pieces and not: 64 tokens behind 131071 beside 64 single ones 406 and 7650, 1024 behind
// 30000 1100 and 2168; in proportion and not: 17 turns of 64 behind 15000 to 30000 1097 and 1883 (16, searched: 844), 40 of 8
// behind 8000 to 16000 486 and 1046, 20 of 150 to 300 behind 4000 to 8000 1051 and 1042).
constexpr int kPieceCost = 10, kMostTurns = 4, kSearched = 16;

__device__ __forceinline__ float over_chunk(const AttnPagedArgs& a, const PagedSched& p) {
  const int lane = threadIdx.x & 63;
  float work = 0.f, workgroups = 0.f;
  int count = 0, tiles = 0, blocks = 0;  // sequences of many rows; lane i: tiles and blocks of the i-th
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const SeqLane s(a, p, b0 + lane);
    work = __builtin_fmaf((float)s.tiles, (float)s.blocks, work);  // the same bits in both kernels
    if (p.which != kMany) continue;
    workgroups += (float)s.tiles;
    for (uint64_t some = __ballot(s.tiles > 0); some && count <= kSearched; some &= some - 1, ++count) {
      const int i = __builtin_ctzll(some), t = __builtin_amdgcn_readlane(s.tiles, i), n = __builtin_amdgcn_readlane(s.blocks, i);
      tiles = lane == count ? t : tiles;
      blocks = lane == count ? n : blocks;
    }
  }
  work = lanes_sum(work) * (float)a.Hkv;
  const float share = __builtin_amdgcn_rcpf(fmaxf(work / (float)p.target, (float)p.least));
  if (p.which != kMany) return share;
  workgroups = lanes_sum(workgroups) * (float)a.Hkv;
  if (workgroups >= (float)kMostTurns * (float)p.target) return 0.f;
  // pieces are fewer than the workgroups and `target` together
  if (count > kSearched) return workgroups < (float)(kMostTurns - 1) * (float)p.target ? share : 0.f;
  const float longest = lanes_reduce(lane < count ? (float)blocks : 0.f, [](float x, float y) { return fmaxf(x, y); });
  const float chunk = fmaxf(longest / (float)(lane + 1), (float)p.least), over = 0.99999f * __builtin_amdgcn_rcpf(chunk);  // not one piece more by its rounding
  float items = 0.f;
  for (int i = 0; i < count; ++i)
    items += (float)__builtin_amdgcn_readlane(tiles, i) * ceilf((float)__builtin_amdgcn_readlane(blocks, i) * over);
  const float turns = ceilf(items * (float)a.Hkv / (float)p.target);
  const float cost = turns > (float)kMostTurns && lane ? FLT_MAX : turns * (chunk + (float)(lane ? kPieceCost : 0));
  const float best = lanes_reduce(cost, [](float x, float y) { return fminf(x, y); });
  const int pick = __builtin_ctzll(__ballot(cost <= best) | (1ull << 63));
  return pick ? __shfl(over, pick, 64) : 0.f;
}

// token of row r of a (sequence, KV head)
__device__ __forceinline__ int token_of(const AttnPagedArgs& a, int r) { return (int)(__umulhi(2u * (uint32_t)r, a.rep_mul) >> a.rep_shift); }

// What workgroup `item` of a launch is asked to do: rows r0 .. of sequence b and KV head kvh, positions of piece z of nz.
// Called by whole waves.
struct PagedTask {
  int b = -1, kvh, z, nz, r0, rows, t0, len, pos, row;  // pos: position of the sequence's first new token
  int64_t part;  // its piece among those that leave partial outputs
  bool fine;
  __device__ PagedTask(const AttnPagedArgs& a, const PagedSched& p, int item) {
    const float over = over_chunk(a, p);
    const int lane = threadIdx.x & 63;
    int64_t before = 0, split_before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const SeqLane s(a, p, b0 + lane);
      const int pieces = s.splits(over), mine = s.tiles * a.Hkv * pieces;
      const int upto = wave_scan(mine), split = wave_scan(pieces > 1 ? mine : 0);
      const int k = __popcll(__ballot(before + upto <= item));
      if (k < 64 && b0 + k < a.B) {
        // the same in every lane, as the compiler cannot see: scalar registers
        const int at = uniform(k);
        b = b0 + at;
        const int inside = uniform(item - (int)before - (at ? __shfl(upto, at - 1, 64) : 0));
        nz = uniform(__shfl(pieces, at, 64));
        rows = uniform(__shfl(s.n, at, 64)) * a.rep;
        part = uniform((int)split_before + (at ? __shfl(split, at - 1, 64) : 0)) + inside;
        const int tiles = uniform(__shfl(s.tiles, at, 64));
        // neighbours: other KV heads, then other rows over the same positions, which an XCD's L2 then holds (pieces
        // of the same rows beside each other: 58 of 100 reads of a chunk of 1024 missed it); the last rows see most: first
        kvh = inside % a.Hkv;
        const int rest = inside / a.Hkv;
        z = rest / tiles;
        r0 = (tiles - 1 - (rest - z * tiles)) << p.lrt;
        const PackedSeq q(a.cu, a.rows, a.lens, b, a.N, a.R, a.W * a.P);
        t0 = uniform(min(max(q.t0, 0), a.N));
        len = uniform(q.len);
        pos = uniform(q.len - q.n);
        row = uniform(q.row);
        fine = uniform(q.fine) && (nz == 1 || part < p.parts);
        return;
      }
      before += __shfl(upto, 63, 64);
      split_before += __shfl(split, 63, 64);
    }
  }
  // (token, head) of row r in q, gate and out, as one index
  __device__ int64_t at(const AttnPagedArgs& a, int r) const {
    const int t = token_of(a, r);
    return (int64_t)(t0 + t) * a.H + kvh * a.rep + (r - t * a.rep);
  }
  // its gates
  __device__ int64_t gate_at(const AttnPagedArgs& a, int r) const {
    const int t = token_of(a, r);
    return (int64_t)(t0 + t) * a.gate_stride + (int64_t)(kvh * a.rep + (r - t * a.rep)) * a.gate_head;
  }
  // blocks of the piece for a tile whose last token is tlast
  __device__ void blocks(int tlast, int& blk0, int& blk1) const {
    const int all = (pos + tlast) / 32 + 1, per = (all + nz - 1) / nz;
    blk0 = min(z * per, all);
    blk1 = min(blk0 + per, all);
  }
};

// Output d .. d + M - 1 (M 4 or 8) of (token, head) i, its gates at `gate`: rounded once, after the gate.
template <bool BF, int M>
__device__ __forceinline__ void put(const AttnPagedArgs& a, int64_t i, int64_t gate, int d, const float* v) {
  using E = Half<BF>;
  float o[M];
#pragma unroll
  for (int e = 0; e < M; ++e) o[e] = v[e];
  if (a.gate) {
    const uint16_t* const g = static_cast<const uint16_t*>(a.gate) + gate + d;
    if (a.gate_wide) {
#pragma unroll
      for (int e = 0; e < M; e += 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(g + e);
        const uint32_t x[2] = {w.x, w.y};
#pragma unroll
        for (int j = 0; j < 4; ++j) o[e + j] *= sigmoid_raw(E::ld((uint16_t)(x[j >> 1] >> (16 * (j & 1)))));
      }
    } else {
#pragma unroll
      for (int e = 0; e < M; ++e) o[e] *= sigmoid_raw(E::ld(g[e]));
    }
  }
  uint32_t w[M / 2];
#pragma unroll
  for (int e = 0; e < M / 2; ++e) w[e] = E::pack((f32x2){o[2 * e], o[2 * e + 1]});
  uint16_t* const out = static_cast<uint16_t*>(a.out);
  if constexpr (M == 8) *reinterpret_cast<u32x4*>(out + i * a.hd + d) = (u32x4){w[0], w[1], w[2], w[3]};
  else *reinterpret_cast<uint2*>(out + i * a.hd + d) = make_uint2(w[0], w[1]);
}

// Zeros in the rows behind the last sequence, shared out over the launch.
__device__ __forceinline__ void clear_tail(const AttnPagedArgs& a) {
  const int from = a.B ? max(a.cu[a.B], 0) : 0;
  const int64_t n8 = (int64_t)(a.N - min(from, a.N)) * a.H * (a.hd / 8);
  u32x4* const p = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.out) + (int64_t)from * a.H * a.hd);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += (int64_t)gridDim.x * blockDim.x) p[i] = (u32x4){0, 0, 0, 0};
}

// The softmax and the sums of a wave's 16 NT rows over the positions it has seen. Weights are powers of two over a
// reference m that moves only when a score passes it by 2^kLazy, for all rows of the wave at once: mostly no rescaling
// and no exchange between lanes in the loop. They are held in kTerms 16-bit values, cut off and the rests: two of fp16 times
// 2^kScale (22 bits, down to 2^-38 of the reference's: what the attention over one sequence keeps; 2^15 at most, which
// leaves 2^1 to kLazy: 1024 tokens behind 30000 1182 us, 1138 with 2^6 and 2^-33), three of bf16 (all 24 bits; two are 2^-17
// of a weight off, which moved one output in some hundreds to its rounding's other neighbour; prompts of 2001 249 us with two
// and 279 with three), small enough that sums of V rows next to float32's largest number stay finite.
template <bool BF, int HD, int NT>
struct PagedRows {
  using E = Half<BF>;
  static constexpr int VB = HD / 16, kTerms = BF ? 3 : 2;
  static constexpr float kLazy = BF ? 6.f : 1.f, kScale = BF ? -24.f : 14.f;  // log2
  float m[NT], l[NT];  // l: this lane's share of the sum
  f32x4 acc[NT][VB];

  __device__ void init() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int i = 0; i < VB; ++i) acc[n][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
  }
  // scores s of 16 NB positions to weights pf (and, in s, as float32); last[n]: the last position that the lane's row
  // n sees, as an offset from the first of these
  template <int NB>
  __device__ void weights(f32x4 (&s)[NT][NB], bool masked, const int (&last)[NT], u32x4 (&pf)[NB / 2][kTerms][NT]) {
    const int g = (threadIdx.x & 63) >> 4;
    const float c = 1.44269504088896340736f / sqrtf((float)HD);
    float mx[NT];
    bool far = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (masked) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * b + 4 * g + e > last[n]) s[n][b][e] = -INFINITY;
      }
      mx[n] = s[n][0][0];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[n] = fmaxf(mx[n], s[n][b][e]);
      far |= (mx[n] - m[n]) * c > kLazy;  // not for -inf - -inf
    }
    if (__any(far)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x = fmaxf(mx[n], __shfl_xor(mx[n], 16, 64));
        x = fmaxf(x, __shfl_xor(x, 32, 64));
        x = fmaxf(x, m[n]);
        const float alpha = m[n] == x ? 1.f : exp2_raw((m[n] - x) * c);
        m[n] = x;
        l[n] *= alpha;
#pragma unroll
        for (int i = 0; i < VB; ++i) acc[n][i] *= alpha;
      }
    }
    // a rest of 0 times a visible V of infinity would be NaN, where its weight is not 0 and the sum is infinite. Weights that
    // are 0 stay 0: below 2^-39 of the reference's in fp16, which thousands of positions would otherwise all weigh
    const uint16_t one = masked ? 0 : E::kLeast;
    const u16x2 least = {one, one};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float off = kScale - (m[n] == -INFINITY ? 0.f : m[n]) * c;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][b][e] = exp2_raw(__builtin_fmaf(s[n][b][e], c, off));
          l[n] += s[n][b][e];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          f32x2 p = j ? s[n][b].zw : s[n][b].xy;
          uint32_t w = E::chop(p);
          pf[b / 2][0][n][2 * (b & 1) + j] = w;
          const u16x2 floor = __builtin_elementwise_min(__builtin_bit_cast(u16x2, w), least);
#pragma unroll
          for (int t = 1; t < kTerms; ++t) {
            if (t + 1 < kTerms) {
              p -= E::unpack(w);
              w = E::chop(p);
            } else {
              w = E::rest(p, w);
            }
            pf[b / 2][t][n][2 * (b & 1) + j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, w), floor));
          }
        }
      }
    }
  }
  // output tile i += V's operand times the weights
  __device__ void add(int i, u32x4 vf, const u32x4 (&pf)[kTerms][NT]) {
#pragma unroll
    for (int t = 0; t < kTerms; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n][i] = E::mma(vf, pf[t][n], acc[n][i]);
  }
  __device__ float sum(int n) const {  // over the lanes of a row
    const float x = l[n] + __shfl_xor(l[n], 16, 64);
    return x + __shfl_xor(x, 32, 64);
  }
  // reference of a row in powers of two
  __device__ float top(int n) const { return m[n] == -INFINITY ? -FLT_MAX : m[n] * (1.44269504088896340736f / sqrtf((float)HD)); }
};

// V rows that some of a tile's rows do not see would reach those as 0 x NaN if they are not finite. Blocks with such
// positions are looked at: values that are not finite are taken out of the product, and added to the sums that see them
// at the end (odd_sum).
template <bool BF>
__device__ __forceinline__ bool odd_pair(uint32_t w) {  // whether a pair of values holds one that is not finite
  const uint32_t e = BF ? 0x7F80u : 0x7C00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}
template <bool BF>
__device__ __forceinline__ uint32_t clean_pair(uint32_t w) {
  const uint32_t e = BF ? 0x7F80u : 0x7C00u;
  if ((w & e) == e) w &= 0xFFFF0000u;
  if (((w >> 16) & e) == e) w &= 0x0000FFFFu;
  return w;
}
// the sum of such values of V, dim d, at positions j0 .. j1 (0 if there is none)
template <bool BF, int HD>
__device__ __forceinline__ float odd_sum(const AttnPagedArgs& a, const int32_t* table, int kvh, int d, int j0, int j1) {
  float x = 0.f;
#pragma unroll 1
  for (int j = j0; j <= j1; ++j) {
    const int page = table[j >> a.lp];
    if (page < 0 || page >= a.n_pages) continue;
    const float v = Half<BF>::ld(static_cast<const uint16_t*>(a.vp)[(((int64_t)page * a.Hkv + kvh) * a.P + (j & (a.P - 1))) * HD + d]);
    if (!(fabsf(v) <= FLT_MAX)) x += v;
  }
  return x;
}

// NaN in the task's rows (of rt), by the whole workgroup
template <bool BF>
__device__ __forceinline__ void nan_rows(const AttnPagedArgs& a, const PagedTask& k, int rt) {
  const float v[8] = {NAN, NAN, NAN, NAN, NAN, NAN, NAN, NAN};
  for (int i = threadIdx.x; i < rt * (a.hd / 8); i += blockDim.x)
    if (k.r0 + i / (a.hd / 8) < k.rows) put<BF, 8>(a, k.at(a, k.r0 + i / (a.hd / 8)), k.gate_at(a, k.r0 + i / (a.hd / 8)), 8 * (i % (a.hd / 8)), v);
}

}  // namespace

// Few rows (16 a workgroup): the cache goes by once, and its bytes bound the kernel. Four waves take the
// blocks in turn, each with a softmax of its own; K and V go from memory to registers in 16-byte pieces, a block
// ahead: no LDS and no barrier in the loop. K's lanes read 8 dims of one position, V's PW neighbouring dims of eight
// positions, each dim of another output tile, so that two rows give a pair of a tile's operand by one permute. The
// waves are merged at the end. Heads of 256, four KV heads: 32 tokens behind 8447 to 16383 301 us, 1.63 GB at 5.4 TB/s; one
// behind 131071 97 us, 537 MB at 5.5; one behind 300 13 us, its chain of lengths, page numbers, K, V and the merge (1 of it the
// look at the last block's V).
template <bool BF, int HD>
__device__ __forceinline__ void paged_rows(const AttnPagedArgs& a, const PagedSched& p, int item, uint8_t* lds) {
  using E = Half<BF>;
  constexpr int KS = HD / 32, VB = HD / 16, PW = VB < 8 ? VB : 8, NP = VB / PW;
  typedef uint32_t vpiece __attribute__((ext_vector_type(PW / 2)));
  constexpr int OS = HD + 4;
  // queries in operand order, which a wave reads a step at a time; the merge of the waves takes the same memory
  u32x4* const qs = reinterpret_cast<u32x4*>(lds);
  float* const mo = reinterpret_cast<float*>(lds);
  float2* const ml = reinterpret_cast<float2*>(mo + 4 * 16 * OS);
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), g = lane >> 4, c = lane & 15;
  const PagedTask k(a, p, item);
  if (k.b < 0) return;
  if (!k.fine) {
    if (k.nz == 1) nan_rows<BF>(a, k, kRowsTile);
    return;
  }
  const int tfirst = uniform(token_of(a, k.r0)), tlast = uniform(token_of(a, min(k.r0 + 15, k.rows - 1)));
  int blk0, blk1;
  k.blocks(tlast, blk0, blk1);
  if (blk0 >= blk1) return;  // the merge knows
  const int klast = k.pos + tlast;  // last position any row sees; later ones of a block repeat it
  const int32_t* const table = a.table + (int64_t)k.row * a.W;
  const int64_t page_size = (int64_t)a.Hkv * a.P * HD, head = (int64_t)k.kvh * a.P * HD;
  bool bad = false;
  // first value of positions 16 j .. + 15 of K or V: they lie in one page
  auto group_at = [&](int j) {
    const int first = min(16 * j, klast), page = scalar_at(table, first >> a.lp);
    const bool out = page < 0 || page >= a.n_pages;
    bad |= out;
    return (out ? 0 : (int64_t)page * page_size) + head + (int64_t)(first & (a.P - 1) & ~15) * HD;
  };
  u32x4 kr[2][KS];
  vpiece vr[8][NP];
  int64_t at[2];
  auto load_k = [&](int blk, int b) {
    const int ln = anew(lane), left = max(klast - 32 * blk - 16 * b, 0);  // rows of the group behind it repeat one
    const uint16_t* const src = static_cast<const uint16_t*>(a.kp) + at[b];
    const uint32_t off = (uint32_t)((left < 15 ? min(ln & 15, left) : ln & 15) * HD + 8 * (ln >> 4));
#pragma unroll
    for (int s = 0; s < KS; ++s) kr[b][s] = *reinterpret_cast<const u32x4*>(src + off + 32 * s);
  };
  auto load_v = [&](int blk, int h) {  // dims (HD / NP) h ..
    const int ln = anew(lane);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int left = max(klast - 32 * blk - 16 * b, 0);
      const uint16_t* const src = static_cast<const uint16_t*>(a.vp) + at[b] + (HD / NP) * h;
      if (left >= 15) {
        const uint32_t off = (uint32_t)(4 * (ln >> 4) * HD + PW * (ln & 15));
#pragma unroll
        for (int i = 0; i < 4; ++i) vr[4 * b + i][h] = *reinterpret_cast<const vpiece*>(src + off + i * HD);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          vr[4 * b + i][h] = *reinterpret_cast<const vpiece*>(src + (uint32_t)(min(4 * (ln >> 4) + i, left) * HD + PW * (ln & 15)));
      }
    }
  };
  // a group that lies behind the last position repeats the group that holds it
  auto locate = [&](int blk) {
    at[0] = group_at(2 * blk);
    at[1] = group_at(2 * blk + 1);
  };
  int blk = blk0 + wave;
  if (blk < blk1) {
    locate(blk);
    load_k(blk, 0);
    load_k(blk, 1);
  }
  {
    const uint16_t* const q = static_cast<const uint16_t*>(a.q) + k.at(a, min(k.r0 + c, k.rows - 1)) * HD + 8 * g;
    for (int s = wave; s < KS; s += 4) qs[s * 64 + lane] = *reinterpret_cast<const u32x4*>(q + 32 * s);
  }
  if (blk < blk1) load_v(blk, 0);
  lds_sync();
  const int qpos = k.pos + token_of(a, min(k.r0 + c, k.rows - 1));
  PagedRows<BF, HD, 1> rows;
  rows.init();
  bool any_odd = false;
  for (; blk < blk1; blk += 4) {
    const bool more = blk + 4 < blk1;
    const u32x4* const ql = qs + anew(lane);
    f32x4 s[1][2] = {{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}};
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      const u32x4 q = ql[st * 64];
#pragma unroll
      for (int b = 0; b < 2; ++b) s[0][b] = E::mma(kr[b][st], q, s[0][b]);
    }
    // where two halves of V are not held beside the next K's: the second half now, K's where the first was
    if (NP == 2) load_v(blk, 1);
    if (more) {
      locate(blk + 4);
      load_k(blk + 4, 0);
      if (NP == 1) load_k(blk + 4, 1);
    }
    const int last[1] = {qpos - 32 * blk};
    const bool masked = 32 * blk + 31 > k.pos + tfirst;
    u32x4 pf[1][decltype(rows)::kTerms][1];
    rows.weights(s, masked, last, pf);
#pragma unroll
    for (int h = 0; h < NP; ++h) {
      if (masked) {  // a single token too: places behind its position repeat its row with a weight of 0
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int w = 0; w < PW / 2; ++w) odd |= odd_pair<BF>(vr[i][h][w]);
        if (__any(odd)) {
          any_odd = true;
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int w = 0; w < PW / 2; ++w) vr[i][h][w] = clean_pair<BF>(vr[i][h][w]);
        }
      }
#pragma unroll
      for (int i = 0; i < PW; ++i) {  // dim (HD / NP) h + PW c + i of the 8 positions
        u32x4 vf;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          vf[j] = __builtin_amdgcn_perm(vr[2 * j + 1][h][i >> 1], vr[2 * j][h][i >> 1], i & 1 ? 0x07060302u : 0x05040100u);
        rows.add(PW * h + i, vf, pf[0]);
      }
      if (NP == 2 && h == 0 && more) load_k(blk + 4, 1);
    }
    if (more) load_v(blk + 4, 0);
  }
  // merge of the waves: every wave's reference, sum and outputs over its own sum
  lds_sync();  // queries are no longer read
  const float ls = bad ? NAN : rows.sum(0), over = ls == 0.f ? 0.f : 1.f / ls;
  float* const mine = mo + (wave * 16 + c) * OS;
#pragma unroll
  for (int h = 0; h < NP; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < PW; i += 4)
        *reinterpret_cast<f32x4*>(mine + (HD / NP) * h + PW * (4 * g + e) + i) =
            (f32x4){rows.acc[0][PW * h + i][e], rows.acc[0][PW * h + i + 1][e], rows.acc[0][PW * h + i + 2][e],
                    rows.acc[0][PW * h + i + 3][e]} * over;
  if (g == 0) ml[wave * 16 + c] = make_float2(rows.top(0), ls);
  if (any_odd) {  // the wave's blocks that were looked at
    for (int x = blk0 + wave; x < blk1; x += 4)
      if (32 * x + 31 > k.pos + tfirst)
        for (int d = g; d < HD; d += 4) mine[d] += odd_sum<BF, HD>(a, table, k.kvh, d, 32 * x, min(32 * x + 31, qpos));
  }
  __syncthreads();
  for (int i = tid; i < 16 * HD / 8; i += 256) {
    const int rr = i / (HD / 8), d = 8 * (i % (HD / 8)), r = k.r0 + rr;
    if (r >= k.rows) continue;
    float mm = -FLT_MAX, ll = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[w * 16 + rr].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 x = ml[w * 16 + rr];
      f[w] = x.y == 0.f ? 0.f : x.y * exp2_raw(x.x - mm);
      ll += f[w];
    }
    const float inv = ll == 0.f && k.nz > 1 ? 0.f : 1.f / ll;  // no weight at all: NaN, unless another piece has one
    f32x4 o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int j = 0; j < 2; ++j) o[j] += *reinterpret_cast<const f32x4*>(mo + (w * 16 + rr) * OS + d + 4 * j) * (f[w] * inv);
    if (k.nz > 1) {
      float* const to = a.part + p.part_at + (k.part * kRowsTile + rr) * (HD + 2);
      // rows of HD + 2 floats: pairs are aligned
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<float2*>(to + d + 2 * j) = make_float2(o[j >> 1][2 * (j & 1)], o[j >> 1][2 * (j & 1) + 1]);
      if (d == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(mm, ll);
    } else {
      const float v[8] = {o[0][0], o[0][1], o[0][2], o[0][3], o[1][0], o[1][1], o[1][2], o[1][3]};
      put<BF, 8>(a, k.at(a, r), k.gate_at(a, r), d, v);
    }
  }
}

// Many rows: 32 a wave, four waves to a workgroup, over tiles of KT positions that come to LDS by DMA, a tile ahead (two
// buffers, one barrier a tile). K's operand is read as it lies, V's by transposing reads (four positions x 16
// dims per 16 lanes); 16-byte pieces of a row are XOR-swizzled by position so that reads are free of bank conflicts.
// Bound by matrix instructions and the softmax's vector ones, which overlap between the two workgroups of a CU in part: 1024
// tokens of 24 heads of 256 behind 30000 (and 23 single ones beside them) 1184 us at least, 650 TFLOP/s by the definition's
// products, half as many again with the weights' second term (bf16: twice as many with three).
constexpr int tile_keys(int hd) { return hd == 256 ? 32 : 64; }
// steps of a wave's queries that it reads from LDS, as its registers do not hold them
constexpr int tile_lds_steps(int hd) { return hd == 256 ? 1 : 0; }
constexpr int tile_lds(int hd) { return 2 * 2 * tile_keys(hd) * hd * 2 + 8192 * tile_lds_steps(hd); }

template <bool BF, int HD>
__device__ __forceinline__ void paged_tile(const AttnPagedArgs& a, const PagedSched& p, int item, uint8_t* paged_lds) {
  using E = Half<BF>;
  constexpr int NT = 2, KS = HD / 32, VB = HD / 16, KT = tile_keys(HD), NB = 2, RB = 2 * HD, NO = HD / 8;  // RB: bytes of a row
  constexpr int TB = KT * RB, NI = KT * NO / 256;  // bytes of a tile; DMA instructions of a wave for one
  constexpr int SH = HD == 64 ? 1 : 0;             // 128-byte rows: two rows to the 64 banks
  constexpr int QL = tile_lds_steps(HD);
  __shared__ int bad_s[4], odd_s[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), g = lane >> 4, c = lane & 15;
  const PagedTask k(a, p, item);
  if (k.b < 0) return;
  if (!k.fine) {
    if (k.nz == 1) nan_rows<BF>(a, k, kTileRows);
    return;
  }
  const int tlast = uniform(token_of(a, min(k.r0 + kTileRows - 1, k.rows - 1)));
  int blk0, blk1;
  k.blocks(tlast, blk0, blk1);
  if (blk0 >= blk1) return;  // the merge knows
  const int klast = k.pos + tlast;
  const int32_t* const table = a.table + (int64_t)k.row * a.W;
  const int64_t page_size = (int64_t)a.Hkv * a.P * HD, head = (int64_t)k.kvh * a.P * HD;
  auto ksw = [](int key) { return (key >> SH) & (NO < 16 ? NO - 1 : 15); };
  auto vsw = [](int key) { return ((key >> SH) & (NO < 16 ? NO / 2 - 1 : 7)) << 1; };
  constexpr int WR = KT / 4;  // positions that a wave brings: they lie in one page
  int bad = 0;
  auto page_of = [&](int j0) { return scalar_at(table, min(j0 + WR * wave, klast) >> a.lp); };
  auto issue = [&](int j0, int page, uint8_t* buf) {  // positions past the last repeat it
    const bool out = page < 0 || page >= a.n_pages;
    bad |= out;
    const int first = min(j0 + WR * wave, klast), left = klast - first, off = first & (a.P - 1);
    const int64_t base = (out ? 0 : (int64_t)page * page_size) + head + (int64_t)off * HD;
    const uint16_t* const kp = static_cast<const uint16_t*>(a.kp) + base;
    const uint16_t* const vp = static_cast<const uint16_t*>(a.vp) + base;
    const int ln = anew(lane);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int e = i * 64 + ln, r = e / NO, key = WR * wave + r, ko = (e % NO) ^ ksw(key), vo = (e % NO) ^ vsw(key);
      uint8_t* const dst = buf + wave * WR * RB + i * 1024;
      dma16(kp, (uint32_t)(min(r, left) * HD + 8 * ko) * 2, dst);
      dma16(vp, (uint32_t)(min(r, left) * HD + 8 * vo) * 2, dst + TB);
    }
  };
  const int j_end = 32 * blk1;
  int j0 = 32 * blk0;
  issue(j0, page_of(j0), paged_lds);
  int next_page = page_of(j0 + KT);
  const int rw = k.r0 + 32 * wave;
  const bool on = rw < k.rows;
  u32x4 qf[NT][KS - QL];
  u32x4* const ql = reinterpret_cast<u32x4*>(paged_lds + 4 * TB) + wave * NT * QL * 64 + lane;
  int qpos[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = min(rw + 16 * n + c, k.rows - 1);
    const uint16_t* const q = static_cast<const uint16_t*>(a.q) + k.at(a, r) * HD + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(q + 32 * s);
      if (s < QL) ql[(n * QL + s) * 64] = w;
      else qf[n][s - QL] = w;
    }
    qpos[n] = k.pos + token_of(a, r);
  }
  const int pfirst = uniform(k.pos + token_of(a, min(rw, k.rows - 1))), plast = uniform(k.pos + token_of(a, min(rw + 31, k.rows - 1)));
  PagedRows<BF, HD, NT> rows;
  rows.init();
  bool any_odd = false;
  const int wfirst = uniform(k.pos + token_of(a, k.r0));  // the workgroup's first token
  if (tid == 0) odd_s[0] = 0;
  int cur = 0;
  for (; j0 < j_end; j0 += KT, cur ^= 1) {
    // the tile has landed; every wave is done with the other buffer
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (j0 + KT < j_end) {
      issue(j0 + KT, next_page, paged_lds + (cur ^ 1) * 2 * TB);
      next_page = page_of(j0 + 2 * KT);
    }
    uint8_t* const kt = paged_lds + cur * 2 * TB;
    if (tid == 0) odd_s[cur ^ 1] = 0;
    if (j0 + KT - 1 > wfirst) {  // positions that some rows do not see
      u32x4* const v = reinterpret_cast<u32x4*>(kt + TB);
      bool odd = false;
#pragma unroll 1
      for (int i = tid; i < TB / 16; i += 256) {
        const u32x4 w = v[i];
        odd |= odd_pair<BF>(w[0]) || odd_pair<BF>(w[1]) || odd_pair<BF>(w[2]) || odd_pair<BF>(w[3]);
      }
      if (odd) odd_s[cur] = 1;
      lds_sync();
      if (odd_s[cur]) {
        any_odd = true;
#pragma unroll 1
        for (int i = tid; i < TB / 16; i += 256) {
          const u32x4 w = v[i];
          v[i] = (u32x4){clean_pair<BF>(w[0]), clean_pair<BF>(w[1]), clean_pair<BF>(w[2]), clean_pair<BF>(w[3])};
        }
        lds_sync();
      }
    }
#pragma unroll 1
    for (int sb = 0; sb < KT; sb += 32) {
      const int js = j0 + sb;
      if (!on || js > plast || js >= j_end) continue;
      f32x4 s[NT][NB];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int b = 0; b < NB; ++b) s[n][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
      const uint8_t* const ks = kt + sb * RB;
      const uint8_t* const vb = ks + TB;
      const int ln = anew(lane), g = ln >> 4, c = ln & 15;
      // operands are read a step (K) or two (V) before the products that take them, which the scheduler would undo
      u32x4 kf[2][NB], qs[2][NT];
      auto k_step = [&](int st) {
#pragma unroll
        for (int b = 0; b < NB; ++b)  // a swizzle changes 4 bits of a piece's number, the others are constants of the step
          kf[st & 1][b] = *reinterpret_cast<const u32x4*>(ks + c * RB + (((4 * (st & 3) + g) ^ ksw(c)) << 4) + 16 * b * RB + st / 4 * 256);
        if (st < QL) {
#pragma unroll
          for (int n = 0; n < NT; ++n) qs[st & 1][n] = ql[(n * QL + st) * 64];
        }
      };
      k_step(0);
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        if (st + 1 < KS) k_step(st + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int n = 0; n < NT; ++n) s[n][b] = E::mma(kf[st & 1][b], st < QL ? qs[st & 1][n] : qf[n][st < QL ? 0 : st - QL], s[n][b]);
        __builtin_amdgcn_sched_barrier(0);
      }
      const int vkey = 4 * g + (c >> 2), vlane = vkey * RB + (((c & 3) >> 1) << 4) + ((c & 1) << 3);
      u32x4 vf[3];
      auto v_tile = [&](int i) {
        const uint8_t* const at = vb + vlane + (((2 * (i & 7)) ^ vsw(vkey)) << 4) + i / 8 * 256;
        const s16x4 lo = tr_read(at), hi = tr_read(at + 16 * RB);
        vf[i % 3] = __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      };
      v_tile(0);
      v_tile(1);
      int last[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) last[n] = qpos[n] - js;
      const bool masked = js + 31 > pfirst;
      u32x4 pf[1][decltype(rows)::kTerms][NT];
      rows.weights(s, masked, last, pf);
#pragma unroll
      for (int i = 0; i < VB; ++i) {
        if (i + 2 < VB) v_tile(i + 2);
        __builtin_amdgcn_sched_barrier(0);
        rows.add(i, vf[i % 3], pf[0]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if (lane == 0) bad_s[wave] = bad;
  __syncthreads();
  bad = bad_s[0] | bad_s[1] | bad_s[2] | bad_s[3];
  if (any_odd) {  // of the piece's positions in blocks that were looked at, to the sums: through the wave's share of LDS
    constexpr int DW = HD < 128 ? HD : 128;  // dims at a time
    static_assert(32 * DW * 4 <= TB);
    float* const x = reinterpret_cast<float*>(paged_lds + wave * TB);
    const int ln = anew(lane), g = ln >> 4, c = ln & 15;
    const int from = max(32 * blk0, wfirst + 1 - KT);
#pragma unroll
    for (int d0 = 0; d0 < HD; d0 += DW) {
#pragma unroll 1
      for (int i = ln; i < 32 * DW; i += 64) {
        const int r = rw + i / DW;
        x[i] = r < k.rows ? odd_sum<BF, HD>(a, table, k.kvh, d0 + i % DW, from, min(j_end - 1, k.pos + token_of(a, r))) : 0.f;
      }
      __builtin_amdgcn_wave_barrier();  // a wave's LDS operations complete in order
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < DW / 16; ++i) rows.acc[n][d0 / 16 + i] += *reinterpret_cast<const f32x4*>(x + (16 * n + c) * DW + 16 * i + 4 * g);
      __builtin_amdgcn_wave_barrier();
    }
  }
  // a lane's outputs: row rw + 16 n + c, dims 16 i + 4 g + e
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = rw + 16 * n + c;
    const float ls = bad ? NAN : rows.sum(n), over = ls == 0.f && k.nz > 1 ? 0.f : 1.f / ls;
    if (r >= k.rows) continue;
    float* const to = a.part + p.part_at + (k.part * kTileRows + (r - k.r0)) * (HD + 2);
    const int64_t i0 = k.at(a, r), g0 = k.gate_at(a, r);
    if (k.nz > 1 && g == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(rows.top(n), ls);
#pragma unroll
    for (int i = 0; i < VB; ++i) {
      const float v[4] = {rows.acc[n][i][0] * over, rows.acc[n][i][1] * over, rows.acc[n][i][2] * over, rows.acc[n][i][3] * over};
      if (k.nz > 1) {
        *reinterpret_cast<float2*>(to + 16 * i + 4 * g) = make_float2(v[0], v[1]);
        *reinterpret_cast<float2*>(to + 16 * i + 4 * g + 2) = make_float2(v[2], v[3]);
      } else {
        put<BF, 4>(a, i0, g0, 16 * i + 4 * g, v);
      }
    }
  }
}

// One launch for both: workgroups of few and of many rows in turn, so that those bound by the cache's bytes run beside
// those bound by the matrix cores; kTurn of them at a time, one to each shader engine of each XCD, as workgroups go round
// those in order (8 at a time, all of one kind met in half of the engines: 1.78 ms in place of 1.1).
constexpr int kTurn = 32;

template <bool BF, int HD>
__global__ void __launch_bounds__(256, 2) attn_paged_kernel(AttnPagedArgs a, PagedSched few, PagedSched many, int few_wgs, int many_wgs) {
  extern __shared__ __attribute__((aligned(16))) uint8_t paged_lds[];
  clear_tail(a);
  const int group = blockIdx.x / kTurn, both = 2 * (min(few_wgs, many_wgs) / kTurn);
  bool tile;
  int item;
  if (group < both) {
    tile = group & 1;
    item = kTurn * (group >> 1) + blockIdx.x % kTurn;
  } else {
    tile = few_wgs < many_wgs;
    item = blockIdx.x - kTurn / 2 * both;
  }
  if (tile) paged_tile<BF, HD>(a, many, item, paged_lds);
  else paged_rows<BF, HD>(a, few, item, paged_lds);
}

// Outputs of split positions, from their pieces' averages weighed by their share of the row's sum: a wave to a row of
// (token, head), or, of more than kMergePieces pieces, the workgroup's waves in turn; loads of eight pieces are in
// flight at once. Bound by its reads: 71 us for 1024 tokens of 24 heads of 256 in pieces, 6 us where nothing is split.
constexpr int kMergeWaves = 8, kMergePieces = 16;

template <bool BF, int HD>
__global__ void __launch_bounds__(64 * kMergeWaves) attn_paged_merge_kernel(AttnPagedArgs a, PagedSched few, PagedSched many, int both) {
  constexpr int V = HD / 64;
  typedef float vec_t __attribute__((ext_vector_type(V)));
  __shared__ __attribute__((aligned(16))) float mo[kMergeWaves][HD];
  __shared__ float2 ml[kMergeWaves];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), d = V * lane;
  int64_t group = blockIdx.x;  // of rows: one, or as many as there are waves
  for (int pass = 0; pass < 1 + both; ++pass) {
    const PagedSched& p = pass ? many : few;
    const float over = over_chunk(a, p);
    int64_t before = 0, part0 = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const SeqLane s(a, p, b0 + lane);
      const int nz_l = s.splits(over), rows_l = nz_l > 1 ? s.n * a.H : 0, pieces = nz_l > 1 ? s.tiles * a.Hkv * nz_l : 0;
      const int upto = wave_scan(nz_l > kMergePieces ? rows_l : (rows_l + kMergeWaves - 1) / kMergeWaves);
      const int part_upto = wave_scan(pieces), all = __shfl(upto, 63, 64);
      for (; group < before + all; group += gridDim.x) {
        const int k = uniform(__popcll(__ballot(before + upto <= group)));
        const int inside = uniform((int)(group - before) - (k ? __shfl(upto, k - 1, 64) : 0));
        const int nz = uniform(__shfl(nz_l, k, 64)), tiles = uniform(__shfl(s.tiles, k, 64)), n = uniform(__shfl(s.n, k, 64));
        const int64_t part = part0 + uniform(k ? __shfl(part_upto, k - 1, 64) : 0);
        const PackedSeq q(a.cu, a.rows, a.lens, b0 + k, a.N, a.R, a.W * a.P);
        const bool shared = nz > kMergePieces;
        const int row = shared ? inside : inside * kMergeWaves + wave;
        const bool on = row < n * a.H;
        const int t = row / a.H, h = row - t * a.H, kvh = token_of(a, h), r = t * a.rep + h - kvh * a.rep, tile = r >> p.lrt;
        const int tlast = token_of(a, min(((tile + 1) << p.lrt) - 1, n * a.rep - 1));
        const int blocks = (q.len - q.n + tlast) / 32 + 1, per = (blocks + nz - 1) / nz, live = (blocks + per - 1) / per;
        float m = -FLT_MAX, l = 0.f;
        vec_t o = 0.f;
        if (!q.fine || part + (int64_t)tiles * nz * a.Hkv > p.parts) {
          l = NAN;
        } else if (on) {
          const float* const first = a.part + p.part_at + ((part + (int64_t)(tiles - 1 - tile) * a.Hkv + kvh) * p.rt() + (r - (tile << p.lrt))) * (HD + 2);
          const int64_t next = (int64_t)tiles * a.Hkv * p.rt() * (HD + 2);  // the same rows' next piece
          const int z0 = shared ? wave : 0, step = shared ? kMergeWaves : 1;
          for (int z = z0; z < live; z += 8 * step) {
            vec_t x[8];
            float2 w[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const float* const at = first + min(z + u * step, live - 1) * next;
              w[u] = *reinterpret_cast<const float2*>(at + HD);
#pragma unroll
              for (int j = 0; j < V; ++j) x[u][j] = at[d + j];
            }
            float mn = m;
#pragma unroll
            for (int u = 0; u < 8; ++u) mn = fmaxf(mn, w[u].x);
            const float keep = l * exp2_raw(m - mn);
            float f[8];
            l = keep;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              f[u] = z + u * step < live && w[u].y != 0.f ? w[u].y * exp2_raw(w[u].x - mn) : 0.f;
              l += f[u];
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            o *= keep * inv;
            m = mn;
#pragma unroll
            for (int u = 0; u < 8; ++u)
              if (f[u] != 0.f) o += x[u] * (f[u] * inv);
          }
        }
        if (shared) {
          __syncthreads();
          *reinterpret_cast<vec_t*>(&mo[wave][d]) = o;
          if (lane == 0) ml[wave] = make_float2(m, l);
          __syncthreads();
          if (wave) continue;
          m = -FLT_MAX;
          for (int w = 0; w < kMergeWaves; ++w) m = fmaxf(m, ml[w].x);
          l = 0.f;
          o = 0.f;
          for (int w = 0; w < kMergeWaves; ++w) {
            const float f = ml[w].y == 0.f ? 0.f : ml[w].y * exp2_raw(ml[w].x - m);
            l += f;
            if (f != 0.f) o += *reinterpret_cast<const vec_t*>(&mo[w][d]) * f;
          }
          o *= 1.f / l;
        }
        if (!on) continue;
        if (l == 0.f || l != l) o = NAN;  // no weight at all
        const int64_t tok = q.t0 + t;
        if (tok < 0 || tok >= a.N) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float x = o[j];
          if (a.gate) x *= sigmoid_raw(Half<BF>::ld(static_cast<const uint16_t*>(a.gate)[tok * a.gate_stride + h * a.gate_head + d + j]));
          static_cast<uint16_t*>(a.out)[(tok * a.H + h) * HD + d + j] = Half<BF>::mk(x);
        }
      }
      before += all;
      part0 += __shfl(part_upto, 63, 64);
    }
    group -= before;
  }
}

// ---- launches ------------------------------------------------------------------------------------

namespace {

struct PagedPlan {
  PagedSched few, many;
  bool tiles;  // whether sequences of many rows may be there
  int64_t floats;
};

// Pieces and workspaces that a launch may need, from what the host knows. A piece of a split sequence holds more than half
// of `target`-th of the work, so there are fewer than 2 target of them (many rows: at most kMostTurns target, as the search
// in over_chunk goes, and fewer than 2 target in proportion).
PagedPlan paged_plan(const AttnPagedArgs& a) {
  PagedPlan r = {};
  const int64_t blocks = (a.W * a.P + 31) / 32;
  r.tiles = (int64_t)a.max_new * a.rep > kFewRows;
  r.few = {4, r.tiles ? kFew : kAll, 4 * a.cus, 8, 0, 0};
  r.many = {7, kMany, (a.hd == 64 ? 4 : 2) * a.cus, 8, 0, 0};
  auto pieces = [&](const PagedSched& s, int64_t tiles, int64_t most) {
    const int64_t each = (blocks + s.least - 1) / s.least;
    return each > 1 ? std::min<int64_t>(most, tiles * a.Hkv * (each + 1)) : 0;
  };
  r.few.parts = pieces(r.few, ((int64_t)a.N * a.rep >> 4) + a.B, 2 * r.few.target + 64);
  r.floats = r.few.parts * kRowsTile * (a.hd + 2);
  if (r.tiles) {
    r.many.parts = pieces(r.many, ((int64_t)a.N * a.rep >> 7) + a.B, kMostTurns * r.many.target + 64);
    r.many.part_at = r.floats;
    r.floats += r.many.parts * kTileRows * (a.hd + 2);
  }
  return r;
}

template <bool BF, int HD>
hipError_t launch_attn_paged_t(const AttnPagedArgs& a, hipStream_t s) {
  constexpr int rows_lds = 4 * 16 * (HD + 4) * 4 + 4 * 16 * 8, most_lds = std::max(rows_lds, tile_lds(HD));
  const PagedPlan p = paged_plan(a);
  auto grid = [&](const PagedSched& q) {  // whole turns
    int64_t tiles = ((int64_t)a.N * a.rep >> q.lrt) + a.B;
    if (q.which == kFew) tiles = std::min<int64_t>(tiles, (int64_t)a.B * (kFewRows >> q.lrt));
    const int64_t most = q.which == kMany ? std::max<int64_t>(tiles * a.Hkv, q.parts) : tiles * a.Hkv + q.target;
    return (most + 64 + kTurn - 1) / kTurn * kTurn;
  };
  const int64_t few = grid(p.few), many = p.tiles ? grid(p.many) : 0;
  if (few + many >= 1 << 24) return hipErrorInvalidConfiguration;  // threads along x are counted in 32 bits
  static LdsLimit limit;
  const hipError_t e = limit.raise((const void*)attn_paged_kernel<BF, HD>, most_lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((attn_paged_kernel<BF, HD>), dim3((unsigned)(few + many)), dim3(256), p.tiles ? most_lds : rows_lds, s, a,
                     p.few, p.many, (int)few, (int)many);
  if (p.few.parts || p.many.parts) {
    const unsigned most = (unsigned)std::min<int64_t>((int64_t)a.N * a.H, 4 * a.cus);
    hipLaunchKernelGGL((attn_paged_merge_kernel<BF, HD>), dim3(most), dim3(64 * kMergeWaves), 0, s, a, p.few, p.many, (int)p.tiles);
  }
  return hipGetLastError();
}

}  // namespace

int64_t attn_paged_work(const AttnPagedArgs& a) {
  if (a.N == 0) return 0;
  return paged_plan(a).floats;
}

hipError_t launch_attn_paged(bool bf16, const AttnPagedArgs& a, hipStream_t s) {
  auto dims = [&](auto bf) -> hipError_t {
    constexpr bool BF = decltype(bf)::value;
    if (a.hd == 256) return launch_attn_paged_t<BF, 256>(a, s);
    if (a.hd == 128) return launch_attn_paged_t<BF, 128>(a, s);
    if (a.hd == 64) return launch_attn_paged_t<BF, 64>(a, s);
    return hipErrorInvalidValue;
  };
  return bf16 ? dims(std::true_type{}) : dims(std::false_type{});
}

}  // namespace gsq
