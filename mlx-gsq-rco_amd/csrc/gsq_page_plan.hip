// Pages of a K/V cache handed out on the GPU: from the lengths of requests and the new tokens of a step's sequences, the
// pages each one takes, its row of the block table, and the position and slot of each packed token. (The reference has
// one sequence and a cache without pages, behind mlx_gsq/models/qwen35.py:114-152.)
//
// One workgroup, a thread to a sequence: need_b = max(0, ceil((len + new) / P) - held) and its prefix sums decide who is
// served, in the order of the sequences; pages come off the end of the list of free ones, and go back to it in the
// opposite order. Whole numbers throughout, every sum in 64 bits, no atomics: the result is the definition's.
// Bound by its chain of three prefix sums and the reads before them: 6 us for 16 single tokens, one workgroup for at most
// 1024 sequences being less than a second launch for a sum across workgroups.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "gsq_common.h"

namespace gsq {

constexpr int kPlanThreads = 1024;  // sequences of a step at most
// Tokens that the one workgroup lays out as well; those of larger steps have a launch of their own (us, without and with:
// one sequence of 512 5.6 and 7.4, of 4096 7.6 and 7.4, of 8191 9.9 and 7.6; four of up to 8191 beside 250 tokens, and
// their release: 46 and 32).
constexpr int kPlanTokens = 4096;

// Inclusive prefix sums over the workgroup; red: 16 values of LDS.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 63) red[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += red[w];
  return v;
}

// Whether an earlier sequence names the request of this thread's. req: every sequence's, in LDS.
__device__ __forceinline__ bool named_before(const int* req, int r, int b) {
  bool again = false;
  const int4* const four = reinterpret_cast<const int4*>(req);
#pragma unroll 4
  for (int i = 0; i < b / 4; ++i) {
    const int4 v = four[i];
    again |= v.x == r || v.y == r || v.z == r || v.w == r;
  }
  for (int i = b & ~3; i < b; ++i) again |= req[i] == r;
  return again;
}

// first b with end[b] > i, of ascending ends (n if there is none)
__device__ __forceinline__ int find_end(const int64_t* end, int n, int64_t i) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (end[mid] <= i) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// TOKENS: positions and slots of the tokens too.
template <bool TOKENS>
__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(PagePlanArgs a) {
  __shared__ __attribute__((aligned(16))) int req[kPlanThreads];
  __shared__ int base[kPlanThreads], old[kPlanThreads], row[kPlanThreads];
  __shared__ int64_t end[kPlanThreads], take[kPlanThreads], red[16];
  const int b = threadIdx.x;
  const bool on = b < a.B;
  const int r = on ? a.requests[b] : -1, at = min(max(r, 0), a.R - 1);
  const int64_t n = on ? a.fresh[b] : 0;
  const int64_t len = a.lengths[at], held = a.held[at];
  const int avail = min(max(a.n_free[0], 0), a.n_pages);
  req[b] = r;
  const int64_t stop = block_scan(n > 0 ? n : 0, red);  // its barriers also publish req
  const int64_t total = len + n;
  const bool fine = on && r >= 0 && r < a.R && n >= 0 && len >= 0 && held >= 0 && held <= a.W && total <= a.W * a.P &&
                    stop <= a.N && !named_before(req, r, b);
  int64_t need = fine ? (total + a.P - 1) / a.P - held : 0;
  if (need < 0) need = 0;
  const int64_t cum = block_scan(need, red);
  const bool served = fine && (need == 0 || cum <= avail);
  // what is taken: the prefix sums of those served (all before the first that is not)
  const int64_t taken = block_scan(served ? need : 0, red);
  end[b] = stop < a.N ? stop : a.N;
  take[b] = taken;
  base[b] = (int)len;
  old[b] = (int)held;
  row[b] = served ? r : -1;
  __syncthreads();
  if (on) {
    a.cu[b + 1] = (int)end[b];
    a.rows[b] = row[b];
    a.lens[b] = served ? (int)total : 0;
    if (served) a.held[r] = (int)(held + need);
  }
  const int64_t all = a.B ? take[a.B - 1] : 0;
  for (int64_t i = b; i < all; i += kPlanThreads) {  // page i of those taken, in the order of the sequences
    const int s = find_end(take, a.B, i);
    const int64_t first = s ? take[s - 1] : 0;
    a.table[(int64_t)row[s] * a.W + old[s] + (i - first)] = a.free[avail - 1 - i];
  }
  for (int64_t t = b; TOKENS && t < a.N; t += kPlanThreads) {
    const int s = find_end(end, a.B, t);
    int64_t p = -1, slot = -1;
    if (s < a.B && row[s] >= 0) {
      p = base[s] + (t - (s ? end[s - 1] : 0));
      const int j = (int)p / a.P;  // positions fit in 32 bits, as lens does
      // a page of this step comes from the list: the table may not hold it yet
      const int page = j < old[s] ? a.table[(int64_t)row[s] * a.W + j] : a.free[avail - 1 - ((s ? take[s - 1] : 0) + j - old[s])];
      slot = page >= 0 && page < a.n_pages ? (int64_t)page * a.P + (p - j * a.P) : -1;
    }
    a.pos[t] = p;
    a.slots[t] = slot;
  }
  if (b == 0) {
    a.cu[0] = 0;
    a.n_free[0] = (int)(avail - all);
  }
}

// Positions and slots of the tokens of a step that has been laid out, a thread to each.
__global__ void __launch_bounds__(256) page_tokens_kernel(PagePlanArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.N) return;
  int lo = 0, hi = a.B;  // first sequence that ends behind t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  int64_t p = -1, slot = -1;
  if (lo < a.B && a.rows[lo] >= 0) {
    p = a.lens[lo] - (a.cu[lo + 1] - (int)t);
    const int j = (int)p / a.P;
    const int page = a.table[(int64_t)a.rows[lo] * a.W + j];
    slot = page >= 0 && page < a.n_pages ? (int64_t)page * a.P + (p - j * a.P) : -1;
  }
  a.pos[t] = p;
  a.slots[t] = slot;
}

__global__ void __launch_bounds__(kPlanThreads) page_advance_kernel(const int32_t* rows, const int32_t* lens, int32_t* lengths,
                                                                    int B, int R) {
  const int b = threadIdx.x;
  if (b < B && rows[b] >= 0 && rows[b] < R) lengths[rows[b]] = lens[b];
}

// Pages of the requests back to the list, so that the first page of the first request ends on top: what page_plan took
// last for these requests, in this order, lies there as before.
__global__ void __launch_bounds__(kPlanThreads) page_release_kernel(PageReleaseArgs a) {
  __shared__ __attribute__((aligned(16))) int req[kPlanThreads];
  __shared__ int64_t back[kPlanThreads], red[16];
  const int b = threadIdx.x;
  const int r = b < a.B ? a.requests[b] : -1;
  const int64_t held = r >= 0 && r < a.R ? a.held[r] : 0;
  const int64_t avail = min(max(a.n_free[0], 0), a.n_pages);
  req[b] = r;
  __syncthreads();
  const bool fine = r >= 0 && r < a.R && held >= 0 && held <= a.W && !named_before(req, r, b);
  back[b] = block_scan(fine ? held : 0, red);
  __syncthreads();
  const int64_t all = a.B ? back[a.B - 1] : 0;
  for (int64_t i = b; i < all; i += kPlanThreads) {
    const int s = find_end(back, a.B, i);
    int32_t* const e = a.table + (int64_t)req[s] * a.W + (i - (s ? back[s - 1] : 0));
    const int64_t to = avail + all - 1 - i;
    if (to < a.n_pages) a.free[to] = *e;  // more pages than there are: not the requests' own
    *e = -1;
  }
  __syncthreads();
  if (fine) {
    a.held[r] = 0;
    a.lengths[r] = 0;
  }
  if (b == 0) a.n_free[0] = (int)(avail + all < a.n_pages ? avail + all : a.n_pages);
}

hipError_t launch_page_plan(const PagePlanArgs& a, hipStream_t s) {
  if (a.N <= kPlanTokens) {
    hipLaunchKernelGGL(page_plan_kernel<true>, dim3(1), dim3(kPlanThreads), 0, s, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(page_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, s, a);
  hipLaunchKernelGGL(page_tokens_kernel, dim3((unsigned)((a.N + 255) / 256)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_page_advance(const int32_t* rows, const int32_t* lens, int32_t* lengths, int B, int R, hipStream_t s) {
  hipLaunchKernelGGL(page_advance_kernel, dim3(1), dim3(kPlanThreads), 0, s, rows, lens, lengths, B, R);
  return hipGetLastError();
}

hipError_t launch_page_release(const PageReleaseArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(page_release_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace gsq
