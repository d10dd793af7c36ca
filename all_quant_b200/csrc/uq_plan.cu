// Block tables and slot maps of a step from its requests' lengths: the two arrays that the append (slot of every new token)
// and the verify launch (page table) take.  No counterpart in the reference, whose engine brings both.
//
//   held_b = ceil((len_b - n_b) / PAGE)     pages that request b had before the step (n_b of its len_b tokens are new)
//   need_b = ceil(len_b / PAGE) - held_b    pages it has to get
//   off_b  = sum of need_i over i < b       its place in the list of free pages
//   table[b, held_b + j] = free[off_b + j], j < need_b
//   slot[t] = table[b, p / PAGE] * PAGE + p % PAGE, with p = len_b - n_b + (t - start_b) for token t of request b
//
// Bound by latency: lengths -> prefix sums -> bisection -> table -> slot, one after the other, behind a launch (3.0 us from a graph for 2
// requests, 4.6 for 300 with 73 121 new tokens, 6.6 for 64 prompts of 257 430 tokens; their bytes would take 0.3 at the most).  The last one's 503 blocks
// are more than the device holds at once (three per SM): those that start late go through the chain again.
// One launch, nothing kept between blocks: every block works the two prefix sums (pages, tokens) out for itself in shared memory
// (a few KB of lengths out of L2), then takes its share of the tokens and of the pages handed out.  A token finds its request by
// bisection of the starts; a page that this step hands out is read from the free list, never from the table, so that no block
// waits for another one's table entries.
#include <climits>

#include "uq_common.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kTokensPerBlock = kThreads;       // tokens a block is launched for (one / two / four per thread: 300 requests 4.6 / 5.5 / 7.6 us, 64 prompts 6.6 / 6.7 / 6.3)
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRequests = 16384;             // two prefix sums and a position of 4 bytes each in shared memory

struct PlanArgs {
  const int32_t* seq_lens;    // [B]
  const int32_t* starts;      // [B + 1] first new token of every request (null: uniform or whole prompts)
  int32_t* table;             // [B, >= max_pages], row stride below
  const int32_t* free_pages;  // [n_free]
  int64_t* slots;             // [T]
  int32_t* taken;             // [1] pages handed out (null: none are, the table is complete already and is only read)
  long long stride;
  long long T, n_free;
  int B, K, PAGE, max_pages;  // K > 0: K new tokens per request; K == 0: starts, or, without them, whole prompts
};

// new tokens of request b and its stored length, both made harmless (a length below zero is zero)
UQ_DEV void request(const PlanArgs& a, int b, int& len, int& n) {
  len = max(a.seq_lens[b], 0);
  n = a.K > 0 ? a.K : (a.starts ? max((int)min((long long)a.starts[b + 1] - a.starts[b], (long long)INT_MAX), 0) : len);
}
UQ_DEV int pages_of(long long tokens, int page, int most) {   // (tokens <= INT_MAX: a 32-bit division)
  return tokens <= 0 ? 0 : (int)min(((unsigned)tokens - 1u) / (unsigned)page + 1u, (unsigned)most);
}

// the last i with v[i] <= x, v[0..n] not decreasing and v[0] <= x
UQ_DEV int last_not_above(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Exclusive prefix sums of `mine` over the block's threads (saturating at INT_MAX); the block's total in `total`.
UQ_DEV long long block_exclusive(long long mine, long long* warp_sums, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  long long before = 0;
  total = 0;
  for (int w = 0; w < kThreads / 32; w++) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  __syncthreads();
  return before + incl - mine;
}
UQ_DEV int saturate(long long v) { return (int)min(v, (long long)INT_MAX); }

__global__ void __launch_bounds__(kThreads) uq_plan_kernel(PlanArgs a, int pdl) {
  extern __shared__ int sm[];
  int* off = sm;                  // [B + 1] pages handed out before request b
  int* first = sm + a.B + 1;      // [B + 1] first new token of request b
  int* behind = first + a.B + 1;  // [B] its position: what was stored before (below zero: more new tokens than stored ones)
  __shared__ long long sums[kWarps];
  const int tid = threadIdx.x;
  uq_pdl_wait();
  if (pdl) uq_pdl_release();
  {
    const int per = (a.B + kThreads - 1) / kThreads, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    long long pages = 0, tokens = 0;
    for (int b = b0; b < b1; b++) {
      int len, n;
      request(a, b, len, n);
      pages += max(pages_of(len, a.PAGE, a.max_pages) - pages_of((long long)len - n, a.PAGE, a.max_pages), 0);
      tokens += n;
    }
    long long all_pages, all_tokens = 0;
    pages = block_exclusive(pages, sums, all_pages);
    if (!a.starts) tokens = block_exclusive(tokens, sums, all_tokens);
    for (int b = b0; b < b1; b++) {
      int len, n;
      request(a, b, len, n);
      off[b] = saturate(pages);
      first[b] = a.starts ? a.starts[b] : saturate(tokens);
      behind[b] = (int)max((long long)len - n, (long long)INT_MIN);
      pages += max(pages_of(len, a.PAGE, a.max_pages) - pages_of((long long)len - n, a.PAGE, a.max_pages), 0);
      tokens += n;
    }
    if (tid == 0) {
      off[a.B] = saturate(all_pages);
      first[a.B] = a.starts ? a.starts[a.B] : saturate(all_tokens);
    }
  }
  __syncthreads();
  const long long step = (long long)gridDim.x * kThreads;
  for (long long t = (long long)blockIdx.x * kThreads + tid; t < a.T; t += step) {
    int64_t slot = -1;
    if (t >= first[0] && t < first[a.B]) {
      const int b = last_not_above(first, a.B - 1, (int)t);
      const long long i = t - first[b], pos = (long long)behind[b] + i;
      // (starts that fall are no starts: such a request has no tokens, whatever lies between it and the next)
      if (pos >= 0 && i < (a.K > 0 ? (long long)a.K : (long long)first[b + 1] - first[b])) {
        const int pi = (int)((unsigned)pos / (unsigned)a.PAGE);
        if (pi < a.max_pages) {
          const int held = pages_of(behind[b], a.PAGE, a.max_pages);
          int page = -1;
          if (pi < held || !a.taken) page = a.table[b * a.stride + pi];
          else {
            const long long at = off[b] + (pi - held);
            if (at < a.n_free) page = a.free_pages[at];
          }
          if (page >= 0) slot = (int64_t)page * a.PAGE + (pos - (long long)pi * a.PAGE);
        }
      }
    }
    a.slots[t] = slot;
  }
  if (a.taken) {
    const int total = off[a.B];
    for (long long i = (long long)blockIdx.x * kThreads + tid; i < total; i += step) {
      const int b = last_not_above(off, a.B - 1, (int)i);
      a.table[b * a.stride + pages_of(behind[b], a.PAGE, a.max_pages) + ((int)i - off[b])] = i < a.n_free ? a.free_pages[i] : -1;
    }
    if (blockIdx.x == 0 && tid == 0) *a.taken = total;
  }
}

}  // namespace

cudaError_t uq_plan_dispatch(const int32_t* seq_lens, const int32_t* starts, int K, int32_t* table, long long stride, const int32_t* free_pages, long long n_free,
                             int64_t* slots, int32_t* taken, int B, long long T, int PAGE, int max_pages, int sms, cudaStream_t s) {
  if (B < 0 || B > kMaxRequests || K < 0 || (K > 0 && starts) || T < 0 || T > INT_MAX || PAGE < 1 || max_pages < 0 || n_free < 0 || stride < max_pages) return cudaErrorInvalidValue;
  if ((long long)B * max_pages > INT_MAX || (B > 0 && (!seq_lens || (max_pages > 0 && !table))) || (T > 0 && !slots) || (n_free > 0 && (!free_pages || !taken))) return cudaErrorInvalidValue;
  const size_t smem = 3 * (size_t)(B + 1) * sizeof(int);
  if (smem + kWarps * sizeof(long long) > 48 * 1024) {   // what a launch gets unasked holds the warps' sums as well
    const cudaError_t e = cudaFuncSetAttribute(uq_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(3 * (kMaxRequests + 1) * sizeof(int)));
    if (e != cudaSuccess) { cudaGetLastError(); return e; }
  }
  PlanArgs a{seq_lens, starts, table, free_pages, slots, taken, stride, T, n_free, B, K, PAGE, max_pages};
  const long long want = (T + kTokensPerBlock - 1) / kTokensPerBlock;
  const unsigned blocks = (unsigned)(want < 1 ? 1 : (want > 4 * sms ? 4 * sms : want));
  const bool pdl = uq_pdl_on();
  return uq_launch(uq_plan_kernel, dim3(blocks), (unsigned)kThreads, smem, s, pdl, a, (int)pdl);
}
