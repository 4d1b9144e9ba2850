// Pages for a batch of requests, from their lengths, on the GPU.
//
// A request b has len_b tokens cached in the first ceil(len_b / 64) pages of its row of the block table and brings
// n_b new ones.  Free pages stand in a ring (head, count).  With cu the exclusive prefix sum of n,
//   total_b = len_b + n_b,  need_b = ceil(total_b / 64) - ceil(len_b / 64),  cum_b = need_0 + ... + need_b,
// request b is admitted if its tokens fit (total_b <= 64 W, cu_b + n_b <= N) and its pages are there (need_b = 0 or
// cum_b <= count); page j of the new ones is free[head + cum_b - need_b + j].  The plan changes no state that is
// committed: table entries past a request's committed pages are scratch, so planning twice gives the same plan.
//
// Bound: latency (a few KB moved).  One launch: every workgroup scans the at most 1024 requests itself (4 per
// thread, two block scans) and then writes its own 256 tokens' slots and positions and its share of the new table
// entries, so no workgroup waits for another and there is no second launch.
#include "paged.h"

using namespace paged;

namespace {

constexpr int NT = 256, PER = MAX_ROWS / NT;

__device__ __forceinline__ long long pages_of(long long tokens) { return (tokens + PAGE - 1) / PAGE; }

__global__ void __launch_bounds__(NT)
page_plan_kernel(const int* __restrict__ new_lens, const int* __restrict__ lengths, int* __restrict__ table,
                 const int* __restrict__ ring_pages, const int* __restrict__ ring, int* __restrict__ cu,
                 int* __restrict__ kv_lens, int* __restrict__ taken, int* __restrict__ positions,
                 int* __restrict__ slots, int B, int W, int num, int N) {
  __shared__ long long red[NT / 64];
  __shared__ int s_end[MAX_ROWS], s_cum[MAX_ROWS], s_len[MAX_ROWS];   // s_len: -1 where the request is not admitted
  __shared__ int s_first[MAX_ROWS];                                   // new pages before the request's own
  const int t = threadIdx.x;
  const int head = ring[0], count = ring[1];

  long long n[PER], len[PER], sum = 0, all;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = t * PER + i;
    n[i] = b < B ? max(new_lens[b], 0) : 0;
    len[i] = b < B ? max(lengths[b], 0) : 0;
    sum += n[i];
  }
  long long end = block_scan<NT>(sum, red, &all) - sum;
  long long need[PER], ends[PER];
  bool fits[PER];
  sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    end += n[i];
    ends[i] = end;
    fits[i] = len[i] + n[i] <= (long long)PAGE * W && end <= N;
    need[i] = fits[i] ? pages_of(len[i] + n[i]) - pages_of(len[i]) : 0;
    sum += need[i];
  }
  long long cum = block_scan<NT>(sum, red, &all) - sum;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = t * PER + i;
    cum += need[i];
    const bool ok = fits[i] && (need[i] == 0 || cum <= count);
    if (b < B) {
      const int e = (int)min(ends[i], (long long)INT_MAX);
      s_end[b] = e;
      s_cum[b] = (int)cum;
      s_first[b] = (int)(cum - need[i]);
      s_len[b] = ok ? (int)len[i] : -1;
      if (blockIdx.x == 0) {
        if (b == 0) cu[0] = 0;
        cu[b + 1] = e;
        kv_lens[b] = ok ? (int)(len[i] + n[i]) : 0;
        taken[b] = ok ? (int)need[i] : -1;
      }
    }
  }
  __syncthreads();

  const long long h = ((long long)head % num + num) % num;   // in bounds whatever the ring says
  // (unsigned: one stride past N up to 2^31 - 1 does not wrap)
  const unsigned stride = gridDim.x * NT, first = blockIdx.x * NT + t;
  for (unsigned i = first; i < (unsigned)N; i += stride) {
    const int b = upper_bound(s_end, B, (int)i);
    int pos = 0, slot = -1;
    if (b < B && s_len[b] >= 0) {
      pos = s_len[b] + ((int)i - (b > 0 ? s_end[b - 1] : 0));
      const int j = pos / PAGE, have = (int)pages_of(s_len[b]);
      const int page = j < have ? table[(size_t)b * W + j] : ring_pages[(h + s_first[b] + j - have) % num];
      slot = page * PAGE + pos % PAGE;
    }
    positions[i] = pos;
    slots[i] = slot;
  }
  // new entries: they lie past the committed pages, which are all that the loop above reads
  const unsigned pages = (unsigned)min(all, (long long)max(count, 0));
  for (unsigned k = first; k < pages; k += stride) {
    const int b = upper_bound(s_cum, B, (int)k);
    if (b < B && s_len[b] >= 0) {
      const int j = (int)pages_of(s_len[b]) + ((int)k - s_first[b]);
      table[(size_t)b * W + j] = ring_pages[(h + k) % num];
    }
  }
}

// Takes the plan's pages out of the ring, sets the lengths and puts the pages of finished requests back, in the
// order of the requests.  Pages taken follow from the lengths before and after, so committing a plan again takes
// none (but for a request that finished with it, whose length is then 0).  One workgroup: a few KB.
__global__ void __launch_bounds__(NT)
page_commit_kernel(const int* __restrict__ kv_lens, const int* __restrict__ taken, const uint8_t* __restrict__ finished,
                   int* __restrict__ lengths, const int* __restrict__ table, int* __restrict__ ring_pages,
                   int* __restrict__ ring, int B, int W, int num) {
  __shared__ long long red[NT / 64];
  __shared__ int s_cum[MAX_ROWS];
  const int t = threadIdx.x;
  const long long head = ((long long)ring[0] % num + num) % num, count = min(max(ring[1], 0), num);
  long long took = 0, back = 0, popped, pushed;
  long long give[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = t * PER + i;
    give[i] = 0;
    if (b < B) {
      const long long before = min((long long)max(lengths[b], 0), (long long)PAGE * W);
      long long now = taken[b] >= 0 ? min((long long)max(kv_lens[b], 0), (long long)PAGE * W) : before;
      took += max(pages_of(now) - pages_of(before), 0ll);
      if (finished != nullptr && finished[b]) {
        give[i] = pages_of(now);
        now = 0;
      }
      lengths[b] = (int)now;
    }
    back += give[i];
  }
  block_scan<NT>(took, red, &popped);
  long long cum = block_scan<NT>(back, red, &pushed) - back;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = t * PER + i;
    cum += give[i];
    if (b < B) s_cum[b] = (int)min(cum, (long long)INT_MAX);
  }
  __syncthreads();
  popped = min(popped, count);
  const long long room = num - (count - popped);
  pushed = min(pushed, room);                       // a ring never holds more than its pages
  const long long tail = head + count;
  for (int k = t; k < (int)pushed; k += NT) {
    const int b = upper_bound(s_cum, B, k);
    const int j = k - (b > 0 ? s_cum[b - 1] : 0);
    ring_pages[(tail + k) % num] = table[(size_t)b * W + j];
  }
  if (t == 0) {
    ring[0] = (int)((head + popped) % num);
    ring[1] = (int)(count - popped + pushed);
  }
}

}  // namespace

extern "C" {

int mivgpu_page_plan(const int* new_lens, const int* lengths, int* table, const int* ring_pages, const int* ring,
                     int* cu, int* kv_lens, int* taken, int* positions, int* slots, int B, int W, int num, int N,
                     hipStream_t s) {
  if (B <= 0 || B > MAX_ROWS || W <= 0 || num <= 0 || N < 0 || (long long)num * PAGE > INT_MAX ||
      (long long)W * PAGE > INT_MAX)
    return -1;
  const int grid = N > 1024 * NT ? 1024 : max(1, (N + NT - 1) / NT);
  hipLaunchKernelGGL(page_plan_kernel, dim3(grid), dim3(NT), 0, s, new_lens, lengths, table, ring_pages, ring, cu,
                     kv_lens, taken, positions, slots, B, W, num, N);
  return (int)hipGetLastError();
}

int mivgpu_page_commit(const int* kv_lens, const int* taken, const void* finished, int* lengths, const int* table,
                       int* ring_pages, int* ring, int B, int W, int num, hipStream_t s) {
  if (B <= 0 || B > MAX_ROWS || W <= 0 || num <= 0 || (long long)num * PAGE > INT_MAX || (long long)W * PAGE > INT_MAX)
    return -1;
  hipLaunchKernelGGL(page_commit_kernel, dim3(1), dim3(NT), 0, s, kv_lens, taken, (const uint8_t*)finished, lengths,
                     table, ring_pages, ring, B, W, num);
  return (int)hipGetLastError();
}

}  // extern "C"
