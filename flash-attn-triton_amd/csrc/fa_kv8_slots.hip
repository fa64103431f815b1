// Pages and slots of the next tokens of a batch of requests, from their
// lengths (fa_kvcache_slots).
//
// Request b holds o tokens and gets n: it needs ceil((o + n) / page) -
// ceil(o / page) pages, taken from the free list in the order of the requests
// (a prefix sum), and packed row cu[b] + i is its token o + i, in slot
// table[b][pos / page] * page + pos % page.  A request that does not fit its
// table row or the packed rows, or whose prefix of page needs passes the free
// pages (unless it needs none), gets no page: its slots are -1 and its length
// stays.  The index handed back counts the needs up to the last request served.
//
// One launch without any exchange between workgroups: every workgroup forms
// the prefix sums of the lengths itself, 12 bytes of LDS per request, and
// serves its own packed rows.  The new pages begin at page boundaries, so the
// row of a page's first token writes the table entry and every row of a new
// page knows its number from the list; only rows on a page that the request
// already holds read the table, in entries no workgroup writes.
//
// Bound: latency.  A step of 64 requests moves 3 KiB; two sums over the
// lengths with their barriers and a binary search are what it takes.
#include "fa_kv8.h"

namespace fa {

namespace {

constexpr int64_t kIntMax = 0x7fffffff;

// Exclusive prefix over a workgroup of kThreads of each thread's `x`; *total gets the sum.
template <int kThreads>
__device__ inline int64_t block_prefix(int64_t x, int64_t* wave_sum, int64_t* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int64_t s = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t t = __shfl_up(s, d, 64);
    if (lane >= d) s += t;
  }
  __syncthreads();   // wave_sum may still be read from the previous call
  if (lane == 63) wave_sum[w] = s;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int u = 0; u < kThreads / 64; ++u) {
    if (u < w) before += wave_sum[u];
    all += wave_sum[u];
  }
  *total = all;
  return before + s - x;
}

__device__ inline int clamp_len(int n) { return n < 0 ? 0 : n > (1 << 30) ? 1 << 30 : n; }

}  // namespace

// kChunk requests' sums are in LDS at a time, kPer per thread.
template <int kThreads, int kPer>
__global__ __launch_bounds__(kThreads) void kvcache_slots_kernel(const SlotsParams p) {
  constexpr int kChunk = kThreads * kPer;
  __shared__ int cu[kChunk + 1];        // first packed row of each request of the chunk (clamped)
  __shared__ int pages[kChunk];         // pages taken before it; -1: not served
  __shared__ int old_len[kChunk];
  __shared__ int64_t wave_sum[kThreads / 64];
  __shared__ int taken;
  const int tid = threadIdx.x;
  const int64_t start = p.free_start != nullptr ? max(p.free_start[0], 0) : 0;
  const int64_t left = max(p.n_free - start, (int64_t)0);
  if (tid == 0) taken = 0;

  int64_t row_base = 0, page_base = 0;   // sums over the chunks before this one
  for (int c0 = 0; c0 < p.batch; c0 += kChunk) {
    const int n = min(kChunk, p.batch - c0);
    // Thread t owns requests kPer t .. of the chunk.
    int o[kPer], a[kPer];
    int64_t rows = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = tid * kPer + i;
      o[i] = b < n ? clamp_len(p.cached[c0 + b]) : 0;
      a[i] = b < n ? clamp_len(p.added[c0 + b]) : 0;
      rows += a[i];
    }
    int64_t all_rows, all_pages;
    int64_t r = row_base + block_prefix<kThreads>(rows, wave_sum, &all_rows);
    int have[kPer], need[kPer];
    bool fits[kPer];
    int64_t want = 0, r1 = r;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      r1 += a[i];
      const int64_t end = (int64_t)o[i] + a[i];
      const int hv = (int)fdiv(o[i] + p.page.d - 1, p.page);
      // (end is at most 2^31: its division stays in 32 bits below 2^31)
      const int upto = end > 0 ? (int)fdiv((uint32_t)(end - 1), p.page) + 1 : 0;
      fits[i] = upto <= p.cols && r1 <= p.rows;
      have[i] = hv;
      need[i] = fits[i] ? upto - hv : 0;
      want += need[i];
    }
    int64_t before = page_base + block_prefix<kThreads>(want, wave_sum, &all_pages);
    int most = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = tid * kPer + i;
      const int64_t upto = before + need[i];
      const bool served = fits[i] && (need[i] == 0 || upto <= left);
      if (b < n) {
        cu[b] = (int)min(r, (int64_t)p.rows);
        pages[b] = served ? (int)min(before, kIntMax) : -1;
        old_len[b] = o[i];
        if (served) most = (int)min(upto, kIntMax - start);
        if (blockIdx.x == 0) {
          p.cu[c0 + b] = (int)min(r, (int64_t)p.rows);
          p.seqlens[c0 + b] = served ? o[i] + a[i] : o[i];
        }
      }
      r += a[i];
      before = upto;
    }
    if (most > 0) atomicMax(&taken, most);
    row_base += all_rows;
    page_base += all_pages;
    if (tid == 0) cu[n] = (int)min(row_base, (int64_t)p.rows);
    __syncthreads();

    const int lo = cu[0], hi = cu[n];
    for (int64_t row = (int64_t)blockIdx.x * kThreads + tid; row < hi;
         row += (int64_t)gridDim.x * kThreads) {
      if (row < lo) continue;
      // The last request that starts at or before the row.
      int b = 0;
      for (int step = kChunk / 2; step > 0; step /= 2)
        if (b + step < n && cu[b + step] <= row) b += step;
      const int pos = old_len[b] + ((int)row - cu[b]);
      int64_t slot = -1;
      if (pages[b] >= 0) {
        const int col = (int)fdiv(pos, p.page), at = pos - col * (int)p.page.d;
        const int held = (int)fdiv(old_len[b] + p.page.d - 1, p.page);
        int32_t* entry = p.table + (int64_t)(c0 + b) * p.table_stride + col;
        int page;
        if (col < held) {
          page = *entry;
        } else {
          page = p.free_pages[start + pages[b] + (col - held)];
          if (at == 0) *entry = page;
        }
        if (page >= 0) slot = (int64_t)page * p.page.d + at;
      }
      p.slots[row] = slot;
      p.positions[row] = pos;
    }
    __syncthreads();   // the next chunk overwrites the sums
  }
  for (int64_t row = min(row_base, (int64_t)p.rows) + (int64_t)blockIdx.x * kThreads + tid; row < p.rows;
       row += (int64_t)gridDim.x * kThreads) {
    p.slots[row] = -1;
    p.positions[row] = 0;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.cu[p.batch] = (int)min(row_base, (int64_t)p.rows);
    p.free_end[0] = (int)(start + taken);
  }
}

}  // namespace fa

namespace fa {

template <int kThreads, int kPer>
hipError_t launch_slots(const SlotsParams& p, hipStream_t st) {
  const int64_t wgs = ((int64_t)p.rows + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(wgs < 1 ? 1 : wgs > 1024 ? 1024 : wgs);
  hipLaunchKernelGGL((kvcache_slots_kernel<kThreads, kPer>), dim3(grid), dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

}  // namespace fa

hipError_t fa_launch_kvcache_slots(const fa::SlotsParams& p, hipStream_t st) {
  // More threads cost a launch of few requests time, more chunks one of many.
  // 64 / 200 / 4096 requests of 64 / 27000 / 134000 tokens, MI355X: 4.6 / 6.1 /
  // 33.8 us with 256 threads of two requests, 5.3 / 6.7 / 16.7 us with 512 of four.
  return p.batch <= 512 ? fa::launch_slots<256, 2>(p, st) : fa::launch_slots<512, 4>(p, st);
}
