// Pages that change hands outside a step's plan: requests cut to fewer tokens in fresh pages (eviction), and tokens taken
// back from their ends (rejected drafts).
#include <hip/hip_runtime.h>

#include "serve.hpp"
#include "wave.hpp"

namespace rehip {

// The table entries of requests b, columns from first[b] (null: 0) on, at[b + 1] - at[b] of them, `total` in all, that hold a page
// go to out[base ..] in that order, `room` at most. Returns how many. All threads of the workgroup call it; a thread has four
// entries that follow one another, so that 4 THREADS of them cost one trip to memory and one scan.
template <int THREADS>
__device__ __forceinline__ int push_pages(const int* at, const int* first, int requests, int total, const int* table,
                                          int table_ld, int n_pages, int* out, int base, int room) {
  int done = 0;
  for (int k0 = 0; k0 < total; k0 += 4 * THREADS) {
    int pid[4], mine = 0, before;
    const int k = k0 + 4 * (int)threadIdx.x;
    int b = k < total ? last_at_most(at, requests, k) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i > 0 && k + i < total && b + 1 < requests && at[b + 1] <= k + i) b = last_at_most(at, requests, k + i);
      pid[i] = k + i < total ? table[(size_t)b * table_ld + (first ? first[b] : 0) + (k + i - at[b])] : -1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (pid[i] < 0 || pid[i] >= n_pages) pid[i] = -1;
      mine += pid[i] >= 0;
    }
    const int all = scan_block<THREADS / 64>(mine, before);
    before += done;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (pid[i] >= 0 && before < room) out[base + before] = pid[i];
      before += pid[i] >= 0;
    }
    done += all;
  }
  return min(done, room);
}

// ---- eviction's plan -----------------------------------------------------------------------------
// A request of len > limit tokens is cut to `keep`, in fresh = ceil(keep / page) pages from the top of the stack, so that its
// old pages are read while the new ones are written; every cut request takes as many, so the i-th of them (from 0) has them
// if (i + 1) fresh <= the free pages, and takes free[n - 1 - (i fresh + j)], j < fresh. Its old pages are pushed afterwards,
// request after request. One workgroup: bound by the latency of its loads, scans and stores, one after the other: 4.1 us for one
// request, 8.5 for 32 of 128 table columns (25 with entries and pushes request by request).
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void kv_evict_plan_kernel(EvictPlanArgs a, int copy_table, int copy_free) {
  constexpr int kMost = THREADS * PER;
  __shared__ int at[kMost], row_of[kMost], rank_of[kMost];         // row_of[i]: the i-th request that is cut; its i, or -1
  const int tid = threadIdx.x, b0 = tid * PER;
  const int free0 = min(max(*a.n_free, 0), a.n_pages);
  const int room = a.table_ld * a.page, fresh = (a.keep + a.page - 1) / a.page;
  int len[PER], over = 0, before;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    len[i] = b0 + i < a.requests ? a.len[b0 + i] : 0;
    over += len[i] > a.limit && len[i] <= room;
  }
  const int wanted = scan_block<THREADS / 64>(over, before);
  const int cuts = min(wanted, free0 / fresh), left = free0 - cuts * fresh;
  int held[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = b0 + i;
    const bool is = len[i] > a.limit && len[i] <= room, ok = is && before < cuts;
    held[i] = ok ? (len[i] + a.page - 1) / a.page : 0;
    if (b < a.requests) {
      rank_of[b] = ok ? before : -1;
      if (ok) row_of[before] = b;
      a.len_out[b] = ok ? a.keep : len[i];
      a.from_len[b] = ok ? len[i] : 0;
      if (a.dropped) {
        if (ok) a.dropped[b] += len[i] - a.keep;
        else if (len[i] == 0) a.dropped[b] = 0;
      }
    }
    before += is;
    sum += held[i];
  }
  int upto;
  const int total = scan_block<THREADS / 64>(sum, upto);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (b0 + i >= a.requests) break;
    at[b0 + i] = upto;
    upto += held[i];
  }
  __syncthreads();
  // Rows: the cut ones' old entries kept and new ones written, the others copied. An entry is read and written by one thread,
  // so that the table may be written in place.
  const int rows = copy_table ? a.requests : cuts, entries = rows * a.table_ld;
  for (int k0 = tid; k0 < entries; k0 += 4 * THREADS) {
    int e[4], rank[4], j[4], old[4], got[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = min(k0 + i * THREADS, entries - 1), r = k / a.table_ld, b = copy_table ? r : row_of[r];
      j[i] = k - r * a.table_ld;
      e[i] = b * a.table_ld + j[i];
      rank[i] = rank_of[b];
      old[i] = a.table[e[i]];
      got[i] = rank[i] >= 0 && j[i] < fresh ? a.free_pages[free0 - 1 - (rank[i] * fresh + j[i])] : -1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (k0 + i * THREADS >= entries) break;
      if (rank[i] >= 0 && a.from_table != a.table) a.from_table[e[i]] = old[i];
      a.table_out[e[i]] = rank[i] >= 0 ? got[i] : old[i];
    }
  }
  if (copy_free) {
    for (int k0 = tid; k0 < left; k0 += 4 * THREADS) {
      int x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = a.free_pages[min(k0 + i * THREADS, left - 1)];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k0 + i * THREADS < left) a.free_out[k0 + i * THREADS] = x[i];
    }
  }
  __threadfence_block();
  __syncthreads();                       // (the stack's top has been read, the old rows are there)
  const int pushed = push_pages<THREADS>(at, nullptr, a.requests, total, a.from_table, a.table_ld, a.n_pages, a.free_out, left,
                                         a.n_pages - left);
  if (tid == 0) {
    *a.n_free_out = left + pushed;
    a.status[0] = wanted - cuts;
    a.status[1] = cuts;
  }
}

// n ints (or *n_at, up to `most`) of src to dst
__global__ __launch_bounds__(256) void copy_ints_kernel(const int* src, int* dst, const int* n_at, int n, int most) {
  if (n_at) n = min(max(*n_at, 0), most);
  for (int k = blockIdx.x * 256 + threadIdx.x; k < n; k += gridDim.x * 256) dst[k] = src[k];
}

template <int THREADS, int PER>
static void launch_evict_plan(const EvictPlanArgs& a, bool copy_table, bool copy_free, hipStream_t s) {
  hipLaunchKernelGGL((kv_evict_plan_kernel<THREADS, PER>), dim3(1), dim3(THREADS), 0, s, a, copy_table ? 1 : 0,
                     copy_free ? 1 : 0);
}

hipError_t launch_kv_evict_plan(const EvictPlanArgs& a, hipStream_t s) {
  // Tables and stacks of more numbers than 32 for each of the plan's threads are copied by many workgroups before (us of a call with
  // those launches / without: 64 x 1024 entries 11.8 / 22.9, 256 x 1024 18 / 79; but 32 x 128 10.6 / 7.2, 64 x 256 21.5 / 17.5)
  constexpr int kCopiedHere = 32768;
  const int entries = a.requests * a.table_ld;
  bool copy_table = a.table_out != a.table, copy_free = a.free_out != a.free_pages;
  if (copy_table && entries > kCopiedHere) {
    hipLaunchKernelGGL(copy_ints_kernel, dim3(512), dim3(256), 0, s, a.table, a.table_out, nullptr, entries, entries);
    copy_table = false;
  }
  if (copy_free && a.n_pages > kCopiedHere) {
    hipLaunchKernelGGL(copy_ints_kernel, dim3(512), dim3(256), 0, s, a.free_pages, a.free_out, a.n_free, 0, a.n_pages);
    copy_free = false;
  }
  // (four waves for a small table, whose barriers are shorter: us of a call with 256 / 1024 threads, one request of 66 entries 4.8 /
  // 5.3, 8 of 128 5.0 / 5.9; but 32 of 128 11.2 / 7.1, 64 of 256 36 / 17.5)
  if (a.requests <= 256 && entries <= 1024) launch_evict_plan<256, 1>(a, copy_table, copy_free, s);
  else if (a.requests <= 1024) launch_evict_plan<1024, 1>(a, copy_table, copy_free, s);
  else launch_evict_plan<1024, kPlanMaxRequests / 1024>(a, copy_table, copy_free, s);
  return hipGetLastError();
}

// ---- rewind --------------------------------------------------------------------------------------
// A request of len tokens gives back min(back, len) of them; the pages ceil(left / page) .. ceil(len / page) - 1 hold none of
// the rest and go to the stack, request after request. One workgroup, as the plan: the lengths, then the table's entries, then
// a scan. Where no request gives back more than kFew pages (drafts are shorter than that) a thread reads those of its own
// requests itself; else entries are handed out one by one, whatever request they are of. 64 requests 2.1 us, 4096 6.2 (9.9 all
// handed out).
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void kv_rewind_kernel(RewindArgs a) {
  constexpr int kMost = THREADS * PER, kFew = 2;
  __shared__ int at[kMost], stay[kMost];
  const int tid = threadIdx.x, b0 = tid * PER;
  const int free0 = min(max(*a.n_free, 0), a.n_pages), room = a.table_ld * a.page;
  int gone[PER], from[PER], sum = 0, most = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = min(b0 + i, a.requests - 1);
    gone[i] = a.len[b];
    from[i] = a.back[b];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = b0 + i, len = gone[i];
    const bool sound = len >= 0 && len <= room && b < a.requests;
    const int left = sound ? len - min(max(from[i], 0), len) : len;
    from[i] = sound ? (left + a.page - 1) / a.page : 0;
    gone[i] = sound ? (len + a.page - 1) / a.page - from[i] : 0;
    if (b < a.requests) a.len_out[b] = left;
    sum += gone[i];
    most = max(most, gone[i]);
  }
  int before, pushed;
  if (!__syncthreads_or(most > kFew)) {
    int pid[PER][kFew], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < kFew; ++j) {
        pid[i][j] = -1;
        if (j < gone[i]) pid[i][j] = a.table[(size_t)(b0 + i) * a.table_ld + from[i] + j];
      }
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < kFew; ++j) {
        if (pid[i][j] >= a.n_pages) pid[i][j] = -1;
        mine += pid[i][j] >= 0;
      }
    pushed = min(scan_block<THREADS / 64>(mine, before), a.n_pages - free0);
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < kFew; ++j) {
        if (pid[i][j] >= 0 && before < a.n_pages - free0) a.free_pages[free0 + before] = pid[i][j];
        before += pid[i][j] >= 0;
      }
  } else {
    const int total = scan_block<THREADS / 64>(sum, before);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (b0 + i >= a.requests) break;
      at[b0 + i] = before;
      stay[b0 + i] = from[i];
      before += gone[i];
    }
    __syncthreads();
    pushed = push_pages<THREADS>(at, stay, a.requests, total, a.table, a.table_ld, a.n_pages, a.free_pages, free0,
                                 a.n_pages - free0);
  }
  if (tid == 0) *a.n_free_out = free0 + pushed;
}

template <int THREADS, int PER>
static void launch_rewind(const RewindArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((kv_rewind_kernel<THREADS, PER>), dim3(1), dim3(THREADS), 0, s, a);
}

hipError_t launch_kv_rewind(const RewindArgs& a, hipStream_t s) {
  if (a.requests <= 256) launch_rewind<256, 1>(a, s);
  else if (a.requests <= 1024) launch_rewind<1024, 1>(a, s);
  else launch_rewind<1024, kPlanMaxRequests / 1024>(a, s);
  return hipGetLastError();
}

// ---- positions -----------------------------------------------------------------------------------
// A request that has been cut stands further on than its cache is long.
__global__ __launch_bounds__(256) void kv_positions_kernel(const int* seq, const int* pos, int rows, const int* dropped,
                                                           int requests, int* out) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= rows) return;
  const int b = seq[r], p = pos[r];
  out[r] = p >= 0 && b >= 0 && b < requests ? p + dropped[b] : -1;
}

hipError_t launch_kv_positions(const int* seq, const int* pos, int rows, const int* dropped, int requests, int* out,
                               hipStream_t s) {
  hipLaunchKernelGGL(kv_positions_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, s, seq, pos, rows, dropped,
                     requests, out);
  return hipGetLastError();
}

}  // namespace rehip
