// Pages that change hands outside a step's plan: requests cut to fewer tokens in fresh pages (eviction), and tokens taken
// back from their ends (rejected drafts).
#include <hip/hip_runtime.h>

#include "serve.hpp"
#include "wave.hpp"

namespace rehip {

// The table entries of requests b, columns from first[b] (null: 0) on, at[b + 1] - at[b] of them, `total` in all, that hold a page
// go to out[base ..] in that order, `room` at most. Returns how many. All threads of the workgroup call it.
template <int THREADS>
__device__ __forceinline__ int push_pages(const int* at, const int* first, int requests, int total, const int* table,
                                          int table_ld, int n_pages, int* out, int base, int room) {
  int done = 0;
  for (int k0 = 0; k0 < total; k0 += THREADS) {
    const int k = k0 + (int)threadIdx.x;
    int pid = -1;
    if (k < total) {
      const int b = last_at_most(at, requests, k);
      pid = table[(size_t)b * table_ld + (first ? first[b] : 0) + (k - at[b])];
    }
    const bool holds = pid >= 0 && pid < n_pages;
    int before;
    const int all = scan_block<THREADS / 64>(holds ? 1 : 0, before);
    if (holds && done + before < room) out[base + done + before] = pid;
    done += all;
  }
  return min(done, room);
}

// ---- eviction's plan -----------------------------------------------------------------------------
// A request of len > limit tokens is cut to `keep`, in fresh = ceil(keep / page) pages from the top of the stack, so that its
// old pages are read while the new ones are written; every cut request takes as many, so the i-th of them (from 0) has them
// if (i + 1) fresh <= the free pages, and takes free[n - 1 - (i fresh + j)], j < fresh. Its old pages are pushed afterwards,
// request after request. One workgroup: bound by the latency of its loads, scans and stores, one after the other.
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void kv_evict_plan_kernel(EvictPlanArgs a, int copy_table, int copy_free) {
  constexpr int kMost = THREADS * PER;
  __shared__ int at[kMost], row_of[kMost];                  // row_of[i]: the i-th request that is cut
  __shared__ bool cut[kMost];
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
  const int cuts = min(wanted, free0 / fresh);
  int held = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = b0 + i;
    const bool is = len[i] > a.limit && len[i] <= room, ok = is && before < cuts;
    if (b < a.requests) {
      cut[b] = ok;
      if (ok) row_of[before] = b;
      a.len_out[b] = ok ? a.keep : len[i];
      a.from_len[b] = ok ? len[i] : 0;
      if (a.dropped) {
        if (ok) a.dropped[b] += len[i] - a.keep;
        else if (len[i] == 0) a.dropped[b] = 0;
      }
    }
    before += is;
    held += ok ? (len[i] + a.page - 1) / a.page : 0;
  }
  int sum;
  const int total = scan_block<THREADS / 64>(held, sum);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (b0 + i >= a.requests) break;
    at[b0 + i] = sum;
    sum += cut[b0 + i] ? (len[i] + a.page - 1) / a.page : 0;
  }
  __syncthreads();
  // the old rows, where the table is written over
  if (a.from_table != a.table) {
    for (int k = tid; k < total; k += THREADS) {
      const int b = last_at_most(at, a.requests, k);
      const size_t e = (size_t)b * a.table_ld + (k - at[b]);
      a.from_table[e] = a.table[e];
    }
  }
  if (copy_table) {
    for (int k = tid; k < a.requests * a.table_ld; k += THREADS)
      if (!cut[k / a.table_ld]) a.table_out[k] = a.table[k];
  }
  if (copy_free) {
    for (int k = tid; k < free0 - cuts * fresh; k += THREADS) a.free_out[k] = a.free_pages[k];
  }
  __threadfence_block();
  __syncthreads();
  // (a request's columns side by side: the stack is read and the rows written in order)
  for (int k = tid; k < cuts * a.table_ld; k += THREADS) {
    const int i = k / a.table_ld, j = k - i * a.table_ld;
    a.table_out[(size_t)row_of[i] * a.table_ld + j] = j < fresh ? a.free_pages[free0 - 1 - (i * fresh + j)] : -1;
  }
  __threadfence_block();
  __syncthreads();
  const int left = free0 - cuts * fresh;
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
  // Tables and stacks of more than a few numbers for each of the plan's threads are copied by many workgroups before
  constexpr int kCopiedHere = 16384;
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
  if (a.requests <= 256) launch_evict_plan<256, 1>(a, copy_table, copy_free, s);
  else if (a.requests <= 1024) launch_evict_plan<1024, 1>(a, copy_table, copy_free, s);
  else launch_evict_plan<1024, kPlanMaxRequests / 1024>(a, copy_table, copy_free, s);
  return hipGetLastError();
}

// ---- rewind --------------------------------------------------------------------------------------
// A request of len tokens gives back min(back, len) of them; the pages ceil(left / page) .. ceil(len / page) - 1 hold none of
// the rest and go to the stack, request after request. One workgroup, as the plan.
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void kv_rewind_kernel(RewindArgs a) {
  constexpr int kMost = THREADS * PER;
  __shared__ int at[kMost], stay[kMost];
  const int tid = threadIdx.x, b0 = tid * PER;
  const int free0 = min(max(*a.n_free, 0), a.n_pages), room = a.table_ld * a.page;
  int gone[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = b0 + i;
    const bool in = b < a.requests;
    const int len = in ? a.len[b] : 0, back = in ? a.back[b] : 0;
    const bool sound = len >= 0 && len <= room;
    const int left = sound ? len - min(max(back, 0), len) : len;
    gone[i] = sound ? (len + a.page - 1) / a.page - (left + a.page - 1) / a.page : 0;
    if (in) {
      a.len_out[b] = left;
      stay[b] = sound ? (left + a.page - 1) / a.page : 0;
    }
    sum += gone[i];
  }
  int before;
  const int total = scan_block<THREADS / 64>(sum, before);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (b0 + i >= a.requests) break;
    at[b0 + i] = before;
    before += gone[i];
  }
  __syncthreads();
  const int pushed = push_pages<THREADS>(at, stay, a.requests, total, a.table, a.table_ld, a.n_pages, a.free_pages, free0,
                                         a.n_pages - free0);
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

}  // namespace rehip
