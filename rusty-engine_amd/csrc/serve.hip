// Steps of batched serving around the paged cache: the plan of a step (pages, block tables, slot maps), rotary
// positions of a ragged batch's rows, log probabilities of logit rows.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "serve.hpp"

namespace rehip {

// ---- plan ----------------------------------------------------------------------------------------
// Request b holds len[b] tokens in ceil(len / page) pages and brings new_len[b] more: need_b = ceil((len + new) / page)
// - ceil(len / page) pages. new_len -1 ends it: its pages are pushed on the free stack first, request after request.
// Needed pages are then popped in request order from the top. With S_b the sum of the needs up to b, b is accepted if
// it needs none or S_b <= the pages there are, so every thread decides for its own requests after one prefix sum.
// The accepted and refused alike keep their rows (the caller laid them out from new_len); a refused one gets count 0
// and keeps its length.
constexpr int kPlanThreads = 1024;
constexpr int kPlanPer = kPlanMaxRequests / kPlanThreads;   // requests per thread

// exclusive prefix sums over the workgroup of three numbers per thread; totals in tot
__device__ __forceinline__ void scan3(int (&v)[3], int (&tot)[3]) {
  __shared__ int part[3][kPlanThreads / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int inc[3];
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    inc[c] = v[c];
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(inc[c], off, 64);
      if (lane >= off) inc[c] += y;
    }
    if (lane == 63) part[c][w] = inc[c];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 64; ++i) {
      const int p = part[c][i];
      before += i < w ? p : 0;
      all += p;
    }
    v[c] = before + inc[c] - v[c];
    tot[c] = all;
  }
  __syncthreads();
}

// seq, pos and slot of row t from the finished plan; rows that no request of the step owns get -1
__device__ __forceinline__ void plan_row(const PlanArgs& a, const int* start, const int* count, const int* len, int t) {
  int lo = 0, hi = a.requests;             // the first request that starts behind t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  const int b = lo - 1;
  const int i = t - start[b];
  const bool live = i < count[b];
  const int pos = len[b] - count[b] + i;
  a.seq[t] = live ? b : -1;
  a.pos[t] = live ? pos : -1;
  const int pid = live ? a.table[(size_t)b * a.table_ld + pos / a.page] : -1;
  a.slot[t] = pid >= 0 && pid < a.n_pages ? pid * a.page + pos % a.page : -1;
}

__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanArgs a, int rows_here) {
  __shared__ int start[kPlanMaxRequests], count[kPlanMaxRequests], len[kPlanMaxRequests];
  const int tid = threadIdx.x;
  const int b0 = tid * kPlanPer;
  int nw[kPlanPer], ln[kPlanPer], need[kPlanPer], back[kPlanPer], held[kPlanPer];
  bool fits[kPlanPer];
  int sum[3] = {0, 0, 0}, tot[3];
  const int room = a.table_ld * a.page;
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const int b = b0 + i;
    const bool in = b < a.requests;
    const int asked = in ? a.new_len[b] : 0;
    nw[i] = min(asked, kPlanMaxNew);
    ln[i] = in ? a.len[b] : 0;
    const bool sound = ln[i] >= 0 && ln[i] <= room;
    fits[i] = sound && nw[i] == asked && ln[i] + max(nw[i], 0) <= room;
    held[i] = sound ? (ln[i] + a.page - 1) / a.page : 0;
    back[i] = nw[i] < 0 ? held[i] : 0;
    need[i] = fits[i] && nw[i] > 0 ? (ln[i] + nw[i] + a.page - 1) / a.page - held[i] : 0;
    sum[0] += back[i];
    sum[1] += need[i];
    sum[2] += max(nw[i], 0);
  }
  const int free0 = min(max(*a.n_free, 0), a.n_pages);
  scan3(sum, tot);
  // pushes: ended requests' pages behind the free ones
  int at = free0 + sum[0];
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i)
    for (int j = 0; j < back[i]; ++j, ++at)
      if (at < a.n_pages) a.free_pages[at] = a.table[(size_t)(b0 + i) * a.table_ld + j];
  const int have = min(free0 + tot[0], a.n_pages);
  int row = sum[2], s = sum[1], refused = 0, taken = 0;
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const int b = b0 + i;
    const int n = max(nw[i], 0);
    s += need[i];
    const bool ok = nw[i] >= 0 && fits[i] && (need[i] == 0 || s <= have);
    if (b < a.requests) {
      start[b] = row;
      count[b] = ok ? n : 0;
      len[b] = nw[i] < 0 ? 0 : ok ? ln[i] + n : ln[i];
      a.start[b] = start[b];
      a.count[b] = count[b];
      a.len_out[b] = len[b];
      refused += n > 0 && !ok;
    }
    taken += ok ? need[i] : 0;
    row += n;
  }
  __threadfence_block();
  __syncthreads();                         // the pushed pages are there for every thread
  s = sum[1];
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const int b = b0 + i;
    s += need[i];
    if (b < a.requests && need[i] > 0 && s <= have) {
      const int base = have - 1 - (s - need[i]);
      for (int j = 0; j < need[i]; ++j) a.table[(size_t)b * a.table_ld + held[i] + j] = a.free_pages[base - j];
    }
  }
  int fin[3] = {taken, refused, 0}, all[3];
  scan3(fin, all);
  if (tid == 0) {
    *a.n_free_out = have - all[0];
    a.status[0] = all[1];
    a.status[1] = tot[2];
  }
  if (!rows_here) return;
  __threadfence_block();
  __syncthreads();
  for (int t = tid; t < a.cap; t += kPlanThreads) plan_row(a, start, count, len, t);
}

__global__ __launch_bounds__(256) void kv_plan_rows_kernel(PlanArgs a) {
  __shared__ int start[kPlanMaxRequests];
  for (int b = threadIdx.x; b < a.requests; b += 256) start[b] = a.start[b];
  __syncthreads();
  for (int t = blockIdx.x * 256 + threadIdx.x; t < a.cap; t += gridDim.x * 256)
    plan_row(a, start, a.count, a.len_out, t);
}

hipError_t launch_kv_plan(const PlanArgs& a, hipStream_t s) {
  const bool rows_here = a.cap <= kPlanThreads;
  hipLaunchKernelGGL(kv_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, rows_here ? 1 : 0);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || rows_here) return e;
  hipLaunchKernelGGL(kv_plan_rows_kernel, dim3((unsigned)std::min((a.cap + 255) / 256, 1024)), dim3(256), 0, s, a);
  return hipGetLastError();
}

// ---- rotary positions ----------------------------------------------------------------------------
// Pair i of each head of row r turns by pos[r] * freqs[i] radians and is scaled by mscale. The angle is taken in turns
// and reduced to half a turn in 64 bits: at position 131071 an angle in 32 bits is off by up to 4e-3.
__device__ __forceinline__ void turn_cs(int pos, double freq, float mscale, float& c, float& s) {
  const double t = (double)pos * (freq * 0.15915494309189533577);
  const float f = (float)(2.0 * (t - rint(t)));
  c = cospif(f) * mscale;
  s = sinpif(f) * mscale;
}

// one workgroup per row; rows at negative positions are left as they are
__global__ __launch_bounds__(256) void rope_rows_kernel(RopeArgs a) {
  __shared__ float2 cs[128];
  const int r = blockIdx.x, half = a.rot >> 1;
  const int pos = a.pos[r];
  if (pos < 0) return;
  for (int i = threadIdx.x; i < half; i += 256) turn_cs(pos, a.freqs[i], a.mscale, cs[i].x, cs[i].y);
  __syncthreads();
  const float* x = a.x + (size_t)r * a.ldx;
  float* o = a.out + (size_t)r * a.ldo;
  for (int e = threadIdx.x; e < a.heads * half; e += 256) {
    const int h = e / half, i = e % half;
    const int d0 = h * a.hd + (a.interleaved ? 2 * i : i), d1 = d0 + (a.interleaved ? 1 : half);
    const float x0 = x[d0], x1 = x[d1];
    o[d0] = x0 * cs[i].x - x1 * cs[i].y;
    o[d1] = x1 * cs[i].x + x0 * cs[i].y;
  }
  if (x == o) return;
  const int rest = a.hd - a.rot;
  for (int e = threadIdx.x; e < a.heads * rest; e += 256) {
    const int d = e / rest * a.hd + a.rot + e % rest;
    o[d] = x[d];
  }
}

hipError_t launch_rope_rows(const RopeArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(rope_rows_kernel, dim3((unsigned)a.rows), dim3(256), 0, s, a);
  return hipGetLastError();
}

// ---- log probabilities ---------------------------------------------------------------------------
// With m the row's largest logit, d = x - m and Z = sum e^d: log p = d_target - ln Z, entropy = ln Z - sum d e^d / Z.
// A logit of -inf has probability 0 and adds nothing to either sum.
__device__ __forceinline__ bool before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

__global__ __launch_bounds__(256) void logprobs_kernel(LogprobArgs a) {
  __shared__ float red[3][4];
  __shared__ float bv[4];
  __shared__ int bi[4];
  const int r = blockIdx.x, tid = threadIdx.x, w = tid >> 6;
  const float* x = a.x + (size_t)r * a.ld;
  float m = -INFINITY, bad = 0.0f;
  for (int i = tid; i < a.vocab; i += 256) {
    m = fmaxf(m, x[i]);
    if (x[i] != x[i]) bad = NAN;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    m = fmaxf(m, __shfl_xor(m, off, 64));
    bad += __shfl_xor(bad, off, 64);
  }
  if ((tid & 63) == 0) { red[0][w] = m; red[1][w] = bad; }
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  m += (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);     // NaN anywhere: a NaN row
  __syncthreads();
  float z = 0.0f, t = 0.0f;
  for (int i = tid; i < a.vocab; i += 256) {
    const float d = x[i] - m, e = expf(d);
    z += e;
    if (e != 0.0f) t += e * d;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    z += __shfl_xor(z, off, 64);
    t += __shfl_xor(t, off, 64);
  }
  if ((tid & 63) == 0) { red[0][w] = z; red[1][w] = t; }
  __syncthreads();
  z = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
  t = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const float lz = logf(z);
  if (tid == 0) {
    if (a.logprob) {
      const int g = a.targets[r];
      a.logprob[r] = g >= 0 && g < a.vocab ? (x[g] - m) - lz : 0.0f;
    }
    if (a.entropy) a.entropy[r] = lz - t / z;
  }
  float lv = INFINITY;
  int li = -1;
  for (int k = 0; k < a.k; ++k) {          // the best behind (lv, li)
    float v = -INFINITY;
    int at = a.vocab;
    for (int i = tid; i < a.vocab; i += 256) {
      const float y = x[i] != x[i] ? -INFINITY : x[i];
      if (before(lv, li, y, i) && (at == a.vocab || before(y, i, v, at))) { v = y; at = i; }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float ov = __shfl_xor(v, off, 64);
      const int oi = __shfl_xor(at, off, 64);
      if (oi < a.vocab && (at == a.vocab || before(ov, oi, v, at))) { v = ov; at = oi; }
    }
    __syncthreads();
    if ((tid & 63) == 0) { bv[w] = v; bi[w] = at; }
    __syncthreads();
    lv = bv[0];
    li = bi[0];
    for (int i = 1; i < 4; ++i)
      if (bi[i] < a.vocab && (li == a.vocab || before(bv[i], bi[i], lv, li))) { lv = bv[i]; li = bi[i]; }
    if (tid == 0) {
      a.ids[(size_t)r * a.k + k] = li;
      a.top[(size_t)r * a.k + k] = (x[li] - m) - lz;
    }
  }
}

size_t logprobs_work_floats(int, int, int) { return 0; }

hipError_t launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(logprobs_kernel, dim3((unsigned)a.rows), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace rehip
