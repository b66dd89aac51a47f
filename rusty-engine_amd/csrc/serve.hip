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
// With m a row's largest logit, d = x - m, Z = sum e^d and T = sum d e^d: log p = d_target - ln Z, entropy = ln Z - T / Z.
// One pass over the logits: each lane keeps (m, Z, T) of what it has seen and moves them when its maximum rises,
//   Z' = c Z, T' = c (T + (m - m') Z), c = e^(m - m');
// a logit of -inf has e^d = 0 and adds nothing, and so do terms whose c is 0 (d may be -inf there).
//
// The k largest (ties to the lower index) in the same pass: a wave keeps candidates in LDS and the k-th of them, once it
// has k, as a border (value, index). A batch whose largest value is below the border costs one comparison per lane; the
// others append what is before the border. When the list is full its k best stay, ranked by counting. A first border
// comes from the first batch: the k-th largest of the 64 lanes' maxima has at least k values at or above it.
// Values in random order push about k ln(batches) candidates behind the first batch; a rising row pushes all.
constexpr int kTopCap = 256;             // candidates of a wave
constexpr int kLogBatch = 16;            // logits of a lane at a time
constexpr int kLogWaves = 4;
constexpr int kLogPart = 64 * kLogBatch * kLogWaves;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ bool before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }
__device__ __forceinline__ float ranked(float x) { return x != x ? -INFINITY : x; }
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.4426950408889634f); }

struct Stats { float m, z, t; };

__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
  const float m = fmaxf(a.m, b.m);
  // (nothing above -inf yet: Z and T are 0, or NaN where a NaN was seen)
  const float da = a.m == -INFINITY ? 0.0f : a.m - m, db = b.m == -INFINITY ? 0.0f : b.m - m;
  const float fa = exp_of(da), fb = exp_of(db);
  return {m, a.z * fa + b.z * fb,
          (fa == 0.0f ? 0.0f : fa * (a.t + da * a.z)) + (fb == 0.0f ? 0.0f : fb * (b.t + db * b.z))};
}
__device__ __forceinline__ Stats wave_join(Stats s) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    s = join(s, Stats{__shfl_xor(s.m, off, 64), __shfl_xor(s.z, off, 64), __shfl_xor(s.t, off, 64)});
  return s;
}

// A wave's candidates. All members but the arrays are the same in every lane.
struct Candidates {
  float* v;
  int* i;
  int n, k;
  float bv;                              // the border: what is not before it cannot be among the k best
  int bi;

  __device__ __forceinline__ void rank_and_keep() {
    const int lane = threadIdx.x & 63;
    float x[kTopCap / 64];
    int at[kTopCap / 64], rank[kTopCap / 64];
#pragma unroll
    for (int q = 0; q < kTopCap / 64; ++q) {
      const int e = lane + 64 * q;
      x[q] = e < n ? v[e] : -INFINITY;
      at[q] = e < n ? i[e] : 0x7fffffff;
      rank[q] = 0;
    }
    for (int e = 0; e < n; ++e) {
      const float y = v[e];
      const int j = i[e];
#pragma unroll
      for (int q = 0; q < kTopCap / 64; ++q) rank[q] += before(y, j, x[q], at[q]);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < kTopCap / 64; ++q)
      if (lane + 64 * q < n && rank[q] < k) {
        v[rank[q]] = x[q];
        i[rank[q]] = at[q];
      }
    __builtin_amdgcn_wave_barrier();
    n = min(n, k);
    if (n == k) {
      bv = v[k - 1];
      bi = i[k - 1];
    }
  }
  __device__ __forceinline__ void push(bool yes, float x, int at) {
    const unsigned long long who = __ballot(yes);
    if (who == 0) return;
    if (yes) {
      const int e = n + __popcll(who & ((1ull << (threadIdx.x & 63)) - 1));
      v[e] = x;
      i[e] = at;
    }
    __builtin_amdgcn_wave_barrier();
    n += __popcll(who);
    if (n > kTopCap - 64) rank_and_keep();
  }
  // a border from the lanes' maxima, before anything is pushed
  __device__ __forceinline__ void first_border(float mx) {
    int rank = 0;
    for (int j = 0; j < 64; ++j) {
      const float y = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mx), j));
      rank += y > mx || (y == mx && j < (int)(threadIdx.x & 63));
    }
    const unsigned long long who = __ballot(rank == k - 1);
    bv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mx), __ffsll(who) - 1));
    bi = 0x7fffffff;
  }
  // x[q] at index at(q), mx their largest
  template <int N, class At>
  __device__ __forceinline__ void batch(const float (&x)[N], float mx, At at, bool first) {
    if (first) first_border(mx);
    if (__ballot(mx >= bv) == 0) return;
#pragma unroll
    for (int q = 0; q < N; ++q) push(at(q) < 0x7fffffff && before(x[q], at(q), bv, bi), x[q], at(q));
    if (first) rank_and_keep();
  }
};

// what a finished row gives: the target's log probability, the entropy, the best ones'
__device__ __forceinline__ void finish_row(const LogprobArgs& a, int r, const Stats& s, const float* v, const int* i,
                                           int n) {
  const float lz = logf(s.z);
  if (threadIdx.x == 0) {
    if (a.logprob) {
      const int g = a.targets[r];
      a.logprob[r] = g >= 0 && g < a.vocab ? (a.x[(size_t)r * a.ld + g] - s.m) - lz : 0.0f;
    }
    if (a.entropy) a.entropy[r] = lz - s.t / s.z;
  }
  // the k best of the n candidates
  for (int e = threadIdx.x; e < n; e += blockDim.x) {
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += before(v[j], i[j], v[e], i[e]);
    if (rank < a.k) {
      a.ids[(size_t)r * a.k + rank] = i[e];
      // (the value itself, a NaN too: candidates hold it as -inf)
      a.top[(size_t)r * a.k + rank] = (a.x[(size_t)r * a.ld + i[e]] - s.m) - lz;
    }
  }
}

// One workgroup per (row, part of it); a part's (m, Z, T) and candidates go to the workspace unless it is the whole row.
template <bool TOP>
__global__ __launch_bounds__(64 * kLogWaves) void logprobs_kernel(LogprobArgs a, int parts) {
  __shared__ float cv[TOP ? kLogWaves * kTopCap : 1];
  __shared__ int ci[TOP ? kLogWaves * kTopCap : 1];
  __shared__ Stats ws[kLogWaves];
  __shared__ int wn[kLogWaves];
  const int r = blockIdx.x / parts, part = blockIdx.x % parts;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float* x = a.x + (size_t)r * a.ld;
  // parts of whole batches, the last one shorter
  const int batches = (a.vocab + 64 * kLogBatch - 1) / (64 * kLogBatch);
  const int b0 = (int)((long long)batches * part / parts), b1 = (int)((long long)batches * (part + 1) / parts);
  Candidates c{cv + (TOP ? w * kTopCap : 0), ci + (TOP ? w * kTopCap : 0), 0, a.k, -INFINITY, 0x7fffffff};
  Stats s{-INFINITY, 0.0f, 0.0f};
  bool first = true;
  for (int bt = b0 + w; bt < b1; bt += kLogWaves) {
    const int base = bt * 64 * kLogBatch + 4 * lane;
    float v[kLogBatch];
    const bool whole = (bt + 1) * 64 * kLogBatch <= a.vocab;
    if (whole) {
#pragma unroll
      for (int q = 0; q < kLogBatch / 4; ++q)
        *reinterpret_cast<f32x4u*>(&v[4 * q]) =
            __builtin_nontemporal_load(reinterpret_cast<const f32x4u*>(x + base + 256 * q));
    } else {
#pragma unroll
      for (int q = 0; q < kLogBatch; ++q) {
        const int at = base + 256 * (q >> 2) + (q & 3);
        v[q] = at < a.vocab ? x[at] : -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int q = 0; q < kLogBatch; ++q) mx = fmaxf(mx, v[q]);
    const float mn = fmaxf(s.m, mx), ref = mn == -INFINITY ? 0.0f : mn;
    if (mn > s.m) {
      const float d = s.m - mn, f = exp_of(d);
      s.t = f == 0.0f ? 0.0f : f * (s.t + d * s.z);
      s.z *= f;
      s.m = mn;
    }
#pragma unroll
    for (int q = 0; q < kLogBatch; ++q) {
      const float d = v[q] - ref, e = exp_of(d);
      s.z += e;
      s.t = __builtin_fmaf(e, fmaxf(d, -3e38f), s.t);
    }
    if constexpr (TOP) {
#pragma unroll
      for (int q = 0; q < kLogBatch; ++q) v[q] = ranked(v[q]);
      c.batch(v, mx, [&](int q) {
        const int at = base + 256 * (q >> 2) + (q & 3);
        return at < a.vocab ? at : 0x7fffffff;             // (not in the row: never a candidate)
      }, first);
      first = false;
    }
  }
  s = wave_join(s);
  if constexpr (TOP) {
    if (c.n > 0) c.rank_and_keep();
  }
  if (lane == 0) { ws[w] = s; wn[w] = TOP ? c.n : 0; }
  __syncthreads();
  const Stats all = join(join(ws[0], ws[1]), join(ws[2], ws[3]));
  int n = 0;
  if constexpr (TOP) {                   // the waves' lists one behind the other
    float y = 0.0f;
    int at = 0, to = -1;
    for (int k = 0; k < kLogWaves; ++k) {
      const int e = (int)threadIdx.x - n;
      if (e >= 0 && e < wn[k]) { y = cv[k * kTopCap + e]; at = ci[k * kTopCap + e]; to = threadIdx.x; }
      n += wn[k];
    }
    __syncthreads();
    if (to >= 0) { cv[to] = y; ci[to] = at; }
    __syncthreads();
  }
  if (parts == 1) {
    finish_row(a, r, all, cv, ci, n);
    return;
  }
  float* o = a.work + (size_t)blockIdx.x * (4 + 2 * a.k);
  if (threadIdx.x == 0) {
    o[0] = all.m;
    o[1] = all.z;
    o[2] = all.t;
    o[3] = __int_as_float(min(n, a.k));
  }
  if constexpr (TOP) {
    const int e = threadIdx.x;
    if (e < n) {
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += before(cv[j], ci[j], cv[e], ci[e]);
      if (rank < a.k) {
        o[4 + 2 * rank] = cv[e];
        o[5 + 2 * rank] = __int_as_float(ci[e]);
      }
    }
  }
}

// A row's parts joined by one wave: their sums in part order, their candidates as one more list.
__global__ __launch_bounds__(64) void logprobs_join_kernel(LogprobArgs a, int parts) {
  __shared__ float cv[kTopCap];
  __shared__ int ci[kTopCap];
  const int r = blockIdx.x, lane = threadIdx.x, stride = 4 + 2 * a.k;
  const float* o = a.work + (size_t)r * parts * stride;
  Stats s{-INFINITY, 0.0f, 0.0f};
  for (int p = lane; p < parts; p += 64) s = join(s, Stats{o[p * stride], o[p * stride + 1], o[p * stride + 2]});
  s = wave_join(s);
  Candidates c{cv, ci, 0, a.k, -INFINITY, 0x7fffffff};
  if (a.k > 0) {
    // round q: the parts' (q + 1)-th best. Lists fall, so a round without a push ends it
    for (int q = 0; q < a.k; ++q) {
      const int was = c.n;
      bool any = false;
      for (int p0 = 0; p0 < parts; p0 += 64) {
        const int p = p0 + lane;
        const bool in = p < parts && q < __float_as_int(o[p * stride + 3]);
        const float y = in ? o[p * stride + 4 + 2 * q] : -INFINITY;
        const int at = in ? __float_as_int(o[p * stride + 5 + 2 * q]) : 0x7fffffff;
        const bool yes = in && before(y, at, c.bv, c.bi);
        any |= __ballot(yes) != 0;
        c.push(yes, y, at);
      }
      if (!any) break;
      if (c.n >= a.k && c.n > was) c.rank_and_keep();
    }
    if (c.n > 0) c.rank_and_keep();
  }
  __syncthreads();
  finish_row(a, r, s, cv, ci, c.n);
}

// Workgroups for one round over the CUs at four each; a part is at least one batch of every wave.
static int logprob_parts(int rows, int vocab) {
  const int most = (vocab + kLogPart - 1) / kLogPart;
  return std::max(1, std::min(most, 1024 / std::max(rows, 1)));
}

size_t logprobs_work_floats(int rows, int vocab, int k) {
  const int parts = logprob_parts(rows, vocab);
  return parts > 1 ? (size_t)rows * parts * (4 + 2 * k) : 0;
}

hipError_t launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  const int parts = logprob_parts(a.rows, a.vocab);
  auto* k = a.k > 0 ? logprobs_kernel<true> : logprobs_kernel<false>;
  hipLaunchKernelGGL(k, dim3((unsigned)(a.rows * parts)), dim3(64 * kLogWaves), 0, s, a, parts);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || parts == 1) return e;
  hipLaunchKernelGGL(logprobs_join_kernel, dim3((unsigned)a.rows), dim3(64), 0, s, a, parts);
  return hipGetLastError();
}

}  // namespace rehip
