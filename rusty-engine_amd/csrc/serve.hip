// Steps of batched serving around the paged cache: the plan of a step (pages, block tables, slot maps), rotary
// positions of a ragged batch's rows, log probabilities of logit rows.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "serve.hpp"
#include "wave.hpp"

namespace rehip {

// ---- plan ----------------------------------------------------------------------------------------
// Request b holds len[b] tokens in ceil(len / page) pages and brings new_len[b] more: need_b = ceil((len + new) / page)
// - ceil(len / page) pages. new_len -1 ends it: its pages are pushed on the free stack first, request after request.
// Needed pages are then popped in request order from the top. With S_b the sum of the needs up to b, b is accepted if
// it needs none or S_b <= the pages there are, so every thread decides for its own requests after one prefix sum.
// The accepted and refused alike keep their rows (the caller laid them out from new_len); a refused one gets count 0
// and keeps its length.
//
// Bound by latency (a few KB): loads, two scans, the stack, the table, then the rows, one after the other in one workgroup:
// 64 requests 7.8 us a call, 5.5 in the kernel; 1024 requests and 19000 rows 12.6 us, 8.5 and 4.2 for the rows' launch (of
// more rows than two per thread; in the plan's own workgroup they would take a trip to memory per 1024 of them).

// exclusive prefix sums over the workgroup of three numbers per thread; totals in tot
template <int THREADS>
__device__ __forceinline__ void scan3(int (&v)[3], int (&tot)[3]) {
  __shared__ int part[3][THREADS / 64];
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
    for (int i = 0; i < THREADS / 64; ++i) {
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
  const int b = last_at_most(start, a.requests, t), n = count[b], i = t - start[b];
  const bool live = i < n;
  const int pos = len[b] - n + i;
  a.seq[t] = live ? b : -1;
  a.pos[t] = live ? pos : -1;
  const int pid = live ? a.table[(size_t)b * a.table_ld + pos / a.page] : -1;
  a.slot[t] = pid >= 0 && pid < a.n_pages ? pid * a.page + pos % a.page : -1;
}

// One workgroup. Pages go back and are taken one per thread, whatever request they are of (a thread that walked its own
// request's pages waited for memory page after page: 23 -> 8 us for 64 requests, 4 of which end).
template <int THREADS, int PER>             // PER requests per thread
__global__ __launch_bounds__(THREADS) void kv_plan_kernel(PlanArgs a, int rows_here) {
  constexpr int kMost = THREADS * PER;
  __shared__ int start[kMost], count[kMost], len[kMost];
  __shared__ int back_at[kMost], need_at[kMost], held_of[kMost];
  const int tid = threadIdx.x;
  const int b0 = tid * PER;
  int nw[PER], ln[PER], need[PER], back[PER], held[PER];
  bool fits[PER];
  int sum[3] = {0, 0, 0}, tot[3];
  const int room = a.table_ld * a.page;
  const int free0 = min(max(*a.n_free, 0), a.n_pages);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
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
  scan3<THREADS>(sum, tot);
  const int have = free0 + min(tot[0], a.n_pages - free0);
  int refused = 0, taken = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = b0 + i;
    const int n = max(nw[i], 0);
    const bool ok = nw[i] >= 0 && fits[i] && (need[i] == 0 || sum[1] + need[i] <= have);
    if (b < a.requests) {
      back_at[b] = sum[0];
      need_at[b] = sum[1];
      held_of[b] = held[i];
      a.start[b] = start[b] = sum[2];
      a.count[b] = count[b] = ok ? n : 0;
      a.len_out[b] = len[b] = nw[i] < 0 ? 0 : ok ? ln[i] + n : ln[i];
      refused += n > 0 && !ok;
    }
    taken += ok ? need[i] : 0;
    sum[0] += back[i];
    sum[1] += need[i];
    sum[2] += n;
  }
  int fin[3] = {taken, refused, 0}, all[3];
  scan3<THREADS>(fin, all);                         // (a barrier: the lists are there)
  if (tid == 0) {
    *a.n_free_out = have - all[0];
    a.status[0] = all[1];
    a.status[1] = tot[2];
  }
  // pushes: ended requests' pages behind the free ones; the stack then holds `have`
  for (int k = tid; k < have - free0; k += THREADS) {
    const int b = last_at_most(back_at, a.requests, k);
    a.free_pages[free0 + k] = a.table[(size_t)b * a.table_ld + (k - back_at[b])];
  }
  __threadfence_block();
  __syncthreads();
  // needed page k is the k-th from the top, if its request's last one is there too
  for (int k = tid; k < min(tot[1], have); k += THREADS) {
    const int b = last_at_most(need_at, a.requests, k);
    const int upto = b + 1 < a.requests ? need_at[b + 1] : tot[1];
    if (upto <= have) a.table[(size_t)b * a.table_ld + held_of[b] + (k - need_at[b])] = a.free_pages[have - 1 - k];
  }
  if (!rows_here) return;
  __threadfence_block();
  __syncthreads();
  for (int t = tid; t < a.cap; t += THREADS) plan_row(a, start, count, len, t);
}

__global__ __launch_bounds__(256) void kv_plan_rows_kernel(PlanArgs a) {
  __shared__ int start[kPlanMaxRequests];
  for (int b = threadIdx.x; b < a.requests; b += 256) start[b] = a.start[b];
  __syncthreads();
  for (int t = blockIdx.x * 256 + threadIdx.x; t < a.cap; t += gridDim.x * 256)
    plan_row(a, start, a.count, a.len_out, t);
}

template <int THREADS, int PER>
static void launch_plan(const PlanArgs& a, bool rows_here, hipStream_t s) {
  hipLaunchKernelGGL((kv_plan_kernel<THREADS, PER>), dim3(1), dim3(THREADS), 0, s, a, rows_here ? 1 : 0);
}

hipError_t launch_kv_plan(const PlanArgs& a, hipStream_t s) {
  const bool small = a.requests <= 256;
  // two rows per thread at most; more go to a launch of their own over many workgroups
  const bool rows_here = a.cap <= (small ? 512 : 2048);
  if (small) launch_plan<256, 1>(a, rows_here, s);
  else if (a.requests <= 1024) launch_plan<1024, 1>(a, rows_here, s);
  else launch_plan<1024, kPlanMaxRequests / 1024>(a, rows_here, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || rows_here) return e;
  hipLaunchKernelGGL(kv_plan_rows_kernel, dim3((unsigned)std::min((a.cap + 255) / 256, 1024)), dim3(256), 0, s, a);
  return hipGetLastError();
}

// ---- rotary positions ----------------------------------------------------------------------------
// Pair i of each head of row r turns by pos[r] * freqs[i] radians and is scaled by mscale. The angle is taken in turns
// and reduced to half a turn in 64 bits: at position 131071 an angle in 32 bits is off by up to 4e-3. A row's angles are
// taken once for all its heads. Bound by HBM: 8192 rows of 36 heads of 128, 302 MB, 57.6 us, 5.2 TB/s (as a large copy);
// 8 rows by the launch, 7 us a call and 2.9 in the kernel.
__device__ __forceinline__ void turn_cs(int pos, double freq, float mscale, float& c, float& s) {
  const double t = (double)pos * (freq * 0.15915494309189533577);
  const float f = (float)(2.0 * (t - rint(t)));
  c = cospif(f) * mscale;
  s = sinpif(f) * mscale;
}

// One workgroup per row; rows at negative positions are left as they are. VEC: four dimensions at a time (strides and
// addresses multiples of 16 bytes, whole fours of pairs in the half layout and of dimensions in the interleaved one).
template <bool VEC>
__global__ __launch_bounds__(256) void rope_rows_kernel(RopeArgs a) {
  __shared__ __attribute__((aligned(16))) float2 cs[128];
  const int r = blockIdx.x, half = a.rot >> 1;
  const int pos = a.pos[r];
  if (pos < 0) return;
  for (int i = threadIdx.x; i < half; i += 256) turn_cs(pos, a.freqs[i], a.mscale, cs[i].x, cs[i].y);
  __syncthreads();
  const float* x = a.x + (size_t)r * a.ldx;
  float* o = a.out + (size_t)r * a.ldo;
  const int rest = a.hd - a.rot;
  if constexpr (VEC) {
    const int pairs = half >> 2, fours = a.rot >> 2;
    if (a.interleaved) {
#pragma unroll 4
      for (int e = threadIdx.x; e < a.heads * fours; e += 256) {
        const int h = e / fours, i = e - h * fours, d = h * a.hd + 4 * i;
        const float4 v = *reinterpret_cast<const float4*>(x + d);
        const float4 t = *reinterpret_cast<const float4*>(&cs[2 * i]);
        *reinterpret_cast<float4*>(o + d) =
            make_float4(v.x * t.x - v.y * t.y, v.y * t.x + v.x * t.y, v.z * t.z - v.w * t.w, v.w * t.z + v.z * t.w);
      }
    } else {
#pragma unroll 4
      for (int e = threadIdx.x; e < a.heads * pairs; e += 256) {
        const int h = e / pairs, i = e - h * pairs, d = h * a.hd + 4 * i;
        const float4 u = *reinterpret_cast<const float4*>(x + d), v = *reinterpret_cast<const float4*>(x + d + half);
        const float4 s = *reinterpret_cast<const float4*>(&cs[4 * i]), t = *reinterpret_cast<const float4*>(&cs[4 * i + 2]);
        *reinterpret_cast<float4*>(o + d) =
            make_float4(u.x * s.x - v.x * s.y, u.y * s.z - v.y * s.w, u.z * t.x - v.z * t.y, u.w * t.z - v.w * t.w);
        *reinterpret_cast<float4*>(o + d + half) =
            make_float4(v.x * s.x + u.x * s.y, v.y * s.z + u.y * s.w, v.z * t.x + u.z * t.y, v.w * t.z + u.w * t.w);
      }
    }
    if (x == o || rest == 0) return;
    const int more = rest >> 2;
#pragma unroll 4
    for (int e = threadIdx.x; e < a.heads * more; e += 256) {
      const int h = e / more, d = h * a.hd + a.rot + 4 * (e - h * more);
      *reinterpret_cast<float4*>(o + d) = *reinterpret_cast<const float4*>(x + d);
    }
  } else {
    for (int e = threadIdx.x; e < a.heads * half; e += 256) {
      const int h = e / half, i = e % half;
      const int d0 = h * a.hd + (a.interleaved ? 2 * i : i), d1 = d0 + (a.interleaved ? 1 : half);
      const float x0 = x[d0], x1 = x[d1];
      o[d0] = x0 * cs[i].x - x1 * cs[i].y;
      o[d1] = x1 * cs[i].x + x0 * cs[i].y;
    }
    if (x == o || rest == 0) return;
    for (int e = threadIdx.x; e < a.heads * rest; e += 256) {
      const int d = e / rest * a.hd + a.rot + e % rest;
      o[d] = x[d];
    }
  }
}

hipError_t launch_rope_rows(const RopeArgs& a, hipStream_t s) {
  const bool fours = a.hd % 4 == 0 && a.rot % (a.interleaved ? 4 : 8) == 0 && a.ldx % 4 == 0 && a.ldo % 4 == 0 &&
                     ((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.out & 15) == 0;
  hipLaunchKernelGGL(fours ? rope_rows_kernel<true> : rope_rows_kernel<false>, dim3((unsigned)a.rows), dim3(256), 0, s, a);
  return hipGetLastError();
}

// ---- log probabilities ---------------------------------------------------------------------------
// With m a row's largest logit, d = x - m, Z = sum e^d and T = sum d e^d: log p = d_target - ln Z, entropy = ln Z - T / Z.
// One pass over the logits: each lane keeps (m, Z, T) of what it has seen and moves them when its maximum rises,
//   Z' = c Z, T' = c (T + (m - m') Z), c = e^(m - m');
// a logit of -inf has e^d = 0 and adds nothing, and so do terms whose c is 0 (d may be -inf there). A lane sums a batch
// and adds that to its sums with their rounding errors kept (2370 equal terms of a row of 151936, added one after the other,
// could round the same way every time: ln Z was off by 3.7e-5).
//
// The k largest (ties to the lower index) in the same pass. A candidate is one 64-bit key, larger for the better one:
// the value's bits made order-preserving, then the index inverted. A wave keeps its candidates in LDS, and a border that
// its k best so far are at or above. A batch whose largest value is below the border costs one comparison per lane; from
// the others the keys above the border are appended. When the list is full its k best stay, ranked by counting. A first
// border comes from the first batch: the k-th largest of the 64 lanes' maxima has at least k values at or above it.
// Values in random order push about k ln(batches) keys behind the first batch; a rising row pushes all.
//
// Bound by HBM: 961 rows of 151936, 20 best, 584 MB in 99 us, 5.9 TB/s (without candidates 93, 6.3 TB/s); one row 11 us,
// 7.2 and 4.4 in its two launches: latency.
constexpr int kTopCap = 256;             // candidates of a wave
constexpr int kLogBatch = 16;            // logits of a lane at a time
constexpr int kLogWaves = 4;
constexpr int kLogPart = 64 * kLogBatch * kLogWaves;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

typedef unsigned long long key_t64;

// a NaN ranks as -inf, -0 as 0
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x != x ? -INFINITY : x + 0.0f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ key_t64 key_of(float x, int i) { return (key_t64)ordered(x) << 32 | (unsigned)~i; }
__device__ __forceinline__ int index_of(key_t64 k) { return (int)~(unsigned)k; }
__device__ __forceinline__ float value_of(key_t64 k) {
  const unsigned u = (unsigned)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
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
  wave_butterfly([&](auto off) {
    constexpr int X = decltype(off)::value;
    s = join(s, Stats{lane_xor<X>(s.m), lane_xor<X>(s.z), lane_xor<X>(s.t)});
  });
  return s;
}

// A list of n keys is followed by kPad zeros, so that it is read kPad at a time.
constexpr int kPad = 8;

// how many of list[0 .. n) are above each of mine
template <int Q>
__device__ __forceinline__ void rank_in(const key_t64* list, int n, const key_t64 (&mine)[Q], int (&rank)[Q]) {
#pragma unroll
  for (int q = 0; q < Q; ++q) rank[q] = 0;
  for (int e = 0; e < n; e += kPad) {
    key_t64 y[kPad];
#pragma unroll
    for (int j = 0; j < kPad; ++j) y[j] = list[e + j];
#pragma unroll
    for (int j = 0; j < kPad; ++j)
#pragma unroll
      for (int q = 0; q < Q; ++q) rank[q] += y[j] > mine[q];
  }
}

// A wave's candidates. The members are the same in every lane.
struct Candidates {
  key_t64* list;                         // kTopCap of them, and the zeros
  int n, k;
  key_t64 border;                        // keys at or below it cannot be among the k best
  float least;                           // .. nor values below this

  template <int Q>
  __device__ __forceinline__ void keep_best_of() {
    const int lane = threadIdx.x & 63;
    key_t64 mine[Q];
    int rank[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) mine[q] = lane + 64 * q < n ? list[lane + 64 * q] : 0;
    if (lane < kPad) list[n + lane] = 0;
    wave_sync();
    rank_in(list, n, mine, rank);
    wave_sync();
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (lane + 64 * q < n && rank[q] < k) list[rank[q]] = mine[q];
    wave_sync();
  }
  __device__ __forceinline__ void keep_best() {
    if (n <= 64) keep_best_of<1>();
    else if (n <= 128) keep_best_of<2>();
    else keep_best_of<kTopCap / 64>();
    n = min(n, k);
    if (n == k) {
      border = list[k - 1];
      least = value_of(border);
    }
  }
  __device__ __forceinline__ void push(bool yes, key_t64 key) {
    const unsigned long long who = __ballot(yes);
    if (who == 0) return;
    if (yes) list[n + __popcll(who & ((1ull << (threadIdx.x & 63)) - 1))] = key;
    wave_sync();
    n += __popcll(who);
    if (n > max(64, 2 * k)) keep_best();
  }
  // a border from the lanes' maxima, before anything is pushed: the least of those with fewer than k above them
  __device__ __forceinline__ void first_border(float mx) {
    const unsigned o = ordered(mx);
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < 64; ++j) rank += (unsigned)__builtin_amdgcn_readlane((int)o, j) > o;
    unsigned low = rank < k ? o : 0xffffffffu;
    wave_butterfly([&](auto off) { low = min(low, lane_xor_u32<decltype(off)::value>(low)); });
    low = (unsigned)__builtin_amdgcn_readfirstlane((int)low);
    border = ((key_t64)low << 32) - 1;   // (equal values pass; ordered() is never 0)
    least = value_of((key_t64)low << 32);
  }
  // x[q] at index at(q) (below 0: no such place), mx their largest
  template <int N, class At>
  __device__ __forceinline__ void batch(const float (&x)[N], float mx, At at, bool first) {
    if (first) first_border(mx);
    if (__ballot(mx >= least) == 0) return;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const bool maybe = !(x[q] < least);  // (NaN counts as -inf, and so may while the border is)
      if (__ballot(maybe) == 0) continue;
      const key_t64 key = key_of(x[q], at(q));
      push(maybe && at(q) >= 0 && key > border, key);
    }
    if (first) keep_best();
  }
};

// the row's target and its logit, on their way from the start
struct Target {
  int id;
  float x;
};
__device__ __forceinline__ Target target_of(const LogprobArgs& a, int r) {
  const int id = a.logprob ? a.targets[r] : -1;
  return {id, a.x[(size_t)r * a.ld + min(max(id, 0), a.vocab - 1)]};
}

// what a finished row gives: the target's log probability, the entropy, the k best of the candidates
// (by `threads` threads, of which this is `tid`)
__device__ __forceinline__ void finish_row(const LogprobArgs& a, int r, const Target& t, const Stats& s,
                                           const key_t64* list, int n, int tid, int threads) {
  const float lz = logf(s.z);
  if (tid == 0) {
    if (a.logprob) a.logprob[r] = t.id >= 0 && t.id < a.vocab ? (t.x - s.m) - lz : 0.0f;
    if (a.entropy) a.entropy[r] = lz - s.t / s.z;
  }
  for (int e = tid; e < n; e += threads) {
    const key_t64 mine[1] = {list[e]};
    int rank[1];
    rank_in(list, n, mine, rank);
    if (rank[0] < a.k) {
      a.ids[(size_t)r * a.k + rank[0]] = index_of(mine[0]);
      a.top[(size_t)r * a.k + rank[0]] = (value_of(mine[0]) - s.m) - lz;   // (of a NaN, held as -inf: NaN by ln Z)
    }
  }
}

// One workgroup per (row, part of it); a part's (m, Z, T) and candidates go to the workspace unless it is the whole row.
// SHORT: a wave per row, four rows per workgroup, and no barrier.
template <bool TOP, bool SHORT>
__global__ __launch_bounds__(64 * kLogWaves) void logprobs_kernel(LogprobArgs a, int parts) {
  __shared__ __attribute__((aligned(16))) key_t64 lists[TOP ? kLogWaves * (kTopCap + kPad) : 1];
  __shared__ Stats ws[kLogWaves];
  __shared__ int wn[kLogWaves];
  constexpr int kStep = SHORT ? 1 : kLogWaves;             // batches between two of a wave
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = SHORT ? blockIdx.x * kLogWaves + w : blockIdx.x / parts, part = SHORT ? 0 : blockIdx.x % parts;
  if (r >= a.rows) return;
  const float* x = a.x + (size_t)r * a.ld;
  Target target{};
  if (parts == 1) target = target_of(a, r);
  // parts of whole batches, the last one shorter
  const int batches = (a.vocab + 64 * kLogBatch - 1) / (64 * kLogBatch);
  const int b0 = (int)((long long)batches * part / parts), b1 = (int)((long long)batches * (part + 1) / parts);
  Candidates c{lists + (TOP ? w * (kTopCap + kPad) : 0), 0, a.k, 0, -INFINITY};
  Stats s{-INFINITY, 0.0f, 0.0f};
  float lost_z = 0.0f, lost_t = 0.0f;      // what the sums' roundings left out, s.z + lost_z the better sum
  auto add = [](float& sum, float& lost, float v) {
    const float was = sum;
    sum += v;
    lost += v - (sum - was);
  };
  bool first = true;
  auto take = [&](const float (&v)[kLogBatch], int base) {
    float mx = -INFINITY;
#pragma unroll
    for (int q = 0; q < kLogBatch; ++q) mx = fmaxf(mx, v[q]);
    const float mn = fmaxf(s.m, mx), ref = mn == -INFINITY ? 0.0f : mn;
    if (mn > s.m) {
      const float d = s.m - mn, f = exp_of(d);
      s.t = f == 0.0f ? 0.0f : f * (s.t + d * s.z);
      lost_t = f == 0.0f ? 0.0f : f * (lost_t + d * lost_z);
      s.z *= f;
      lost_z *= f;
      s.m = mn;
    }
    float z = 0.0f, t = 0.0f;
#pragma unroll
    for (int q = 0; q < kLogBatch; ++q) {
      const float d = v[q] - ref, e = exp_of(d);
      z += e;
      t = __builtin_fmaf(e, fmaxf(d, -3e38f), t);
    }
    add(s.z, lost_z, z);
    add(s.t, lost_t, t);
    if constexpr (TOP) {
      c.batch(v, mx, [&](int q) {
        const int at = base + 256 * (q >> 2) + (q & 3);
        return at < a.vocab ? at : -1;
      }, first);
      first = false;
    }
  };
  auto load = [&](float (&v)[kLogBatch], int bt) {
#pragma unroll
    for (int q = 0; q < kLogBatch / 4; ++q)
      *reinterpret_cast<f32x4u*>(&v[4 * q]) = __builtin_nontemporal_load(
          reinterpret_cast<const f32x4u*>(x + bt * 64 * kLogBatch + 4 * lane + 256 * q));
  };
  // whole batches, the next one loading meanwhile, then the row's last part of one
  const int whole = min(b1, a.vocab / (64 * kLogBatch));
  int bt = SHORT ? 0 : b0 + w;
  if (bt < whole) {
    float v[kLogBatch], nx[kLogBatch];
    load(v, bt);
    for (; bt < whole; bt += kStep) {
      load(nx, bt + kStep < whole ? bt + kStep : bt);
      take(v, bt * 64 * kLogBatch + 4 * lane);
#pragma unroll
      for (int q = 0; q < kLogBatch; ++q) v[q] = nx[q];
    }
  }
  if (bt < b1) {
    const int base = bt * 64 * kLogBatch + 4 * lane;
    float v[kLogBatch];
#pragma unroll
    for (int q = 0; q < kLogBatch; ++q) {
      const int at = base + 256 * (q >> 2) + (q & 3);
      const float y = x[min(at, a.vocab - 1)];           // (loaded whatever: a load under a condition is waited for)
      v[q] = at < a.vocab ? y : -INFINITY;
    }
    take(v, base);
  }
  s.z += lost_z;
  s.t += lost_t;
  s = wave_join(s);
  if constexpr (TOP) {
    // (k at most 64: a workgroup's lists then have a thread per key. Longer lists of a small k would be ranked against each
    // other below: 300 rows of 20000, 5 best 17.7 us instead of 16.6)
    if (c.n > min(a.k + 8, 64)) c.keep_best();
  }
  if constexpr (SHORT) {
    if (TOP && lane < kPad) c.list[c.n + lane] = 0;
    wave_sync();
    finish_row(a, r, target, s, c.list, c.n, lane, 64);
    return;
  }
  if (lane == 0) { ws[w] = s; wn[w] = TOP ? c.n : 0; }
  __syncthreads();
  const Stats all = join(join(ws[0], ws[1]), join(ws[2], ws[3]));
  int n = 0;
  if constexpr (TOP) {                   // the waves' lists one behind the other
    key_t64 y = 0;
    bool have = false;
    for (int k = 0; k < kLogWaves; ++k) {
      const int e = (int)threadIdx.x - n;
      if (e >= 0 && e < wn[k]) { y = lists[k * (kTopCap + kPad) + e]; have = true; }
      n += wn[k];
    }
    __syncthreads();
    if (have) lists[threadIdx.x] = y;
    if (threadIdx.x < kPad) lists[n + threadIdx.x] = 0;
    __syncthreads();
  }
  if (parts == 1) {
    finish_row(a, r, target, all, lists, n, threadIdx.x, 64 * kLogWaves);
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
    if ((int)threadIdx.x < n) {
      const key_t64 mine[1] = {lists[threadIdx.x]};
      int rank[1];
      rank_in(lists, n, mine, rank);
      if (rank[0] < a.k) reinterpret_cast<key_t64*>(o + 4)[rank[0]] = mine[0];
    }
  }
}

// A row's parts joined: their sums in part order, their candidates. With q = ceil(k / parts), the least of the parts'
// q-th best has k keys at or above it; those above or at it are gathered (in any order) and ranked by counting.
constexpr int kLogJoin = 256;
constexpr int kLogMaxParts = 64;

__global__ __launch_bounds__(kLogJoin) void logprobs_join_kernel(LogprobArgs a, int parts) {
  constexpr int kMost = kLogMaxParts * kLogprobsMaxTop;
  __shared__ __attribute__((aligned(16))) key_t64 every[kMost], list[kMost + kPad];
  __shared__ Stats all;
  __shared__ key_t64 low;
  __shared__ int count;
  const int r = blockIdx.x, tid = threadIdx.x, stride = 4 + 2 * a.k;
  const Target target = target_of(a, r);
  const float* o = a.work + (size_t)r * parts * stride;
  // the parts' keys, 0 where a part has fewer
  for (int e = tid; e < parts * a.k; e += kLogJoin) {
    const float* p = o + e / a.k * stride;
    const key_t64 key = reinterpret_cast<const key_t64*>(p + 4)[e % a.k];
    every[e] = e % a.k < __float_as_int(p[3]) ? key : 0;
  }
  const float* p = o + min(tid, parts - 1) * stride;
  const Stats mine = tid < parts ? Stats{p[0], p[1], p[2]} : Stats{-INFINITY, 0.0f, 0.0f};
  if (tid == 0) count = 0;
  __syncthreads();
  if (tid < 64) {                          // (a lane per part)
    const Stats s = wave_join(mine);
    // a part shorter than q keys: all keys count
    key_t64 least = a.k > 0 && tid < parts ? every[tid * a.k + (a.k + parts - 1) / parts - 1] : ~0ull;
    wave_butterfly([&](auto off) {
      constexpr int X = decltype(off)::value;
      least = min(least, (key_t64)lane_xor_u32<X>((unsigned)(least >> 32)) << 32 | lane_xor_u32<X>((unsigned)least));
    });
    if (tid == 0) {
      all = s;
      low = max(least, (key_t64)1);
    }
  }
  __syncthreads();
  for (int e = tid; e < parts * a.k; e += kLogJoin)
    if (every[e] >= low) list[atomicAdd(&count, 1)] = every[e];
  __syncthreads();
  const int n = count;
  if (tid < kPad) list[n + tid] = 0;
  __syncthreads();
  finish_row(a, r, target, all, list, n, tid, kLogJoin);
}

// About three workgroups for each CU; a part is at least one batch of every wave (64 rows of 151936, top 20: 29.7 / 25.3
// / 26.6 us at 256 / 768 / 1024 workgroups; 256 rows: 53.1 / 42.3 / 42.6).
// The join's launch takes 3 us, a batch 0.2 and more with candidates: parts if they take more than that off (us whole / in
// parts: one row of 32000, none 8.0 / 11.3, 20 best 21 / 12; 12289, 2 best 8.5 / 11.3; 12963, 17 best 14 / 11.6; 157 rows of
// 29551, none 8.4 / 11.0, 4 best 18.2 / 15.9); two of them only of long rows (300 of 20000 16.5 / 18.1, 380 of 151936 50 / 46).
static int logprob_parts(int rows, int vocab, int k) {
  const int batches = (vocab + kLogPart - 1) / kLogPart;           // of a wave of a whole row
  const int parts = std::min({batches, kLogMaxParts, 768 / std::max(rows, 1)});
  return (parts > 2 || (parts == 2 && batches >= 16)) && (long)batches * (parts - 1) * (1 + k) > 20L * parts ? parts : 1;
}

size_t logprobs_work_floats(int rows, int vocab, int k) {
  const int parts = logprob_parts(rows, vocab, k);
  return parts > 1 ? (size_t)rows * parts * (4 + 2 * k) : 0;
}

hipError_t launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  const int parts = logprob_parts(a.rows, a.vocab, a.k);
  // a wave per row where one batch is the row, or where rows alone fill the GPU's waves (us of a wave / a workgroup per
  // row, top 5 or 20: 4000 x 1000 11.5 / 25, 2000 x 32000 54 / 63, 8000 x 32000 161 / 182; but 1000 x 16000 25.4 / 20.2;
  // long rows just above the border, top 20: 1536 x 50000 67.4 / 67.6, x 151936 156 / 158, 2048 x 151936 192 / 197)
  if (a.vocab <= 64 * kLogBatch || a.rows >= 1536) {
    auto* k = a.k > 0 ? logprobs_kernel<true, true> : logprobs_kernel<false, true>;
    hipLaunchKernelGGL(k, dim3((unsigned)((a.rows + kLogWaves - 1) / kLogWaves)), dim3(64 * kLogWaves), 0, s, a, 1);
    return hipGetLastError();
  }
  auto* k = a.k > 0 ? logprobs_kernel<true, false> : logprobs_kernel<false, false>;
  hipLaunchKernelGGL(k, dim3((unsigned)(a.rows * parts)), dim3(64 * kLogWaves), 0, s, a, parts);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || parts == 1) return e;
  hipLaunchKernelGGL(logprobs_join_kernel, dim3((unsigned)a.rows), dim3(kLogJoin), 0, s, a, parts);
  return hipGetLastError();
}

}  // namespace rehip
