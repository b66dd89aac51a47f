// Drafted tokens against the target model's probabilities.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "serve.hpp"
#include "wave.hpp"

namespace rehip {

// Row i of a request's count rows gives the target's distribution p of the token behind row i, p = softmax(x / T); the token
// drafted there is tokens[row + 1], with probability q of its draft's distribution (1 without one), i < count - 1. It is
// accepted if u q < p (T <= 0: if it is the largest logit, ties to the lower id). The first that is not ends the drafts, and
// in its place comes a token drawn from max(0, p - q) / sum (without a distribution: from p without the draft; where that
// leaves nothing, from p); behind the last draft it comes from p. Drawn: the lowest t with sum over j <= t of w_j > r W.
//
// Which token r falls on depends on sums over the whole vocabulary to about 1 / vocab of a share each: with sums off by
// 2^-24 one row in a hundred of 151936 would draw a neighbour. So exponentials and sums are in 64 bits: 2^y by its
// Taylor series at the nearest integer, |f| <= 1/2, 13 terms, off by (ln 2 / 2)^13 / 13! = 2e-16.
//
// Three launches: maxima and sums of parts of all rows; every request's last row found from them, and the sums of its
// weights by parts of the vocabulary; the part where r falls, and the token in it.
constexpr int kVerWaves = 4;
constexpr int kVerBatch = 8;             // logits of a lane at a time
constexpr int kVerStep = 64 * kVerBatch * kVerWaves;
constexpr int kVerParts = 64;            // a lane each

struct RowPart {
  double z;                              // sum of 2^((x - m) c)
  float m;
  int best;                              // where the largest is first
  int bad, pad;                          // a NaN or +inf was seen
};
struct Decision {
  double z;
  float m;
  int accepted, row, state;              // the row that the next token comes from; state: below
  int best, pad;
};
constexpr int kNone = 0, kGreedy = 1, kTarget = 2, kRest = 3;  // no distribution; the largest; p; p without the draft

__device__ __forceinline__ double pow2_64(double y) {
  y = fmax(y, -1100.0);
  const double n = rint(y), f = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 479001600.0;
  p = fma(p, f, 1.0 / 39916800.0);
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return ldexp(p, (int)n);
}

__device__ __forceinline__ double lane_xor64(double v, int off) {
  const int lo = __shfl_xor(__double2loint(v), off, 64), hi = __shfl_xor(__double2hiint(v), off, 64);
  return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += lane_xor64(v, off);
  return v;
}

// powers of 2 for each unit of logit; greedy below 0
__device__ __forceinline__ double units_of(const VerifyArgs& a, int req) {
  const float t = a.temperature ? a.temperature[req] : 1.0f;
  return t > 0.0f ? 1.4426950408889634074 / (double)t : -1.0;
}
// 2^((x - m) c), 0 for a logit of -inf
__device__ __forceinline__ double weight(float x, float m, double c) {
  return x == -INFINITY ? 0.0 : pow2_64(((double)x - (double)m) * c);
}

__device__ __forceinline__ PagedBatch rows_of(const VerifyArgs& a) {
  return {a.start, a.count, a.count, nullptr, a.requests, a.rows, 1, 1, 1};
}

// One workgroup per (row, part).
__global__ __launch_bounds__(64 * kVerWaves) void verify_rows_kernel(VerifyArgs a, int parts) {
  __shared__ RowPart ws[kVerWaves];
  const int r = blockIdx.x / parts, part = blockIdx.x % parts;
  const RequestRows q = request_of_unit(r, rows_of(a), 1, 0);
  if (q.req < 0 || r >= q.row0 + q.count) return;
  const double c = units_of(a, q.req);
  const float* x = a.x + (size_t)r * a.ld;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int steps = (a.vocab + kVerStep - 1) / kVerStep;
  const int s0 = (int)((long long)steps * part / parts), s1 = (int)((long long)steps * (part + 1) / parts);
  RowPart mine{0.0, -INFINITY, 0x7fffffff, 0, 0};
  for (int s = s0; s < s1; ++s) {
    const int base = s * kVerStep + w * 64 * kVerBatch + lane;
    float v[kVerBatch], mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVerBatch; ++k) {
      const int at = base + 64 * k;
      const float y = x[min(at, a.vocab - 1)];
      v[k] = at < a.vocab ? y : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < kVerBatch; ++k) {
      mine.bad |= !(v[k] < INFINITY);
      mx = fmaxf(mx, v[k]);
    }
    if (mx > mine.m) {
      mine.z *= mine.m == -INFINITY ? 0.0 : weight(mine.m, mx, fabs(c));
      mine.m = mx;
#pragma unroll
      for (int k = kVerBatch - 1; k >= 0; --k)
        if (v[k] == mx) mine.best = base + 64 * k;
    }
    if (c >= 0.0 && mine.m > -INFINITY) {
#pragma unroll
      for (int k = 0; k < kVerBatch; ++k) mine.z += weight(v[k], mine.m, c);
    }
  }
  auto join = [&](const RowPart& x, const RowPart& y) {
    RowPart o{0.0, fmaxf(x.m, y.m), x.m > y.m ? x.best : y.m > x.m ? y.best : min(x.best, y.best), x.bad | y.bad, 0};
    if (x.m > -INFINITY) o.z += x.z * weight(x.m, o.m, fabs(c));
    if (y.m > -INFINITY) o.z += y.z * weight(y.m, o.m, fabs(c));
    return o;
  };
#pragma unroll
  for (int off = 1; off < 64; off <<= 1)
    mine = join(mine, RowPart{lane_xor64(mine.z, off), __shfl_xor(mine.m, off, 64), __shfl_xor(mine.best, off, 64),
                              __shfl_xor(mine.bad, off, 64), 0});
  if (lane == 0) ws[w] = mine;
  __syncthreads();
  if (threadIdx.x == 0)
    reinterpret_cast<RowPart*>(a.work)[blockIdx.x] = join(join(ws[0], ws[1]), join(ws[2], ws[3]));
}

// A row's parts joined, the same in every lane.
__device__ __forceinline__ RowPart joined_row(const VerifyArgs& a, int row, int parts, double c) {
  const int lane = threadIdx.x & 63;
  RowPart p = reinterpret_cast<const RowPart*>(a.work)[(size_t)row * parts + min(lane, parts - 1)];
  if (lane >= parts) p = {0.0, -INFINITY, 0x7fffffff, 0, 0};
  float m = wave_max(p.m);
  const double z = wave_sum64(p.m > -INFINITY ? p.z * weight(p.m, m, fabs(c)) : 0.0);
  int best = p.m == m ? p.best : 0x7fffffff, bad = p.bad;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    best = min(best, __shfl_xor(best, off, 64));
    bad |= __shfl_xor(bad, off, 64);
  }
  return {z, m, best, bad | (m == -INFINITY), 0};
}

// How many drafts of a request are accepted, and where its next token comes from. Every wave of the workgroup looks at a row of
// its own at a time.
template <int WAVES>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, const RequestRows& q, int parts) {
  __shared__ Decision found[WAVES];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const double c = units_of(a, q.req);
  Decision d{};
  for (int i0 = 0; i0 < q.count; i0 += WAVES) {
    const int i = i0 + w, row = q.row0 + min(i, q.count - 1);
    const RowPart p = joined_row(a, row, parts, c);
    bool accepted = false;
    if (i < q.count - 1 && !p.bad) {
      const int t = a.tokens[row + 1];
      if (c < 0.0) {
        accepted = t == p.best;
      } else if (t >= 0 && t < a.vocab) {
        const double share = a.probs ? (double)a.probs[(size_t)row * a.ldp + t] : 1.0;
        accepted = (double)a.accept_u[row] * share * p.z < weight(a.x[(size_t)row * a.ld + t], p.m, c);
      }
    }
    if ((threadIdx.x & 63) == 0)
      found[w] = {p.z, p.m, accepted ? -1 : i, row, p.bad ? kNone : c < 0.0 ? kGreedy : i < q.count - 1 ? kRest : kTarget, p.best, 0};
    __syncthreads();
    bool done = false;
#pragma unroll
    for (int k = WAVES - 1; k >= 0; --k)
      if (found[k].accepted >= 0 && i0 + k < q.count) {
        d = found[k];
        done = true;
      }
    __syncthreads();
    if (done) break;
  }
  return d;
}

// The weight of token t: p, less the draft's share of it
struct Weights {
  const float* x;
  const float* probs;                    // the draft's row, or null
  double c, z;
  float m;
  int drop;                              // a draft without a distribution: this token has no weight (-1: none)
  __device__ __forceinline__ double operator()(int t) const {
    const double e = weight(x[t], m, c);
    if (probs) return fmax(e / z - (double)probs[t], 0.0);
    return t == drop ? 0.0 : e;
  }
};
__device__ __forceinline__ Weights weights_of(const VerifyArgs& a, const Decision& d, double c, bool rest) {
  const int t = rest && !a.probs ? a.tokens[d.row + 1] : -1;
  return {a.x + (size_t)d.row * a.ld, rest && a.probs ? a.probs + (size_t)d.row * a.ldp : nullptr, c, d.z, d.m, t};
}

__device__ __forceinline__ Decision* decisions_at(const VerifyArgs& a, int parts) {
  return reinterpret_cast<Decision*>(reinterpret_cast<RowPart*>(a.work) + (size_t)a.rows * parts);
}

// One workgroup per (request, part of the vocabulary): the sum of its weights.
constexpr int kRestWaves = 4;
__global__ __launch_bounds__(64 * kRestWaves) void verify_rest_kernel(VerifyArgs a, int parts, int cuts) {
  __shared__ double sums[kRestWaves];
  const int req = blockIdx.x / cuts, cut = blockIdx.x % cuts, tid = threadIdx.x;
  const RequestRows q = request_rows(req, a.start[req], a.count[req], 0, a.rows);
  if (q.count <= 0) return;
  const Decision d = decide<kRestWaves>(a, q, parts);
  Decision* const at = decisions_at(a, parts);
  if (cut == 0 && tid == 0) at[req] = d;
  if (d.state != kTarget && d.state != kRest) return;
  const Weights of = weights_of(a, d, units_of(a, req), d.state == kRest);
  const int t0 = (int)((long long)a.vocab * cut / cuts), t1 = (int)((long long)a.vocab * (cut + 1) / cuts);
  double s = 0.0;
  for (int t = t0 + tid; t < t1; t += 64 * kRestWaves) s += of(t);
  s = wave_sum64(s);
  if ((tid & 63) == 0) sums[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) reinterpret_cast<double*>(at + a.requests)[(size_t)req * cuts + cut] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The lowest token of t0 .. t1 - 1 whose running sum, from `from` on, is above `target`; the last with any weight if rounding
// leaves none (-1: no weight at all). All threads call it.
constexpr int kDrawThreads = 512;
__device__ __forceinline__ int draw_from(const Weights& of, int t0, int t1, double from, double target) {
  __shared__ double part[kDrawThreads / 64];
  __shared__ int lowest[kDrawThreads / 64], highest[kDrawThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int per = (t1 - t0 + kDrawThreads - 1) / kDrawThreads, a0 = min(t0 + tid * per, t1), a1 = min(a0 + per, t1);
  double s = 0.0;
  int some = -1;
  for (int t = a0; t < a1; ++t) {
    const double v = of(t);
    s += v;
    if (v > 0.0) some = t;
  }
  double inc = s;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double y = __hiloint2double(__shfl_up(__double2hiint(inc), off, 64), __shfl_up(__double2loint(inc), off, 64));
    if (lane >= off) inc += y;
  }
  if (lane == 63) part[w] = inc;
  __syncthreads();
  double before = from;
  for (int i = 0; i < w; ++i) before += part[i];
  const double start = before + (inc - s);
  int low = 0x7fffffff;
  if (before + inc > target || start > target) {
    double run = start;
    for (int t = a0; t < a1; ++t) {
      const double v = of(t);
      run += v;
      if (v > 0.0 && run > target) {
        low = t;
        break;
      }
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    low = min(low, __shfl_xor(low, off, 64));
    some = max(some, __shfl_xor(some, off, 64));
  }
  if (lane == 0) {
    lowest[w] = low;
    highest[w] = some;
  }
  __syncthreads();
  for (int i = 0; i < kDrawThreads / 64; ++i) {
    low = min(low, lowest[i]);
    some = max(some, highest[i]);
  }
  __syncthreads();
  return low < 0x7fffffff ? low : some;
}

// One workgroup per request: the token, and the request's outputs.
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyArgs a, int parts, int cuts) {
  const int req = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const RequestRows q = request_rows(req, a.start[req], a.count[req], 0, a.rows);
  if (q.count <= 0) {
    if (tid == 0) a.accepted[req] = a.back[req] = 0;
    return;
  }
  const Decision d = decisions_at(a, parts)[req];
  int token = d.state == kGreedy ? d.best : -1;
  if (d.state == kTarget || d.state == kRest) {
    const double c = units_of(a, req), r = (double)a.sample_u[req];
    const Weights of = weights_of(a, d, c, d.state == kRest);
    const double* sums = reinterpret_cast<const double*>(decisions_at(a, parts) + a.requests) + (size_t)req * cuts;
    const double mine = lane < cuts ? sums[lane] : 0.0;
    double inc = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double y = __hiloint2double(__shfl_up(__double2hiint(inc), off, 64), __shfl_up(__double2loint(inc), off, 64));
      if (lane >= off) inc += y;
    }
    const double all = __hiloint2double(__shfl(__double2hiint(inc), 63, 64), __shfl(__double2loint(inc), 63, 64));
    if (all > 0.0) {
      const double target = r * all;
      const unsigned long long above = __ballot(mine > 0.0 && inc > target), any = __ballot(mine > 0.0);
      const int k = above ? __ffsll(above) - 1 : 63 - __clzll(any);
      const double upto = inc - mine;
      const double from = __hiloint2double(__shfl(__double2hiint(upto), k, 64), __shfl(__double2loint(upto), k, 64));
      token = draw_from(of, (int)((long long)a.vocab * k / cuts), (int)((long long)a.vocab * (k + 1) / cuts), from, target);
    } else {                             // nothing is left of p: from p itself
      token = draw_from(weights_of(a, d, c, false), 0, a.vocab, 0.0, r * d.z);
    }
  }
  for (int i = tid; i < q.count; i += kDrawThreads)
    a.out[q.row0 + i] = i < d.accepted ? a.tokens[q.row0 + i + 1] : i == d.accepted ? token : -1;
  if (tid == 0) {
    a.accepted[req] = d.accepted;
    a.back[req] = q.count - 1 - d.accepted;
  }
}

static int verify_parts(int rows, int vocab) {
  return std::max(1, std::min({(vocab + kVerStep - 1) / kVerStep, kVerParts, 1536 / std::max(rows, 1)}));
}
static int verify_cuts(int requests, int vocab) {
  return std::max(1, std::min({(vocab + 2047) / 2048, kVerParts, 1024 / std::max(requests, 1)}));
}

size_t verify_work_bytes(int rows, int requests, int vocab) {
  return (size_t)rows * verify_parts(rows, vocab) * sizeof(RowPart) + (size_t)requests * sizeof(Decision) +
         (size_t)requests * verify_cuts(requests, vocab) * sizeof(double);
}

hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
  const int parts = verify_parts(a.rows, a.vocab), cuts = verify_cuts(a.requests, a.vocab);
  hipLaunchKernelGGL(verify_rows_kernel, dim3((unsigned)(a.rows * parts)), dim3(64 * kVerWaves), 0, s, a, parts);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(verify_rest_kernel, dim3((unsigned)(a.requests * cuts)), dim3(64 * kRestWaves), 0, s, a, parts, cuts);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)a.requests), dim3(kDrawThreads), 0, s, a, parts, cuts);
  return hipGetLastError();
}

}  // namespace rehip
