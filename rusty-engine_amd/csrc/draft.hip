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
// 2^-24 one row in a hundred of 151936 would draw a neighbour. So exponentials and sums are in 64 bits. 2^(k / 64 + f / 64),
// |f| <= 1/2: from a table of 64 in LDS and the series of 2^(f / 64) - 1 to its third power, off by (ln 2 / 128)^4 / 24 = 3.6e-11
// at most: a token at the border of 151936 equal ones is then taken for its neighbour once in 200000 times.
//
// Small vocabularies: one launch. Else two: maxima and sums of parts of all rows; then every request's last row found from them, and
// the sums of its weights by blocks of the vocabulary, of which the last workgroup finds the one where r falls, and the token in
// it.
//
// 64 requests of up to 4 drafts, 189 rows of 151936 and the drafts' probabilities, 153 MB: 52 us, 32 + 23 in the two
// kernels. The rows: 115 MB, 3.6 TB/s. Without the exponentials they take 23; the 64-bit operations, 15 of 5 clocks for each logit, are
// 14 on all SIMDs: neither bounds by itself, the two run mostly one after the other (a table of 32 and one term more: 34.5). One
// request of 4 drafts 10.5 .. 13 us: two launches of latency, 5 + 9.
constexpr int kVerWaves = 4;
constexpr int kVerBatch = 16;            // logits of a lane at a time
constexpr int kVerStep = 64 * kVerBatch * kVerWaves;
constexpr int kVerParts = 64;            // a lane each
constexpr int kVerTable = 64;

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
  int best;
};
constexpr int kNone = 0, kGreedy = 1, kTarget = 2, kRest = 3;  // no distribution; the largest; p; p without the draft

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// 2^y, y <= 0: the series at the nearest integer, 13 terms, off by (ln 2 / 2)^13 / 13! = 2e-16
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

// The table: 2^(i / 64). All threads of the workgroup call it.
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < kVerTable) table[threadIdx.x] = 2.0 * pow2_64(((int)threadIdx.x - kVerTable) / (double)kVerTable);
  __syncthreads();
}

// 2^((x - m) c), c64 = 64 c; what is below 2^-1000 comes out as that
__device__ __forceinline__ double share_of(float x, double m, double c64, const double* table) {
  constexpr double kRound = 6755399441055744.0;                // 1.5 2^52: a sum's low word is then the nearest integer
  constexpr double k1 = 0.69314718055994530942 / kVerTable, k2 = k1 * k1 / 2.0, k3 = k1 * k1 * k1 / 6.0;
  const double y = fmax(((double)x - m) * c64, -1000.0 * kVerTable), t = y + kRound;
  const double f = y - (t - kRound);
  const int n = __double2loint(t);
  const double b = table[n & (kVerTable - 1)];
  const double q = f * fma(f, fma(f, k3, k2), k1), w = fma(b, q, b);
  return __hiloint2double(__double2hiint(w) + (n >> 6) * (1 << 20), __double2loint(w));
}
// .. and exactly 0 there and for a logit of -inf
__device__ __forceinline__ double weight_of(float x, double m, double c64, const double* table) {
  const double w = share_of(x, m, c64, table);
  return x == -INFINITY || ((double)x - m) * c64 < -1000.0 * kVerTable ? 0.0 : w;
}

template <int OFF>
__device__ __forceinline__ double lane_xor64(double v) {
  return __hiloint2double((int)lane_xor_u32<OFF>((unsigned)__double2hiint(v)), (int)lane_xor_u32<OFF>((unsigned)__double2loint(v)));
}
__device__ __forceinline__ double wave_sum64(double v) {
  wave_butterfly([&](auto off) { v += lane_xor64<decltype(off)::value>(v); });
  return v;
}
// inclusive sums over the lanes of a wave
__device__ __forceinline__ double wave_scan64(double v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double y = __hiloint2double(__shfl_up(__double2hiint(v), off, 64), __shfl_up(__double2loint(v), off, 64));
    if ((int)(threadIdx.x & 63) >= off) v += y;
  }
  return v;
}

// 64 powers of 2 for each unit of logit; greedy below 0
__device__ __forceinline__ double units_of(const VerifyArgs& a, int req) {
  const float t = a.temperature ? a.temperature[req] : 1.0f;
  return t > 0.0f ? kVerTable * 1.4426950408889634074 / (double)t : -1.0;
}

__device__ __forceinline__ PagedBatch rows_of(const VerifyArgs& a) {
  return {a.start, a.count, a.count, nullptr, a.requests, a.rows, 1, 1, 1};
}

// A wave's lanes joined, the same in every lane: sums of shares to the largest maximum.
__device__ __forceinline__ RowPart joined_wave(const RowPart& p, double c64) {
  const float m = wave_max(p.m);
  double z = 0.0;
  if (c64 >= 0.0) z = wave_sum64(p.m > -INFINITY ? p.z * pow2_64(((double)p.m - (double)m) * (c64 / kVerTable)) : 0.0);
  int best = p.m == m ? p.best : 0x7fffffff, bad = p.bad;
  wave_butterfly([&](auto off) {
    constexpr int X = decltype(off)::value;
    best = min(best, (int)lane_xor_u32<X>((unsigned)best));
    bad |= (int)lane_xor_u32<X>((unsigned)bad);
  });
  return {z, m, best, bad, 0};
}

// A lane's part of a row: elements 256 i + 4 lane .. + 3, i < 4, from `base` on, and so on every `step`, of steps s0 .. s1 - 1; whole
// steps first, the next one loading meanwhile (a load under a condition would be waited for), then the row's last part of one.
// begin() is called while the first is on its way; it gives the units, and whether the row counts.
template <class Begin>
__device__ __forceinline__ RowPart row_part(const float* x, int vocab, int s0, int s1, int step, int base, const double* table,
                                            double& c64, Begin begin) {
  const int lane = threadIdx.x & 63;
  auto place = [&](int s, int k) { return s * step + base + 256 * (k >> 2) + 4 * lane + (k & 3); };
  auto load = [&](int s, float (&v)[kVerBatch]) {
#pragma unroll
    for (int k = 0; k < kVerBatch; k += 4)
      *reinterpret_cast<f32x4u*>(&v[k]) = *reinterpret_cast<const f32x4u*>(x + place(s, k));
  };
  const int whole = min(s1, vocab / step);
  float v[kVerBatch], nx[kVerBatch];
  if (s0 < whole) load(s0, v);
  RowPart mine{0.0, -INFINITY, 0x7fffffff, 0, 0};
  if (!begin()) return mine;
  auto take = [&](const float (&v)[kVerBatch], int s) {
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVerBatch; ++k) {
      mine.bad |= !(v[k] < INFINITY);
      mx = fmaxf(mx, v[k]);
    }
    if (mx > mine.m) {
      if (c64 >= 0.0 && mine.m > -INFINITY) mine.z *= share_of(mine.m, (double)mx, c64, table);
      mine.m = mx;
#pragma unroll
      for (int k = kVerBatch - 1; k >= 0; --k)
        if (v[k] == mx) mine.best = place(s, k);
    }
    if (c64 >= 0.0 && mine.m > -INFINITY) {
      double z[4] = {};
      const double m = (double)mine.m;
#pragma unroll
      for (int k = 0; k < kVerBatch; ++k) z[k & 3] += share_of(v[k], m, c64, table);
      mine.z += (z[0] + z[1]) + (z[2] + z[3]);
    }
  };
  int s = s0;
  for (; s < whole; ++s) {
    load(min(s + 1, whole - 1), nx);
    take(v, s);
#pragma unroll
    for (int k = 0; k < kVerBatch; ++k) v[k] = nx[k];
  }
  if (s < s1) {
#pragma unroll
    for (int k = 0; k < kVerBatch; ++k) {
      const int at = place(s, k);
      const float y = x[min(at, vocab - 1)];
      v[k] = at < vocab ? y : -INFINITY;
    }
    take(v, s);
  }
  return mine;
}

// behind the rows' parts: of each request the workgroups that are done with it, then the sums of its blocks (never negative, and
// kNotYet until they are there)
constexpr double kNotYet = -1.0;
__device__ __forceinline__ int* done_at(const VerifyArgs& a, int parts) {
  return reinterpret_cast<int*>(reinterpret_cast<RowPart*>(a.work) + (size_t)a.rows * parts);
}
__device__ __forceinline__ double* sums_at(const VerifyArgs& a, int parts) {
  return reinterpret_cast<double*>(done_at(a, parts) + ((a.requests + 1) & ~1));
}

// One workgroup per (row, part).
__global__ __launch_bounds__(64 * kVerWaves) void verify_rows_kernel(VerifyArgs a, int parts, int blocks) {
  __shared__ double table[kVerTable];
  __shared__ RowPart ws[kVerWaves];
  const int r = blockIdx.x / parts, part = blockIdx.x % parts;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int steps = (a.vocab + kVerStep - 1) / kVerStep;
  const int s0 = (int)((long long)steps * part / parts), s1 = (int)((long long)steps * (part + 1) / parts);
  double c64 = 0.0;
  bool counts = false;
  const RowPart mine = row_part(a.x + (size_t)r * a.ld, a.vocab, s0, s1, kVerStep, w * 64 * kVerBatch, table, c64, [&] {
    const RequestRows q = request_of_unit(r, rows_of(a), 1, 0);
    counts = q.req >= 0 && r < q.row0 + q.count;
    if (!counts) return false;
    c64 = units_of(a, q.req);
    if (r == q.row0 && part == 0) {
      if (threadIdx.x == 0) done_at(a, parts)[q.req] = 0;
      double* const sums = sums_at(a, parts) + (size_t)q.req * blocks;
      for (int k = threadIdx.x; k < blocks; k += 64 * kVerWaves) sums[k] = kNotYet;
    }
    fill_table(table);
    return true;
  });
  if (!counts) return;
  const RowPart all = joined_wave(mine, c64);
  if (lane == 0) ws[w] = all;
  __syncthreads();
  if (w == 0) {
    const RowPart p = lane < kVerWaves ? ws[lane] : RowPart{0.0, -INFINITY, 0x7fffffff, 0, 0};
    const RowPart o = joined_wave(p, c64);
    if (lane == 0) reinterpret_cast<RowPart*>(a.work)[blockIdx.x] = o;
  }
}

// How many drafts of a request are accepted, and where its next token comes from. Every wave of the workgroup looks at a row of
// its own at a time; part(row) gives what its lanes hold of it.
template <int WAVES, class Part>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, const RequestRows& q, double c64, Part part) {
  __shared__ Decision found[WAVES];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Decision d{};
  for (int i0 = 0; i0 < q.count; i0 += WAVES) {
    const int i = i0 + w, row = q.row0 + min(i, q.count - 1);
    const bool drafted = i < q.count - 1;
    // (the draft's logit and probability are on their way with the row's parts; the last row has no draft, and no more than its
    // logits need be there)
    const int t = drafted ? a.tokens[row + 1] : 0, at = min(max(t, 0), a.vocab - 1);
    const float x = a.x[(size_t)row * a.ld + at];
    const float share = drafted && a.probs ? a.probs[(size_t)row * a.ldp + at] : 1.0f, u = drafted ? a.accept_u[row] : 0.0f;
    const RowPart p = joined_wave(part(row), c64);
    const bool none = p.bad || p.m == -INFINITY;
    bool accepted = false;
    if (drafted && !none && t == at)
      accepted = c64 < 0.0 ? t == p.best
                           : (double)u * (double)share * p.z <
                                 (x == -INFINITY ? 0.0 : pow2_64(((double)x - (double)p.m) * (c64 / kVerTable)));
    if (lane == 0)
      found[w] = {p.z, p.m, accepted ? -1 : i, row, none ? kNone : c64 < 0.0 ? kGreedy : drafted ? kRest : kTarget, p.best};
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

// The weight of token t, of logit x and the draft's probability there: p, less the draft's share of it
struct Weights {
  const float* x;
  const float* probs;                    // the draft's row, or null
  double c64, m, inverse;               // 1 / z
  int drop;                              // a draft without a distribution: this token has no weight (-1: none)
  const double* table;
  __device__ __forceinline__ double operator()(int t, float xt, float qt) const {
    const double e = weight_of(xt, m, c64, table);
    if (probs) return fmax(fma(e, inverse, -(double)qt), 0.0);
    return t == drop ? 0.0 : e;
  }
};
__device__ __forceinline__ Weights weights_of(const VerifyArgs& a, const Decision& d, double c64, bool rest, const double* table) {
  const int t = rest && !a.probs ? a.tokens[d.row + 1] : -1;
  return {a.x + (size_t)d.row * a.ld, rest && a.probs ? a.probs + (size_t)d.row * a.ldp : nullptr, c64, (double)d.m,
          1.0 / d.z, t, table};
}

// Exclusive sums over a workgroup of WAVES waves; the total in `all`.
template <int WAVES>
__device__ __forceinline__ double scan_block64(double v, double& all) {
  __shared__ double part[WAVES];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const double inc = wave_scan64(v);
  if (lane == 63) part[w] = inc;
  __syncthreads();
  double before = 0.0;
  all = 0.0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    before += i < w ? part[i] : 0.0;
    all += part[i];
  }
  __syncthreads();
  return before + (inc - v);
}
// the least over the workgroup, and the largest
template <int WAVES>
__device__ __forceinline__ int2 ends_block(int low, int high) {
  __shared__ int part[2][WAVES];
  wave_butterfly([&](auto off) {
    constexpr int X = decltype(off)::value;
    low = min(low, (int)lane_xor_u32<X>((unsigned)low));
    high = max(high, (int)lane_xor_u32<X>((unsigned)high));
  });
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    part[0][w] = low;
    part[1][w] = high;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    low = min(low, part[0][i]);
    high = max(high, part[1][i]);
  }
  __syncthreads();
  return make_int2(low, high);
}

// Of places t0 .. t1 - 1 with value(t) each the lowest whose running sum, from `from` on, is above target(their sum), or the last
// with a value above 0 if rounding leaves none (-1: there is none at all); `upto`: the sum of the places before it. A thread
// has `per` places that follow one another. All threads call it.
template <int WAVES, class F, class Target>
__device__ __forceinline__ int first_above(F value, int t0, int t1, int per, double from, Target target_of, double& upto) {
  __shared__ double found;
  const int a0 = min(t0 + (int)threadIdx.x * per, t1), a1 = min(a0 + per, t1);
  double s = 0.0, all;
  int some = -1;
  for (int t = a0; t < a1; ++t) {
    const double v = value(t);
    s += v;
    if (v > 0.0) some = t;
  }
  double run = from + scan_block64<WAVES>(s, all), before = run;
  const double target = target_of(all);
  const int last = some;
  int low = 0x7fffffff;
  if (some >= 0 && !(run + s <= target)) {
    for (int t = a0; t < a1; ++t) {
      const double v = value(t);
      if (v > 0.0 && run + v > target) {
        low = t;
        break;
      }
      run += v;
    }
  }
  const int2 e = ends_block<WAVES>(low, some);
  const int at = e.x < 0x7fffffff ? e.x : e.y;
  if (at >= 0 && (e.x < 0x7fffffff ? low == at : last == at)) {
    if (e.x == 0x7fffffff) {             // (up to the last one)
      run = before;
      for (int t = a0; t < at; ++t) run += value(t);
    }
    found = run;
  }
  __syncthreads();
  upto = found;
  __syncthreads();
  return at;
}

template <int WAVES>
__device__ __forceinline__ void write_request(const VerifyArgs& a, const RequestRows& q, const Decision& d, int token) {
  for (int i = threadIdx.x; i < q.count; i += 64 * WAVES)
    a.out[q.row0 + i] = i < d.accepted ? a.tokens[q.row0 + i + 1] : i == d.accepted ? token : -1;
  if (threadIdx.x == 0) {
    a.accepted[q.req] = d.accepted;
    a.back[q.req] = q.count - 1 - d.accepted;
  }
}

// One workgroup per (request, run of blocks of the vocabulary), a block to a wave at a time: the sums of their weights. The last one
// of a request that is done with them draws the token (whichever it is, the sums are added in the blocks' order).
constexpr int kRestWaves = 8;
constexpr int kBlock = 1024;             // tokens of a block
constexpr int kRestMost = 512;           // workgroups, about (us of 256 / 512 / 1024: 64 requests of 151936 tokens 51.8 / 49.6 / 57.0, 200 of
                                         // 32000 40.3 / 40.1 / 45.1)
constexpr int kMostWaits = 1 << 16;      // loads, about a microsecond each
template <bool PROBS>
__global__ __launch_bounds__(64 * kRestWaves) void verify_rest_kernel(VerifyArgs a, int parts, int cuts, int blocks) {
  constexpr int kThreads = 64 * kRestWaves;
  __shared__ double table[kVerTable];
  __shared__ int last;
  const int req = blockIdx.x / cuts, cut = blockIdx.x % cuts, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const RequestRows q = request_rows(req, a.start[req], a.count[req], 0, a.rows);
  if (q.count <= 0) {
    if (cut == 0 && threadIdx.x == 0) a.accepted[req] = a.back[req] = 0;
    return;
  }
  const double c64 = units_of(a, req);
  fill_table(table);
  const Decision d = decide<kRestWaves>(a, q, c64, [&](int row) {
    const RowPart p = reinterpret_cast<const RowPart*>(a.work)[(size_t)row * parts + min(lane, parts - 1)];
    return lane < parts ? p : RowPart{0.0, -INFINITY, 0x7fffffff, 0, 0};
  });
  if (d.state != kTarget && d.state != kRest) {
    if (cut == 0) write_request<kRestWaves>(a, q, d, d.state == kGreedy ? d.best : -1);
    return;
  }
  Weights of = weights_of(a, d, c64, d.state == kRest, table);
  double* const sums = sums_at(a, parts) + (size_t)req * blocks;
  const int b0 = (int)((long long)blocks * cut / cuts), b1 = (int)((long long)blocks * (cut + 1) / cuts);
  auto place = [&](int b, int k) { return b * kBlock + 256 * (k >> 2) + 4 * lane + (k & 3); };
  const float* probs = of.probs ? of.probs : of.x;                 // (loaded whatever)
  auto load = [&](int b, float (&x)[16], float (&p)[16]) {
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      *reinterpret_cast<f32x4u*>(&x[k]) = *reinterpret_cast<const f32x4u*>(of.x + place(b, k));
      if (PROBS) *reinterpret_cast<f32x4u*>(&p[k]) = *reinterpret_cast<const f32x4u*>(probs + place(b, k));
    }
  };
  auto take = [&](const float (&x)[16], const float (&p)[16], int b) {
    double s[4] = {};
#pragma unroll
    for (int k = 0; k < 16; ++k) s[k & 3] += of(place(b, k), x[k], PROBS ? p[k] : 0.0f);
    const double all = wave_sum64((s[0] + s[1]) + (s[2] + s[3]));
    if (lane == 0) __hip_atomic_store(sums + b, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  float x[16], p[16], nx[16], np[16];
  const int whole = min(b1, a.vocab / kBlock);
  int b = b0 + w;
  if (b < whole) load(b, x, p);
  for (; b < whole; b += kRestWaves) {
    load(b + kRestWaves < whole ? b + kRestWaves : b, nx, np);
    take(x, p, b);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      x[k] = nx[k];
      if (PROBS) p[k] = np[k];
    }
  }
  if (b < b1) {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int t = min(place(b, k), a.vocab - 1);
      const float y = of.x[t];
      x[k] = place(b, k) < a.vocab ? y : -INFINITY;
      if (PROBS) p[k] = probs[t];
    }
    take(x, p, b);
  }
  if (cuts > 1) {
    __syncthreads();
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(done_at(a, parts) + req, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == cuts - 1;
    __syncthreads();
    if (!last) return;
  } else {
    __syncthreads();
  }
  // The counter orders nothing: a sum that is not here yet is waited for, by itself. (us of 64 requests and of one: so 52.4 and 11.8, with
  // a counter that releases and acquires, which writes the L2 back in every workgroup, 55.5 and 12, with a launch of its own for
  // what follows 53.5 and 14.) All sums have been stored by then, so it takes a trip to memory more or none; that the wait
  // ends does not depend on it.
  auto sum = [&](int k) {
    double v = kNotYet;
    for (int i = 0; i < kMostWaits && v == kNotYet; ++i) v = __hip_atomic_load(sums + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return v;
  };
  const double r = (double)a.sample_u[req];
  auto value = [&](int t) { return of(t, of.x[t], of.probs ? of.probs[t] : 0.0f); };
  double target = 0.0, upto, none;
  const int found = first_above<kRestWaves>(sum, 0, blocks, (blocks + kThreads - 1) / kThreads, 0.0,
                                            [&](double all) { return target = r * all; }, upto);
  int token;
  if (found >= 0) {
    token = first_above<kRestWaves>(value, found * kBlock, min((found + 1) * kBlock, a.vocab), kBlock / kThreads, upto,
                                    [&](double) { return target; }, none);
  } else {                               // nothing is left of p: from p itself
    of = weights_of(a, d, c64, false, table);
    token = first_above<kRestWaves>(value, 0, a.vocab, (a.vocab + kThreads - 1) / kThreads, 0.0,
                                    [&](double) { return r * d.z; }, none);
  }
  write_request<kRestWaves>(a, q, d, token);
}

// Small vocabularies: all of a request in one workgroup, a wave for each row, then the weights from the row again.
constexpr int kSmallWaves = 8, kSmallVocab = 2048;
__global__ __launch_bounds__(64 * kSmallWaves) void verify_small_kernel(VerifyArgs a) {
  constexpr int kThreads = 64 * kSmallWaves, kStep = 64 * kVerBatch;
  __shared__ double table[kVerTable];
  const int req = blockIdx.x;
  const RequestRows q = request_rows(req, a.start[req], a.count[req], 0, a.rows);
  if (q.count <= 0) {
    if (threadIdx.x == 0) a.accepted[req] = a.back[req] = 0;
    return;
  }
  double c64 = units_of(a, req);
  fill_table(table);
  const Decision d = decide<kSmallWaves>(a, q, c64, [&](int row) {
    return row_part(a.x + (size_t)row * a.ld, a.vocab, 0, (a.vocab + kStep - 1) / kStep, kStep, 0, table, c64, [] { return true; });
  });
  int token = d.state == kGreedy ? d.best : -1;
  if (d.state == kTarget || d.state == kRest) {
    const double r = (double)a.sample_u[req];
    Weights of = weights_of(a, d, c64, d.state == kRest, table);
    auto value = [&](int t) { return of(t, of.x[t], of.probs ? of.probs[t] : 0.0f); };
    const int per = (a.vocab + kThreads - 1) / kThreads;
    auto target = [&](double all) { return r * all; };
    double none;
    token = first_above<kSmallWaves>(value, 0, a.vocab, per, 0.0, target, none);
    if (token < 0) {                     // nothing is left of p: from p itself
      of = weights_of(a, d, c64, false, table);
      token = first_above<kSmallWaves>(value, 0, a.vocab, per, 0.0, target, none);
    }
  }
  write_request<kSmallWaves>(a, q, d, token);
}

// about four workgroups for each CU (us of 768 / 1024 / 1536 / 2048: 200 requests of up to 3 drafts, 32000 tokens 38.5 / 38.3 / 40.1 / 41.1, 32 of
// up to 4, 64000 24.0 / 23.8 / 24.7 / 24.4, 8 of up to 4, 151936 21.2 / 20.7 / 20.5 / 20.2)
constexpr int kVerGroups = 1024;
static int verify_parts(int rows, int vocab) {
  return std::max(1, std::min({(vocab + kVerStep - 1) / kVerStep, kVerParts, kVerGroups / std::max(rows, 1)}));
}
static int verify_blocks(int vocab) { return (vocab + kBlock - 1) / kBlock; }

// (at least what fewer rows, requests or tokens take, so that a program's largest step may size it for all)
size_t verify_work_bytes(int rows, int requests, int vocab) {
  const size_t parts = std::max((size_t)rows, std::min((size_t)kVerGroups, (size_t)rows * verify_parts(1, vocab)));
  return parts * sizeof(RowPart) + (size_t)((requests + 1) & ~1) * sizeof(int) +
         (size_t)requests * verify_blocks(vocab) * sizeof(double);
}

hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
  // (us of one / two launches, 4 drafts each: one request of 500 tokens 8.8 / 11.6, of 2000 8.8 / 12.3, of 4000 12.0 / 12.6; 64 of 500
  // 8.7 / 15.8, of 2000 11.3 / 16.6, of 4000 18.2 / 16.9; 32 of 2000, 16 drafts 16.2 / 18.6)
  if (a.vocab <= kSmallVocab) {
    hipLaunchKernelGGL(verify_small_kernel, dim3((unsigned)a.requests), dim3(64 * kSmallWaves), 0, s, a);
    return hipGetLastError();
  }
  const int parts = verify_parts(a.rows, a.vocab), blocks = verify_blocks(a.vocab);
  const int cuts = std::max(1, std::min((blocks + kRestWaves - 1) / kRestWaves, kRestMost / a.requests));
  hipLaunchKernelGGL(verify_rows_kernel, dim3((unsigned)(a.rows * parts)), dim3(64 * kVerWaves), 0, s, a, parts, blocks);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(a.probs ? verify_rest_kernel<true> : verify_rest_kernel<false>, dim3((unsigned)(a.requests * cuts)),
                     dim3(64 * kRestWaves), 0, s, a, parts, cuts, blocks);
  return hipGetLastError();
}

}  // namespace rehip
