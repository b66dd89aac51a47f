// K/V cache in int8 pages with one scale for each page and KV head, and the attention that reads it.
//
// Codes of one page and head are blocks of 32 tokens x 32 dimensions, 1 KiB each, [page / 32][hd / 32], in the
// order in which the lanes of a wave hold the operands of the 16 x 16 x 32 matrix instruction: lane l's 16 bytes
// follow one another, so a block is one load of 16 bytes per lane. With m = l % 16 and g = l / 16,
//   K: byte 16 l + 8 t + j        is token 16 t + m,         dimension 8 g + j   (t < 2, j < 8)
//   V: byte 16 l + 8 b + 4 t + i  is token 16 t + 4 g + i,   dimension 16 b + m  (b, t < 2, i < 4)
#include <hip/hip_runtime.h>

#include <algorithm>

#include "serve.hpp"
#include "wave.hpp"

namespace rehip {

// ---- append --------------------------------------------------------------------------------------
// A page and head's scale s is the largest finite magnitude of what it holds / 127 (0 below the smallest normal
// float: such values are stored as 0), a value's code round(x / s), ties to even. Rows that raise the scale of a
// page with earlier rows in it round those rows' codes to the new one: round(c * (s_old / s_new)). Infinities
// are stored as +-127 and NaN as 0, so that one bad value does not reach the page's other tokens.
//
// The quotient is the correctly rounded one: with y = 1 / s rounded, q = x y, then twice q += (x - q s) y in fused
// multiply-adds, whose remainders are exact (the first leaves q within one unit of the last place, the second rounds it
// right: Markstein). Below 2^-100 remainders could underflow: there the division itself is used. Of finite values
// |q| <= 127 (1 + 2^-23), and q + 1.5 2^23 rounds it to an integer, whose low byte is the code.
//
// Bound by HBM for prompts: 9260 rows of 8 heads of 128, 94.8 MB, 18.4 us, 5.1 TB/s (as a copy of 1 GiB). A decode
// step (64 rows, 0.33 MB) is three dependent trips to memory, the rows' places, the page number, the values: 3.9 us in the
// kernel.
constexpr float kCodeMagic = 12582912.0f;

__device__ __forceinline__ unsigned code_of(float x, float s, float y) {
  float q = x * y;
  q = __builtin_fmaf(__builtin_fmaf(-q, s, x), y, q);
  q = __builtin_fmaf(__builtin_fmaf(-q, s, x), y, q);
  return __float_as_uint(q + kCodeMagic);
}
__device__ unsigned code_of_any(float x, float s) {
  const float q = rintf(x / s);
  return x != x || s == 0.0f ? 0u : (unsigned)(int)fminf(fmaxf(q, -127.0f), 127.0f);
}
// the low bytes of four
__device__ __forceinline__ unsigned bytes4(unsigned a, unsigned b, unsigned c, unsigned d) {
  const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// Token of a lane's first code in a block (blocks of the page in order, nb for 32 tokens), and of its code e.
template <bool IS_V>
__device__ __forceinline__ int first_token(int blk, int nb) {
  const int lane = threadIdx.x & 63;
  return 32 * (blk / nb) + (IS_V ? 4 * (lane >> 4) : lane & 15);
}
template <bool IS_V>
__device__ __forceinline__ int token_of(int first, int e) {
  return first + (IS_V ? 16 * ((e >> 2) & 1) + (e & 3) : 16 * (e >> 3));
}
__device__ __forceinline__ int held_code(const uint4& u, int e) { return (int)(int8_t)((&u.x)[e >> 2] >> (8 * (e & 3))); }

// The page's scale from the threads' largest magnitudes of the new tokens and of what it held (s_old). W waves work
// together, the whole workgroup or one.
struct PageScale {
  float s, ratio, inverse;   // of old codes to new ones; 1 / s
  bool grown, plain;         // plain: every value is finite and the quotient may be taken by remainders
};
constexpr int kAppendWaves = 16;
typedef float AppendRed[2][kAppendWaves];

template <int W>
__device__ __forceinline__ float largest_of(const float (&v)[kAppendWaves]) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < W; ++i) m = fmaxf(m, v[i]);
  return m;
}
template <int W>
__device__ __forceinline__ PageScale page_scale(float top, float odd, float s_old, const float* __restrict__ x, int ld,
                                                int o0, int o1, int hd, AppendRed& red) {
  const int tid = W == 1 ? threadIdx.x & 63 : threadIdx.x, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  top = wave_max(top);
  odd = wave_sum(odd);
  if constexpr (W > 1) {
    if ((tid & 63) == 0) { red[0][w] = top; red[1][w] = odd; }
    __syncthreads();
    top = largest_of<W>(red[0]);
    odd = red[1][0];
#pragma unroll
    for (int i = 1; i < W; ++i) odd += red[1][i];
  }
  if (odd != odd) {                        // the finite ones only
    top = 0.0f;
    for (int e = tid; e < (o1 - o0) * hd; e += 64 * W) {
      const float v = fabsf(x[e / hd * ld + e % hd]);
      if (v < INFINITY) top = fmaxf(top, v);
    }
    top = wave_max(top);
    if constexpr (W > 1) {
      __syncthreads();
      if ((tid & 63) == 0) red[0][w] = top;
      __syncthreads();
      top = largest_of<W>(red[0]);
    }
  }
  if (o0 == 0) s_old = 0.0f;               // the page is begun: what it held before does not count
  float s = top * (1.0f / 127.0f);
  if (s < 1.17549435e-38f) s = 0.0f;
  s = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(fmaxf(s, s_old))));
  const bool grown = o0 > 0 && s > s_old;
  return {s, grown ? s_old / s : 1.0f, 1.0f / s, grown, s >= 7.8886091e-31f && odd == odd};
}

// One page's new tokens o0 .. o1 - 1 of one head: x is token o0's row, codes and scale the page's. A thread has U units of
// 16 codes that lie together in memory (K: 2 tokens x 8 dimensions, V: 8 tokens x 2), 64 lanes' units a block of 32 x 32:
// it loads their values, and the codes of a page that is not all new, before the largest magnitude is known, so that all
// of this is one round trip to memory. Units past the page's (U rounded up) repeat the last and are not stored.
// U = 0 (a prompt of large pages in a decode step): the units in turn, their values read twice.
template <bool IS_V, int U, int W>
__device__ __forceinline__ void append_page(const float* __restrict__ x, int ld, int o0, int o1, int page, int hd,
                                            int8_t* codes, float* scale, AppendRed& red) {
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4;
  const int nb = hd >> 5, blocks = (page >> 5) * nb;
  const bool all_new = o0 == 0 && o1 == page;
  auto load = [&](int blk, float (&y)[16]) {
    const int t = first_token<IS_V>(blk, nb), d = 32 * (blk % nb) + (IS_V ? m : 8 * g);
    // (of a token that is not new, some new one's values: a load under a condition of its lane waits for the one before)
    auto row = [&](int e) { return x + ((min(max(token_of<IS_V>(t, e), o0), o1 - 1) - o0) * ld + d); };
    if constexpr (IS_V) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float* r = row(e);
        y[e] = r[0];
        y[e + 8] = r[16];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; e += 8) {
        const float* r = row(e);
        *reinterpret_cast<float4*>(&y[e]) = *reinterpret_cast<const float4*>(r);
        *reinterpret_cast<float4*>(&y[e + 4]) = *reinterpret_cast<const float4*>(r + 4);
      }
    }
  };
  uint4* const units = reinterpret_cast<uint4*>(codes) + lane;    // unit of block blk: units[64 * blk]
  float y[U > 0 ? U : 1][16];
  uint4 old[U > 0 ? U : 1];
  const float s_old = *scale;
  float top = 0.0f, odd = 0.0f;            // odd: NaN once an infinity or a NaN was seen
  auto largest = [&](const float (&z)[16]) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      top = fmaxf(top, fabsf(z[e]));
      odd = __builtin_fmaf(z[e], 0.0f, odd);
    }
  };
  if constexpr (U > 0) {
#pragma unroll
    for (int i = 0; i < U; ++i) load(min(w + W * i, blocks - 1), y[i]);
    if (!all_new) {
#pragma unroll
      for (int i = 0; i < U; ++i) old[i] = units[64 * min(w + W * i, blocks - 1)];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) largest(y[i]);
  } else {
    for (int blk = w; blk < blocks; blk += W) {
      load(blk, y[0]);
      largest(y[0]);
    }
  }
  const PageScale sc = page_scale<W>(top, odd, s_old, x, ld, o0, o1, hd, red);
  auto store = [&](int blk, const float (&z)[16], const uint4& was) {
    unsigned c[16], out[4];
    if (sc.plain) {
#pragma unroll
      for (int e = 0; e < 16; ++e) c[e] = code_of(z[e], sc.s, sc.inverse);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) c[e] = code_of_any(z[e], sc.s);
    }
    if (!all_new) {
      const int t = first_token<IS_V>(blk, nb);
      bool changes = false;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int tok = token_of<IS_V>(t, e), held = held_code(was, e);
        if (tok < o0) c[e] = sc.grown ? (unsigned)(int)rintf((float)held * sc.ratio) : (unsigned)held;
        if (tok >= o1) c[e] = (unsigned)held;
        changes |= tok < o1 && (tok >= o0 || sc.grown);
      }
      if (!changes) return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = bytes4(c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]);
    units[64 * blk] = make_uint4(out[0], out[1], out[2], out[3]);
  };
  if constexpr (U > 0) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (w + W * i < blocks) store(w + W * i, y[i], old[i]);
  } else {
    for (int blk = w; blk < blocks; blk += W) {
      load(blk, y[0]);
      if (!all_new) old[0] = units[64 * blk];
      store(blk, y[0], old[0]);
    }
  }
  if (tid == 0) *scale = sc.s;
}

// The same where the new tokens have at most four values for each thread of W waves: their codes go straight to their bytes, and
// the page's other codes are read and written only if its scale grows (us of the workgroup's four waves / by whole units: 64
// tokens, 4 heads of 128 4.8 / 8.7 in the kernel, 256 tokens, 8 heads of 256, pages of 256 15 / 162, 512 times 8 rows, 4 of
// 128 19 / 34. Old codes loaded beforehand, on their way with the values, did not pay: 1000 tokens, 8 heads of 128 64 -> 72).
template <bool IS_V, int W>
__device__ __forceinline__ void append_few(const float* __restrict__ x, int ld, int o0, int o1, int page, int hd,
                                           int8_t* codes, float* scale, AppendRed& red) {
  const int lane = threadIdx.x & 63, w = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tid = 64 * w + lane;
  const int nb = hd >> 5, blocks = (page >> 5) * nb, n = (o1 - o0) * hd;
  const int at = min(4 * tid, n - 4), row = at / hd, d = at - row * hd;
  const float4 y = *reinterpret_cast<const float4*>(x + (row * ld + d));
  const float z[4] = {y.x, y.y, y.z, y.w};
  float top = 0.0f, odd = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    top = fmaxf(top, fabsf(z[e]));
    odd = __builtin_fmaf(z[e], 0.0f, odd);
  }
  const PageScale sc = page_scale<W>(top, odd, *scale, x, ld, o0, o1, hd, red);
  if (sc.grown) {
    uint4* const units = reinterpret_cast<uint4*>(codes) + lane;
    for (int b0 = w; b0 < blocks; b0 += 4 * W) {
      uint4 old[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) old[i] = units[64 * min(b0 + W * i, blocks - 1)];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int blk = b0 + W * i, t = first_token<IS_V>(blk, nb);
        if (blk >= blocks) break;
        unsigned c[16], out[4];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int held = held_code(old[i], e);
          c[e] = token_of<IS_V>(t, e) < o0 ? (unsigned)(int)rintf((float)held * sc.ratio) : (unsigned)held;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = bytes4(c[4 * j], c[4 * j + 1], c[4 * j + 2], c[4 * j + 3]);
        units[64 * blk] = make_uint4(out[0], out[1], out[2], out[3]);
      }
    }
    if constexpr (W == 1) wave_sync();     // the new codes come after
    else __syncthreads();
  }
  if (tid == 0) *scale = sc.s;
  if (4 * tid >= n) return;
  unsigned c[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] = sc.plain ? code_of(z[e], sc.s, sc.inverse) : code_of_any(z[e], sc.s);
  const int tok = o0 + row, t = tok & 31, dd = d & 31;
  int8_t* const block = codes + 1024 * ((tok >> 5) * nb + (d >> 5));
  if constexpr (IS_V) {
    int8_t* const o = block + 256 * (t >> 2 & 3) + 16 * (dd & 15) + 8 * (dd >> 4) + 4 * (t >> 4) + (t & 3);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[16 * e] = (int8_t)c[e];
  } else {
    *reinterpret_cast<unsigned*>(block + 256 * (dd >> 3) + 16 * (t & 15) + 8 * (t >> 4) + (dd & 7)) =
        bytes4(c[0], c[1], c[2], c[3]);
  }
}

// One workgroup per (run of one request's new rows inside one page, head or four heads, K or V).
template <bool IS_V, int U, int W>
__device__ __forceinline__ void append_head(const float* __restrict__ x, int ld, int o0, int o1, int page, int hd,
                                            int8_t* codes, float* scale, AppendRed& red) {
  if ((o1 - o0) * hd <= 256 * W) append_few<IS_V, W>(x, ld, o0, o1, page, hd, codes, scale, red);
  else append_page<IS_V, U, W>(x, ld, o0, o1, page, hd, codes, scale, red);
}

template <bool IS_V, int U, int W, bool FOUR>
__device__ __forceinline__ void append_run(const PagedBatch& b, const Kv8Cache& c, const float* __restrict__ x, int ld,
                                           int8_t* codes, float* scale, AppendRed& red) {
  const int u = blockIdx.x;
  const RequestRows q = request_of_unit(u, b, b.page, 2);
  const int n = q.count, len = q.len, first = len - n;
  if (n == 0 || first < 0 || len > b.table_ld * b.page) return;
  const int pi = first / b.page + (u - (q.row0 / b.page + 2 * q.req));
  const int lo = max(pi * b.page, first), hi = min((pi + 1) * b.page, len);   // positions
  if (lo >= hi) return;
  const int pid = b.table[(size_t)q.req * b.table_ld + pi];
  if (pid < 0 || pid >= b.n_pages) return;
  const int o0 = lo - pi * b.page, o1 = hi - pi * b.page, size = b.page * c.hd;
  const size_t page0 = (size_t)pid * c.kv_heads;
  x += (size_t)(q.row0 + lo - first) * ld;
  if constexpr (!FOUR) {
    const int h = blockIdx.y;
    append_head<IS_V, U, W>(x + h * c.hd, ld, o0, o1, b.page, c.hd, codes + (page0 + h) * size, scale + page0 + h, red);
  } else {
    const int h0 = 4 * blockIdx.y, h1 = min(h0 + 4, c.kv_heads);
    if ((o1 - o0) * c.hd <= 256) {
      const int h = h0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
      if (h < h1)
        append_few<IS_V, 1>(x + h * c.hd, ld, o0, o1, b.page, c.hd, codes + (page0 + h) * size, scale + page0 + h, red);
      return;
    }
    for (int h = h0; h < h1; ++h) {
      append_head<IS_V, U, W>(x + h * c.hd, ld, o0, o1, b.page, c.hd, codes + (page0 + h) * size, scale + page0 + h, red);
      __syncthreads();
    }
  }
}

template <int U, int W, bool FOUR>
__global__ __launch_bounds__(64 * W) void kv8_append_kernel(PagedBatch b, Kv8Cache c, const float* __restrict__ k, int ldk,
                                                            const float* __restrict__ v, int ldv) {
  __shared__ AppendRed red;
  if (blockIdx.z == 0) append_run<false, U, W, FOUR>(b, c, k, ldk, c.k, c.ks, red);
  else append_run<true, U, W, FOUR>(b, c, v, ldv, c.v, c.vs, red);
}

template <int U, int W, bool FOUR>
static void launch_append(const PagedBatch& b, const Kv8Cache& c, const float* k, int ldk, const float* v, int ldv,
                          hipStream_t s) {
  const dim3 grid((unsigned)(b.rows / b.page + 2 * b.requests), (unsigned)(FOUR ? (c.kv_heads + 3) / 4 : c.kv_heads), 2);
  hipLaunchKernelGGL((kv8_append_kernel<U, W, FOUR>), grid, dim3(64 * W), 0, s, b, c, k, ldk, v, ldv);
}

hipError_t launch_kv8_append(const PagedBatch& b, const Kv8Cache& c, const float* k, int ldk, const float* v, int ldv,
                             hipStream_t s) {
  const int units = b.page * c.hd / 16;
  // a token for each request at most on average: a wave per head, four to a workgroup (us of that / of a workgroup per head:
  // 64 tokens, 4 heads of 128 4.0 / 4.8 in the kernel, 1000, 8 of 128 18 / 47, 4000, 2 of 64 25 / 42: starting workgroups)
  if (b.rows <= b.requests) {
    if (units <= 256) launch_append<1, 4, true>(b, c, k, ldk, v, ldv, s);
    else if (units <= 512) launch_append<2, 4, true>(b, c, k, ldk, v, ldv, s);
    else if (units <= 1024) launch_append<4, 4, true>(b, c, k, ldk, v, ldv, s);
    else launch_append<0, 4, true>(b, c, k, ldk, v, ldv, s);
  } else {
    // more waves for large pages, not units in turn (us: chunks of 737 rows of 11 requests, 4 heads of 256, pages of 128 17 /
    // 26, of 300 of 4, 8 heads of 256, pages of 256 16 / 26); twice the waves with half the units each does as well
    if (units <= 256) launch_append<1, 4, false>(b, c, k, ldk, v, ldv, s);
    else if (units <= 512) launch_append<2, 4, false>(b, c, k, ldk, v, ldv, s);
    else if (units <= 1024) launch_append<4, 4, false>(b, c, k, ldk, v, ldv, s);
    else if (units <= 2048) launch_append<4, 8, false>(b, c, k, ldk, v, ldv, s);
    else launch_append<4, 16, false>(b, c, k, ldk, v, ldv, s);
  }
  return hipGetLastError();
}

// ---- attention -----------------------------------------------------------------------------------
// Row i of request r stands at position p = len - count + i and sees the keys max(0, p - window + 1) .. p that lie
// in a page (none does behind the table): softmax over scale * q . k, then the weighted values. A row that sees no key gets zeros.
//
// All products run on v_mfma_f32_16x16x32_f16: an int8 code is exact in f16, and the f32 operands (q, the
// probabilities) are split into two f16 parts, hi + lo, good to 2^-22 of the largest: two instructions per product,
// f32 sums. q is first scaled by the power of two that takes its vector's largest element to 2^13 .. 2^14, so no part
// falls out of f16's range; the terms exp(s - m) are taken times 2^kTermBits, which cancels in the division by their
// sum. m is the vector's largest score so far or up to kSlack (in powers of 2) below it: sums are moved to a new m only
// when a score passes that, which after the first steps is rare. Each step's products with V's codes are summed from
// zero and scaled by the page's scale in f32 (scales taken into the f16 weights cost a row that sees only pages of small
// scale its precision).
//
// Measured, with the join: one row of 24 heads behind 131071 tokens (8 heads of 128, 268 MB) 49.0 us, 5.5 TB/s: HBM; 64
// requests of 1 .. 16384 tokens (4 heads of 128, 135 MB) 34.4 us, 30 of them here: HBM behind the first three trips to
// memory; one row of 14 heads, 211 tokens 9.6 us, 6.7 in the kernel: those trips. Prompts of 1000 rows behind up to 5000
// tokens (four, 32 heads of 128) 189 .. 194 us, 465 .. 475 TFLOP/s of products and as many again of low parts: 0.9 of the rate of a large
// f16 matrix product (1.06 PFLOP/s) on the matrix cores.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
constexpr float kTermBits = 10.0f, kSlack = 5.0f;     // 2^(10 + 5) stays below f16's 65504
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// eight codes as f16: 0x6400 + u is the f16 value 1024 + u for a byte u = c + 128, less 1152 is c
__device__ __forceinline__ h8 codes8(unsigned a, unsigned b) {
  union { unsigned u[4]; h2 h[4]; h8 v; } r;
  a ^= 0x80808080u;
  b ^= 0x80808080u;
  r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
  r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
  r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
  r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
  const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
#pragma unroll
  for (int i = 0; i < 4; ++i) r.h[i] += off;
  return r.v;
}

// x = hi + lo, each rounded to the nearest f16. minus_one: -1, but unknown to the compiler, which then subtracts hi in
// one mixed-precision fma instead of converting it back first
__device__ __forceinline__ void split8(const float (&x)[8], float minus_one, h8& hi, h8& lo) {
  union { h2 h[4]; h8 v; } a, b;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a.h[i] = __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), h2);
    const f32x2 r = {__builtin_fmaf((float)a.h[i][0], minus_one, x[2 * i]),
                     __builtin_fmaf((float)a.h[i][1], minus_one, x[2 * i + 1])};
    b.h[i] = __builtin_convertvector(r, h2);
  }
  hi = a.v;
  lo = b.v;
}

// 2^x for x <= 16: what is below the smallest normal float may come out as 0
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// the largest over the four lanes that share a column of the 16 x 16 layouts (one of the swapped values is the lane's
// own, so both may be taken), and the sum
__device__ __forceinline__ float column_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  v += lane_xor<16>(v);
  return v + lane_xor<32>(v);
}

// How a launch cuts the batch: a tile holds up to vecs query vectors of one request and KV head, rows_per rows of its
// grp heads (grp <= vecs), or vecs of the grp heads of one row (group_tiles of them).
//   direct: no request has more than one tile. Its keys are cut into pieces of about the same size over all requests,
//     `pieces` of them in all (and one more for each request), of at least kAttnMinSteps steps: a batch of lengths 1 ..
//     16384 then takes the time of its sum, not of its longest request. Up to kAttnScanned requests every workgroup finds
//     its piece from all the lengths; of more a launch before lists them (listed, at float `list` of the workspace), and with
//     16 vectors a tile of short contexts a wave takes a piece alone, four to a workgroup (solo).
//   else: unit u is a tile, every tile is cut into `splits` pieces.
// A head's pieces have `slots` places in the workspace, a tile's one behind the other, each of `used` vectors.
struct AttnTiles {
  int vecs, grp, rows_per, group_tiles, units, direct, splits, pieces, slots, used, listed, solo;
  size_t list;
};

// A tile's place: request, rows, and the 32-key steps it has to walk, and their cut into splits.
struct AttnTile {
  int req, row0, n, i0, i1;  // request, its first row, its rows, the tile's rows i0 .. i1 - 1 of them
  int p0;                    // position of the request's row 0 (may be below 0)
  int first, steps, per;     // first step, number of steps, steps per split
  int slot;                  // its first place in the workspace
};

constexpr int kAttnMaxSplits8 = 256;  // one thread of the join each
constexpr int kAttnMinSteps = 16;     // steps of a split, at least (four waves take turns)
constexpr int kAttnScanned = 256;     // one thread of a workgroup each

// rows i0 .. of a request; false if it has none
__device__ __forceinline__ bool place_tile(const PagedBatch& b, const Attn8Args& a, const AttnTiles& t,
                                           const RequestRows& q, int i0, AttnTile& o) {
  o.req = q.req;
  o.row0 = q.row0;
  o.n = min(q.count, a.max_rows);
  o.p0 = max(q.len, 0) - q.count;
  o.i0 = i0;
  o.i1 = min(i0 + t.rows_per, o.n);
  const int last = min(o.p0 + o.i1, b.table_ld * b.page) - 1;      // (no key behind the table)
  const int lo = a.window > 0 ? max(0, o.p0 + i0 - a.window + 1) : 0;
  o.first = last < lo ? 0 : lo >> 5;
  o.steps = last < lo ? 0 : (last >> 5) - o.first + 1;
  return i0 >= 0 && i0 < o.n;
}
__device__ __forceinline__ bool place_request(const PagedBatch& b, const Attn8Args& a, const AttnTiles& t, int r,
                                              AttnTile& o) {
  return place_tile(b, a, t, request_rows(r, b.start[r], b.count[r], b.len[r], b.rows), 0, o);
}
__device__ __forceinline__ int steps_per(int steps, int pieces) {
  return max(kAttnMinSteps, ((steps + pieces - 1) / pieces + 3) & ~3);
}

// .. of a piece of the whole batch's sum over `live` requests. Their last pieces are half empty on average; while they are
// few that half is taken off, so that there are about `pieces` workgroups in all (us without / with: 64 requests of up to
// 16384, 4 heads of 128 38.8 / 35.4, 16 of up to 20000, 8 of 256 43.8 / 36.2; but 128 requests, 64 pieces a head 90 / 99,
// 48 of up to 32000, 64 69 / 82: the longest piece then comes last). A float sum is at most 2^-8 too small, and pieces
// that are too small in all would be more than the launch has workgroups for.
__device__ __forceinline__ int piece_steps(float sum, float live, int pieces) {
  const float n = 2.0f * live <= (float)pieces ? (float)pieces - 0.5f * live : (float)pieces;
  return max(kAttnMinSteps, ((int)fminf(ceilf(sum * 1.005f / n), 1e9f) + 3) & ~3);
}

// inclusive sums over the lanes of a wave
__device__ __forceinline__ int wave_scan(int v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(v, off, 64);
    if ((int)(threadIdx.x & 63) >= off) v += y;
  }
  return v;
}

// The sum over a workgroup of WAVES waves, and in `before` that of the threads below this one.
template <int WAVES>
__device__ __forceinline__ int scan_block(int v, int& before) {
  __shared__ int part[WAVES];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, inc = wave_scan(v);
  if (lane == 63) part[w] = inc;
  __syncthreads();
  int all = 0;
  before = inc - v;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    before += i < w ? part[i] : 0;
    all += part[i];
  }
  __syncthreads();
  return all;
}
// .. of floats, in one order
template <int WAVES>
__device__ __forceinline__ float sum_block(float v) {
  __shared__ float part[WAVES];
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float all = 0.0f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) all += part[i];
  __syncthreads();
  return all;
}

// The tile and split of workgroup `u` of a head; false if there is none.
__device__ __forceinline__ bool find_piece(const PagedBatch& b, const Attn8Args& a, const AttnTiles& t, int u,
                                           AttnTile& o, int& sp) {
  if (!t.direct) {
    sp = u / t.units;
    u = t.units - 1 - (u + sp) % t.units;             // (a prompt's last rows see the most keys: first)
    const RequestRows q = request_of_unit(u, b, t.rows_per, 1);
    if (q.req < 0 || !place_tile(b, a, t, q, (u - (q.row0 / t.rows_per + q.req)) * t.rows_per, o)) return false;
    o.per = steps_per(o.steps, t.splits);
    o.slot = u * t.splits;
    return sp == 0 || sp * o.per < o.steps;
  }
  // steps of a piece over the whole batch, then the request that piece u falls into: up to 64 requests a lane of every
  // wave each (nothing then goes through LDS), else one for each thread
  if (b.requests <= 64) {
    const int i = threadIdx.x & 63, r = min(i, b.requests - 1);
    const RequestRows q = request_rows(r, b.start[r], b.count[r], b.len[r], b.rows);
    const bool has = place_tile(b, a, t, q, 0, o) && i < b.requests;
    const int piece = piece_steps(wave_sum(has ? (float)o.steps : 0.0f), (float)__popcll(__ballot(has)), t.pieces);
    const int per = max(piece, steps_per(o.steps, t.splits));
    const int mine = has ? max(1, (o.steps + per - 1) / per) : 0, upto = wave_scan(mine);
    const unsigned long long at = __ballot(u < upto);
    if (at == 0) return false;
    const int l = __ffsll(at) - 1;
    place_tile(b, a, t, lane_rows(q, l), 0, o);
    o.per = __builtin_amdgcn_readlane(per, l);
    sp = u - __builtin_amdgcn_readlane(upto - mine, l);
    o.slot = u - sp;
    return true;
  }
  if (t.listed) {
    const int4 e = reinterpret_cast<const int4*>(a.work + t.list)[u];
    if (e.x < 0) return false;
    place_request(b, a, t, e.x, o);
    o.per = e.z;
    sp = e.y;
    o.slot = u - sp;
    return true;
  }
  __shared__ AttnTile found;
  __shared__ int found_sp;
  const int i = threadIdx.x;
  const bool has = place_request(b, a, t, min(i, b.requests - 1), o) && i < b.requests;
  const float sum = sum_block<4>(has ? (float)o.steps : 0.0f), live = sum_block<4>(has ? 1.0f : 0.0f);
  o.per = max(piece_steps(sum, live, t.pieces), steps_per(o.steps, t.splits));
  const int mine = has ? max(1, (o.steps + o.per - 1) / o.per) : 0;
  int before;
  if (u >= scan_block<4>(mine, before)) return false;
  if (u >= before && u < before + mine) {
    found = o;
    found_sp = u - before;
  }
  __syncthreads();
  o = found;
  sp = found_sp;
  o.slot = u - sp;
  return true;
}

// The list of pieces of a large batch: {request, split, steps per split} for each, request -1 behind the last. One
// workgroup, every thread some requests that follow one another.
__global__ __launch_bounds__(1024) void attention_kv8_pieces_kernel(PagedBatch b, Attn8Args a, AttnTiles t) {
  int4* const list = reinterpret_cast<int4*>(a.work + t.list);
  const int chunk = (b.requests + 1023) / 1024, r0 = threadIdx.x * chunk, r1 = min(r0 + chunk, b.requests);
  AttnTile o;
  float sum = 0.0f, live = 0.0f;
  for (int r = r0; r < r1; ++r)
    if (place_request(b, a, t, r, o)) {
      sum += (float)o.steps;
      live += 1.0f;
    }
  sum = sum_block<16>(sum);
  live = sum_block<16>(live);
  const int piece = piece_steps(sum, live, t.pieces);
  auto pieces_of = [&](int r, int& per) {
    if (!place_request(b, a, t, r, o)) return 0;
    per = max(piece, steps_per(o.steps, t.splits));
    return max(1, (o.steps + per - 1) / per);
  };
  int mine = 0, per = 0, at;
  for (int r = r0; r < r1; ++r) mine += pieces_of(r, per);
  const int all = scan_block<16>(mine, at);
  for (int r = r0; r < r1; ++r) {
    const int n = pieces_of(r, per);
    for (int sp = 0; sp < n; ++sp, ++at)
      if (at < t.slots) list[at] = make_int4(r, sp, per, 0);
  }
  for (int u = all + threadIdx.x; u < t.slots; u += 1024) list[u] = make_int4(-1, 0, 0, 0);
}

// The workspace holds (m, l) of every vector of every piece, then (16-byte aligned) their sums, then every unit's number
// of splits and first place, then the list of pieces.
__host__ __device__ inline size_t piece_vectors(const AttnTiles& t, int kv_heads) {
  return (size_t)kv_heads * t.group_tiles * t.slots * t.used;
}
__host__ __device__ inline size_t sums_at(size_t vectors) { return (2 * vectors + 3) & ~(size_t)3; }
// place of split 0, vector 0 of a tile's head and group yy
__device__ __forceinline__ size_t place_of(const AttnTiles& t, const AttnTile& tile, int yy) {
  return ((size_t)yy * t.slots + tile.slot) * t.used;
}

// the same in every lane, so that what follows from it is scalar
__device__ __forceinline__ AttnTile uniform(const AttnTile& o) {
  auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  return {u(o.req), u(o.row0), u(o.n), u(o.i0), u(o.i1), u(o.p0), u(o.first), u(o.steps), u(o.per), u(o.slot)};
}

__device__ __forceinline__ int2* splits_at(const Attn8Args& a, const AttnTiles& t, int kv_heads, int hd) {
  const size_t n = piece_vectors(t, kv_heads);
  return reinterpret_cast<int2*>(a.work + sums_at(n) + n * hd);
}

constexpr int kAttnPages = 256;       // pages whose numbers and scales are staged at a time: one per thread

// One workgroup of four waves per (tile, KV head, split of the keys). A wave takes every fourth step of 32 keys, for
// VT groups of 16 query vectors:
//   S^T = K Q^T (two 16-key tiles; lane l has keys 4 (l / 16) + i of each for vector l % 16), the running maximum
//   and sum, and O^T += V^T P^T, whose operand P^T is what the lane holds of S^T.
// Codes go from memory to registers in fragment order: 16 bytes per lane and 1 KiB per load, no LDS. The next K block
// loads while the softmax and V's products run, the next V block while K's do. With one group its q stays in
// registers; with more (prompts) the groups' q lies in LDS, in fragment order too, and every code is converted to f16
// once for all of them.
// SOLO (listed pieces, one group): every wave its own piece, no joins between waves.
template <int NB, int VT, bool SOLO>
__global__ __launch_bounds__(256) void attention_kv8_kernel(PagedBatch b, Kv8Cache c, Attn8Args a, AttnTiles t) {
  constexpr int HD = 32 * NB, LD = HD + 4, kW = SOLO ? 1 : 4, kPages = SOLO ? kAttnPages / 4 : kAttnPages;
  static_assert(!SOLO || VT == 1, "a wave alone has one group");
  __shared__ int all_ids[kAttnPages];
  __shared__ float all_kss[kAttnPages], all_vss[kAttnPages];
  __shared__ float Ms[4][16], Ls[4][16];
  constexpr size_t kQ = VT > 1 ? (size_t)VT * NB * 2 * 1024 : 0, kO = sizeof(float) * 4 * 16 * LD;
  __shared__ __attribute__((aligned(16))) char big[kQ > kO ? kQ : kO];    // q, and after the steps the waves' sums
  float (*Os)[16][LD] = reinterpret_cast<float (*)[16][LD]>(big);
  h8* const qf = reinterpret_cast<h8*>(big);                              // [VT][NB][hi, lo][lane]
  __shared__ float qss[VT][16];
  AttnTile tile;
  const int ht = c.kv_heads * t.group_tiles, yy = blockIdx.x % ht;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w = SOLO ? 0 : wave, tid = SOLO ? lane : threadIdx.x;            // within the piece
  const int u = blockIdx.x / ht * (4 / kW) + (SOLO ? wave : 0);
  int sp;
  if (u >= t.slots || !find_piece(b, a, t, u, tile, sp)) return;
  int* const ids = all_ids + (SOLO ? kPages * wave : 0);
  float* const kss = all_kss + (SOLO ? kPages * wave : 0);
  float* const vss = all_vss + (SOLO ? kPages * wave : 0);
  auto sync = [] {
    if constexpr (SOLO) wave_sync();
    else __syncthreads();
  };
  tile = uniform(tile);
  sp = __builtin_amdgcn_readfirstlane(sp);
  const int head = yy / t.group_tiles, g0 = (yy % t.group_tiles) * t.vecs;
  const int col = lane & 15, g = lane >> 4;
  const int s0 = tile.first + sp * tile.per, s1 = min(s0 + tile.per, tile.first + tile.steps);
  // every vector of the tile sees the keys see_from .. see_all (a place without one may see anything: it is not stored)
  const int see_all = tile.p0 + tile.i0, see_from = a.window > 0 ? tile.p0 + tile.i1 - a.window : 0;
  // vector col of group v: row and head, the last key it sees (-1: no such vector)
  auto row_of = [&](int vec) { return t.grp <= t.vecs ? tile.i0 + vec / t.grp : tile.i0; };
  auto head_of = [&](int vec) { return t.grp <= t.vecs ? vec % t.grp : g0 + vec; };
  int pos[VT];
#pragma unroll
  for (int v = 0; v < VT; ++v)
    pos[v] = row_of(16 * v + col) < tile.i1 && head_of(16 * v + col) < t.grp ? tile.p0 + row_of(16 * v + col) : -1;
  const size_t head_bytes = (size_t)b.page * HD;
  const int page_steps = b.page >> 5, page0 = s0 / page_steps, page_last = max(s1 - 1, 0) / page_steps;
  const unsigned page_inv = 65536u / page_steps + 1;
  auto entry = [&](int pg) {
    const int pid = b.table[(size_t)tile.req * b.table_ld + pg];
    return pid >= 0 && pid < b.n_pages ? pid : -1;
  };
  auto block = [&](const int8_t* base, int pid, int in_page) {     // (an absent page: any one, its scores are hidden)
    return base + ((size_t)__builtin_amdgcn_readfirstlane(max(pid, 0)) * c.kv_heads + head) * head_bytes +
           (size_t)in_page * (NB * 1024);
  };
  // (a decode step reads every code once, tiles of 32 and 64 vectors read them again, from L2: us of nontemporal / plain
  // loads for one row behind 131071 tokens 50 / 56, 64 requests of up to 16384 36 / 35. Prompts in tiles of 16 take either: 961
  // rows of 14 heads in 2 of 64 16.4 / 16.5, behind 4000 tokens 69 / 70.6, 100 of 32 in 8 of 128 behind 1000 21.7 / 21.7)
  auto load = [&](const int8_t* p, u32x4 (&x)[NB]) {
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const u32x4* at = reinterpret_cast<const u32x4*>(p + 1024 * k + 16 * lane);
      x[k] = VT > 1 ? *at : __builtin_nontemporal_load(at);
    }
  };
  // the wave's first block straight from the table, and the pages this thread stages: on their way while q is split
  u32x4 kf[NB], vf[NB];
  const int first = max(min(s0 + w, s1 - 1), 0);
  int my_page = entry(min(page0 + tid, page_last));
  {
    const int pid = entry(first / page_steps), in_page = first - first / page_steps * page_steps;
    load(block(c.k, pid, in_page), kf);
    load(block(c.v, pid, in_page), vf);
  }
  float my_ks = c.ks[(size_t)max(my_page, 0) * c.kv_heads + head], my_vs = c.vs[(size_t)max(my_page, 0) * c.kv_heads + head];
  float minus_one = -1.0f;
  asm volatile("" : "+v"(minus_one));
  h8 qh[NB], ql[NB];
  float qs = 0.0f;
#pragma unroll
  for (int v = 0; v < VT; ++v) {
    if (VT > 1 && v % 4 != w) continue;                            // (a wave each)
    const bool live = row_of(16 * v + col) < tile.i1 && head_of(16 * v + col) < t.grp;
    const float* q = a.q + (size_t)(tile.row0 + (live ? row_of(16 * v + col) : tile.i0)) * a.ldq +
                     (size_t)(head * t.grp + (live ? head_of(16 * v + col) : 0)) * HD + 8 * g;
    float x[NB][8];
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      *reinterpret_cast<float4*>(&x[k][0]) = *reinterpret_cast<const float4*>(q + 32 * k);
      *reinterpret_cast<float4*>(&x[k][4]) = *reinterpret_cast<const float4*>(q + 32 * k + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[k][j]) & 0x7fffffffu);
    }
    top = max(top, lane_xor_u32<16>(top));
    top = max(top, lane_xor_u32<32>(top));
    const int e = (int)(top >> 23);                               // 2^13 <= largest * 2^(f - 127) < 2^14
    const int f = e == 255 ? 127 : min(267 - e, 253);
    const float up = copysignf(__uint_as_float((unsigned)f << 23), a.scale);   // (scores' factor is then positive)
    qs = __uint_as_float((unsigned)(254 - f) << 23) * (fabsf(a.scale) * 1.4426950408889634f);
#pragma unroll
    for (int k = 0; k < NB; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[k][j] *= up;
      split8(x[k], minus_one, qh[k], ql[k]);
      if (VT > 1) {
        qf[((v * NB + k) * 2 + 0) * 64 + lane] = qh[k];
        qf[((v * NB + k) * 2 + 1) * 64 + lane] = ql[k];
      }
    }
    if (VT > 1 && g == 0) qss[v][col] = qs;
  }
  if (VT > 1) __syncthreads();
  float qsv[VT], m[VT], l[VT];
  f32x4 o[VT][NB][2];
#pragma unroll
  for (int v = 0; v < VT; ++v) {
    qsv[v] = VT > 1 ? qss[v][col] : qs;
    m[v] = -INFINITY;
    l[v] = 0.0f;
#pragma unroll
    for (int k = 0; k < NB; ++k) o[v][k][0] = o[v][k][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  bool huge = false;                     // some vector's m is beyond 2^20
  for (int pg0 = page0; pg0 * page_steps < s1; pg0 += kPages) {
    // the pages of these steps: their numbers and scales
    if (pg0 != page0) {
      my_page = entry(min(pg0 + tid, page_last));
      my_ks = c.ks[(size_t)max(my_page, 0) * c.kv_heads + head];
      my_vs = c.vs[(size_t)max(my_page, 0) * c.kv_heads + head];
      sync();                            // the pages before have been read
    }
    ids[tid] = my_page;
    kss[tid] = my_page >= 0 ? my_ks : 0.0f;
    vss[tid] = my_page >= 0 ? my_vs : 0.0f;
    sync();
    // steps from here on count from page pg0's first (below kAttnPages * 8): the quotient by page_steps is exact
    const int c0 = pg0 * page_steps, e0 = max(s0 - c0, 0), e1 = min(s1 - c0, kPages * page_steps);
    auto page_of = [&](int s) { return (int)((unsigned)s * page_inv >> 16); };
    auto next_block = [&](const int8_t* base, int s) {
      const int pi = page_of(s);
      return block(base, ids[pi], s - pi * page_steps);
    };
    int s = e0 + w;
    if (pg0 != page0 && s < e1) {
      load(next_block(c.k, s), kf);
      load(next_block(c.v, s), vf);
    }
    for (; s < e1; s += kW) {
      const int next = min(s + kW, e1 - 1);
      const int pi = page_of(s), key0 = 32 * (s + c0);
      const bool have = ids[pi] >= 0;
      const float ks = kss[pi], vs = vss[pi];
      f32x4 st[VT][2] = {};
      int at = lane;                     // (q is read in every step: held in registers it costs a SIMD its third wave)
      if (VT > 1) asm volatile("" : "+v"(at));
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const h8 k0 = codes8(kf[k][0], kf[k][1]), k1 = codes8(kf[k][2], kf[k][3]);
#pragma unroll
        for (int v = 0; v < VT; ++v) {
          const h8 hi = VT > 1 ? qf[((v * NB + k) * 2 + 0) * 64 + at] : qh[k];
          const h8 lo = VT > 1 ? qf[((v * NB + k) * 2 + 1) * 64 + at] : ql[k];
          st[v][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, hi, st[v][0], 0, 0, 0);
          st[v][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, hi, st[v][1], 0, 0, 0);
          st[v][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, lo, st[v][0], 0, 0, 0);
          st[v][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, lo, st[v][1], 0, 0, 0);
        }
      }
      load(next_block(c.k, next), kf);
      // f > 0, so the largest product is the largest score (0 would make NaN of the hidden ones' -inf)
      float f[VT], mx[VT];
      const bool hides = !have || key0 + 31 > see_all || key0 < see_from;      // some vector does not see some key
      if (hides) {
#pragma unroll
        for (int v = 0; v < VT; ++v) {
          const int low = a.window > 0 ? pos[v] - a.window + 1 : 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int j = key0 + 16 * (e >> 2) + 4 * g + (e & 3);
            if (!have || j > pos[v] || j < low) st[v][e >> 2][e & 3] = -INFINITY;
          }
        }
      }
      bool rises = false;
#pragma unroll
      for (int v = 0; v < VT; ++v) {
        f[v] = fmaxf(ks * qsv[v], 1.17549435e-38f);
        const f32x4 y = st[v][0], z = st[v][1];
        mx[v] = column_max(fmaxf(fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(z[0], z[1])), fmaxf(z[2], z[3]))) *
                f[v];
        rises |= mx[v] > m[v] + kSlack;
      }
      if (__ballot(rises) != 0) {
        bool far = false;
#pragma unroll
        for (int v = 0; v < VT; ++v) {
          const float mn = fmaxf(m[v], mx[v]);
          const float alpha = mn == -INFINITY ? 1.0f : pow2(m[v] - mn);
          l[v] *= alpha;
#pragma unroll
          for (int k = 0; k < NB; ++k) { o[v][k][0] *= alpha; o[v][k][1] *= alpha; }
          m[v] = mn;
          far |= fabsf(mn) > 1048576.0f && mn != -INFINITY;
        }
        huge = __ballot(far) != 0;
      }
      if (huge) {                        // m's own rounding would come out of the fma below: products rounded as m was
#pragma unroll
        for (int v = 0; v < VT; ++v) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float y = st[v][e >> 2][e & 3] * f[v];
            asm volatile("" : "+v"(y));
            st[v][e >> 2][e & 3] = m[v] == -INFINITY ? y : y - m[v];
          }
          f[v] = 1.0f;
        }
      }
      h8 ph[VT], pl[VT];
#pragma unroll
      for (int v = 0; v < VT; ++v) {
        const float off = m[v] == -INFINITY || huge ? kTermBits : kTermBits - m[v];
        float x[8], ps = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = pow2(__builtin_fmaf(st[v][e >> 2][e & 3], f[v], off));
          ps += x[e];
        }
        l[v] += ps;
        split8(x, minus_one, ph[v], pl[v]);
      }
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const h8 v0 = codes8(vf[k][0], vf[k][1]), v1 = codes8(vf[k][2], vf[k][3]);
#pragma unroll
        for (int v = 0; v < VT; ++v) {
          f32x4 y0 = {}, y1 = {};
          y0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[v], y0, 0, 0, 0);
          y1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[v], y1, 0, 0, 0);
          y0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[v], y0, 0, 0, 0);
          y1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[v], y1, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[v][k][0][i] = __builtin_fmaf(y0[i], vs, o[v][k][0][i]);
            o[v][k][1][i] = __builtin_fmaf(y1[i], vs, o[v][k][1][i]);
          }
        }
      }
      load(next_block(c.v, next), vf);
    }
  }
  // the waves' (m, l, O) joined in wave order, group after group
  const bool whole = tile.steps <= tile.per;                      // one split: nothing left to join
  if (t.splits > 1 && sp == 0 && yy == 0 && tid == 0)
    splits_at(a, t, c.kv_heads, HD)[t.direct ? tile.req : tile.row0 / t.rows_per + tile.req + tile.i0 / t.rows_per] =
        make_int2((tile.steps + tile.per - 1) / tile.per, tile.slot);
  const size_t place = place_of(t, tile, yy) + (size_t)sp * t.used;
  float* const sums = a.work + sums_at(piece_vectors(t, c.kv_heads));
  const int first_wave = SOLO ? wave : 0;
#pragma unroll
  for (int v = 0; v < VT; ++v) {
    const float lv = column_sum(l[v]);
    if (VT > 1) __syncthreads();                                   // q, or the group before, has been read
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float4*>(&Os[wave][col][32 * k + 16 * h + 4 * g]) =
            make_float4(o[v][k][h][0], o[v][k][h][1], o[v][k][h][2], o[v][k][h][3]);
    if (g == 0) { Ms[wave][col] = m[v]; Ls[wave][col] = lv; }
    sync();
#pragma unroll
    for (int vec = tid >> 4; vec < 16; vec += 4 * kW) {
      const int oi = row_of(16 * v + vec), oh = head_of(16 * v + vec);
      if (oi >= tile.i1 || oh >= t.grp) continue;
      float M = Ms[first_wave][vec];
#pragma unroll
      for (int k = 1; k < kW; ++k) M = fmaxf(M, Ms[k][vec]);
      float f[kW], L = 0.0f;
#pragma unroll
      for (int k = 0; k < kW; ++k) {
        // (a wave that saw nothing: m = -inf, l = 0 and O = 0, unless the vector holds NaN)
        const float mk = Ms[first_wave + k][vec];
        f[k] = mk == M ? 1.0f : pow2(mk - M);
        L = __builtin_fmaf(Ls[first_wave + k][vec], f[k], L);
      }
      const size_t at = (size_t)(tile.row0 + oi) * a.heads + (size_t)head * t.grp + oh, mine = place + 16 * v + vec;
      const float inv = whole ? (L == 0.0f ? 0.0f : 1.0f / L) : 1.0f;
      float* out = whole ? a.ctx + at * HD : sums + mine * HD;
      for (int d = 4 * (tid & 15); d < HD; d += 64) {
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kW; ++k) {
          const float4 x = *reinterpret_cast<const float4*>(&Os[first_wave + k][vec][d]);
          y.x = __builtin_fmaf(x.x, f[k], y.x);
          y.y = __builtin_fmaf(x.y, f[k], y.y);
          y.z = __builtin_fmaf(x.z, f[k], y.z);
          y.w = __builtin_fmaf(x.w, f[k], y.w);
        }
        *reinterpret_cast<float4*>(out + d) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
      }
      if (!whole && (tid & 15) == 0) {
        a.work[2 * mine] = M;
        a.work[2 * mine + 1] = L;
      }
    }
  }
}

// The tile of workgroup blockIdx.x (.y: head and group of vectors) and its number of splits; false if there are none to
// join.
__device__ __forceinline__ bool find_joint(const PagedBatch& b, const Kv8Cache& c, const Attn8Args& a, const AttnTiles& t,
                                           AttnTile& tile, int& n) {
  const int2 at = splits_at(a, t, c.kv_heads, c.hd)[blockIdx.x];  // (no tile: not written, and not used)
  n = at.x;
  bool has;
  if (t.direct) {
    has = place_request(b, a, t, blockIdx.x, tile);
  } else {
    const RequestRows q = request_of_unit(blockIdx.x, b, t.rows_per, 1);
    has = q.req >= 0 && place_tile(b, a, t, q, ((int)blockIdx.x - (q.row0 / t.rows_per + q.req)) * t.rows_per, tile);
  }
  tile.slot = at.y;
  return has && n > 1;
}

// Joins splits: M = max m_s, out = sum O_s 2^(m_s - M) / sum l_s 2^(m_s - M). Up to kJoinFew splits: one workgroup per tile
// and head, a thread per vector and four dimensions (a workgroup per vector, as below, cost 502 tiles of 28 vectors and
// two splits 30 us of 48).
constexpr int kJoinFew = 32;

__global__ __launch_bounds__(256) void attention_kv8_join_few_kernel(PagedBatch b, Kv8Cache c, Attn8Args a, AttnTiles t) {
  AttnTile tile;
  int n;
  if (!find_joint(b, c, a, t, tile, n)) return;
  const int head = blockIdx.y / t.group_tiles, g0 = (blockIdx.y % t.group_tiles) * t.vecs;
  const int hd = c.hd, cols = hd >> 2;
  const size_t place = place_of(t, tile, blockIdx.y);
  const float* const sums = a.work + sums_at(piece_vectors(t, c.kv_heads));
  const int vecs = t.grp <= t.vecs ? (tile.i1 - tile.i0) * t.grp : min(t.vecs, t.grp - g0);
  for (int e = threadIdx.x; e < vecs * cols; e += 256) {
    const int vec = e / cols, col = e - vec * cols;
    const int oi = t.grp <= t.vecs ? tile.i0 + vec / t.grp : tile.i0, oh = t.grp <= t.vecs ? vec % t.grp : g0 + vec;
    const size_t at = (size_t)(tile.row0 + oi) * a.heads + (size_t)head * t.grp + oh;
    const float2* ml = reinterpret_cast<const float2*>(a.work) + place + vec;
    const float* os = sums + (place + vec) * hd + 4 * col;
    float M = -INFINITY;
#pragma unroll 4
    for (int s = 0; s < n; ++s) M = fmaxf(M, ml[s * t.used].x);
    float L = 0.0f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float2 p = ml[s * t.used];
      const float f = p.x == M ? 1.0f : pow2(p.x - M);
      const float4 x = *reinterpret_cast<const float4*>(os + (size_t)s * t.used * hd);
      L = __builtin_fmaf(p.y, f, L);
      y.x = __builtin_fmaf(x.x, f, y.x);
      y.y = __builtin_fmaf(x.y, f, y.y);
      y.z = __builtin_fmaf(x.z, f, y.z);
      y.w = __builtin_fmaf(x.w, f, y.w);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    *reinterpret_cast<float4*>(a.ctx + at * hd + 4 * col) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
  }
}

// More splits (few tiles then): a workgroup per vector, a thread per split for its weight; then 256 / (hd / 4) groups of
// threads add every so-manieth split, and their sums are added in order.
__global__ __launch_bounds__(256) void attention_kv8_join_kernel(PagedBatch b, Kv8Cache c, Attn8Args a, AttnTiles t) {
  __shared__ float f[kAttnMaxSplits8], red[2][4];
  __shared__ float4 part[256];
  AttnTile tile;
  int n;
  if (!find_joint(b, c, a, t, tile, n)) return;
  const int tid = threadIdx.x, w = tid >> 6, vec = blockIdx.z, hd = c.hd;
  const int head = blockIdx.y / t.group_tiles, g0 = (blockIdx.y % t.group_tiles) * t.vecs;
  const int oi = t.grp <= t.vecs ? tile.i0 + vec / t.grp : tile.i0, oh = t.grp <= t.vecs ? vec % t.grp : g0 + vec;
  if (oi >= tile.i1 || oh >= t.grp) return;
  const size_t at = (size_t)(tile.row0 + oi) * a.heads + (size_t)head * t.grp + oh;
  const size_t place = place_of(t, tile, blockIdx.y) + vec;
  const float2 mine = reinterpret_cast<const float2*>(a.work)[place + (size_t)min(tid, n - 1) * t.used];
  const float m = tid < n ? mine.x : -INFINITY;
  float l = tid < n ? mine.y : 0.0f, M = m;
  M = wave_max(M);
  if ((tid & 63) == 0) red[0][w] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float fs = m == M ? 1.0f : pow2(m - M);
  f[tid] = fs;
  l *= fs;
  l = wave_sum(l);
  if ((tid & 63) == 0) red[1][w] = l;
  __syncthreads();
  const float L = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const int cols = hd >> 2, groups = 256 / cols;
  const int col = tid % cols, grp = tid / cols;
  const float* os = a.work + sums_at(piece_vectors(t, c.kv_heads)) + place * hd + 4 * col;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  if (grp < groups) {
#pragma unroll 4
    for (int s = grp; s < n; s += groups) {
      const float4 x = *reinterpret_cast<const float4*>(os + (size_t)s * t.used * hd);
      y.x = __builtin_fmaf(x.x, f[s], y.x);
      y.y = __builtin_fmaf(x.y, f[s], y.y);
      y.z = __builtin_fmaf(x.z, f[s], y.z);
      y.w = __builtin_fmaf(x.w, f[s], y.w);
    }
  }
  part[tid] = y;
  __syncthreads();
  if (tid >= cols) return;
  for (int k = 1; k < groups; ++k) {
    const float4 x = part[k * cols + tid];
    y.x += x.x;
    y.y += x.y;
    y.z += x.z;
    y.w += x.w;
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  *reinterpret_cast<float4*>(a.ctx + at * hd + 4 * tid) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
}

// the most groups of 16 vectors of a tile: their sums, 64 and 128 registers, leave a SIMD two waves
constexpr int most_groups(int hd) { return hd <= 128 ? 4 : 2; }

// (a window only ever makes the workspace smaller)
static AttnTiles attn_tiles(int rows, int requests, int max_rows, int max_len, int window, int heads, int kv_heads,
                            int hd) {
  AttnTiles t;
  t.grp = heads / kv_heads;
  const long vecs = (long)max_rows * t.grp;
  // Wide tiles convert a code once for all their vectors, but there are fewer of them and each starts and ends later. They
  // pay where more than half of a tile is filled and
  //   - tiles stay at four for each CU (us of 16 / 32 / 64 vectors: 2000 rows of 32 heads in 4 of 128 116 / 89 / 92, behind
  //     20000 tokens 1632 / 1307 / 1191; but 1000 rows of 14 in 2 of 64, 502 tiles of 32, 15.8 / 24.9 / 29.2), or
  //   - one tile holds all of a request, cut into pieces, and there is work for many of them (4 rows of 8 heads: 64
  //     requests of up to 4000 tokens 47.8 / 32.3 / 41.4, 8 requests of up to 3000 19.2 / 24.5 / 29.6 for 3 rows).
  for (int groups = most_groups(hd); groups > 0; groups >>= 1) {
    t.vecs = 16 * groups;
    t.rows_per = t.grp <= t.vecs ? std::min(t.vecs / t.grp, max_rows) : 1;
    t.group_tiles = (t.grp + t.vecs - 1) / t.vecs;
    t.direct = max_rows <= t.rows_per;
    t.units = t.direct ? requests : rows / t.rows_per + requests;
    const long tiles = (long)t.units * kv_heads * t.group_tiles;
    if (2 * vecs > t.vecs && (t.direct ? (long)requests * kv_heads * (max_len / 32) >= 16384 : tiles >= 1024)) break;
  }
  const long ht = (long)kv_heads * t.group_tiles;
  t.listed = t.direct && requests > kAttnScanned;
  // A wave for each short request where there are enough of them: most of a workgroup's four waves would have no step, but a
  // wave alone takes four times as long (us of a wave / four: 1000 requests of up to 64 tokens, 8 heads of 128 39 / 79, of up
  // to 500 74 / 96, 300 of up to 64, 4 heads 15.2 / 20.5; but of up to 500 27 / 24, 500 of up to 500, 2 of 64 21 / 16, 1000 of
  // up to 4096, 8 of 128 268 / 247)
  t.solo = t.listed && t.vecs == 16 && max_len <= 2048 && requests * ht >= 4L * max_len;
  long steps = (std::max(max_len, 1) + 31) / 32;                   // of the longest tile
  if (window > 0) steps = std::min(steps, ((long)window + t.rows_per - 2) / 32 + 2);
  // two workgroups of a piece for each CU, four of heads up to 64, whose steps are half as many bytes on their way (us of
  // 512 / 1024 / 1536: one request of 131071 tokens, 8 heads of 128 50.5 / 53.7 / 56, 64 of up to 16384, 4 of 128 35.4 /
  // 41 / 42; but one of 131071, 2 of 64 17.5 / 16.8 / 16.8, 128 of up to 8000, 4 of 64 32.7 / 24.4 / 26.7, 300, 2 of 32
  // 31.5 / 24.4 / 25.0)
  t.pieces = (int)std::max(1L, (hd <= 64 ? 1024 : 512) * (t.solo ? 4 : 1) / ht);
  // Prompts' tiles are cut into about three pieces for each CU; a cut in two that makes more than two for each CU does not pay
  // (us of 1024 / 768 / 512: three prompts of 77 rows behind 1500 tokens, 8 heads of 128, 264 tiles 24.5 / 22.8 / 18.7, 50
  // rows each behind 4000 of 4, 12 heads of 64, 192 tiles 18.2 / 18.7 / 19.3, 100 behind 20000, 104 tiles 45.8 / 45.0 / 48.8)
  const long tiles = t.units * ht, cuts = t.direct ? t.pieces : tiles <= 256 ? 768 / tiles : 512 / tiles;
  const long n = std::min({(steps + kAttnMinSteps - 1) / kAttnMinSteps, cuts, (long)kAttnMaxSplits8});
  // The second launch takes 4 .. 6 us, a step of 32 keys about hd / 170 us of a wave: cut if it takes more than that off (us
  // whole / cut: one row, 8 heads of 128, 544 tokens 11.1 / 13.6, 1024 13.5 / 14.1; 4 heads, 1500 17.6 / 14.4; 100 rows, 8
  // heads of 128, 1000 tokens 15.4 / 20.4; one row, 8 heads of 256, 902 tokens 20.6 / 17.4)
  t.splits = n > 1 && steps * hd * (n - 1) > 2816 * n ? (int)n : 1;
  t.slots = t.direct ? t.pieces + requests : t.units * t.splits;
  t.used = t.grp <= t.vecs ? t.rows_per * t.grp : t.vecs;
  const size_t vectors = piece_vectors(t, kv_heads);
  t.list = t.splits > 1 ? (sums_at(vectors) + vectors * hd + 2 * (size_t)t.units + 3) & ~(size_t)3 : 0;
  return t;
}

static size_t attn_workgroups(const AttnTiles& t, int kv_heads) {
  return (size_t)kv_heads * t.group_tiles * (t.solo ? (t.slots + 3) / 4 : t.slots);
}

size_t attention_kv8_workgroups(int rows, int requests, int max_rows, int max_len, int heads, int kv_heads, int hd) {
  return attn_workgroups(attn_tiles(rows, requests, max_rows, max_len, 0, heads, kv_heads, hd), kv_heads);
}

size_t attention_kv8_work_floats(int rows, int requests, int max_rows, int max_len, int heads, int kv_heads, int hd) {
  const AttnTiles t = attn_tiles(rows, requests, max_rows, max_len, 0, heads, kv_heads, hd);
  return t.list + (t.listed ? 4 * (size_t)t.slots : 0);
}

template <int NB>
static void launch_attention_hd(const PagedBatch& b, const Kv8Cache& c, const Attn8Args& a, const AttnTiles& t,
                                unsigned workgroups, hipStream_t s) {
  auto* k = t.solo ? attention_kv8_kernel<NB, 1, true> : t.vecs == 16 ? attention_kv8_kernel<NB, 1, false>
          : t.vecs == 32 ? attention_kv8_kernel<NB, 2, false> : attention_kv8_kernel<NB, most_groups(32 * NB), false>;
  hipLaunchKernelGGL(k, dim3(workgroups), dim3(256), 0, s, b, c, a, t);
}

hipError_t launch_attention_kv8(const PagedBatch& b, const Kv8Cache& c, const Attn8Args& a, hipStream_t s) {
  const AttnTiles t = attn_tiles(b.rows, b.requests, a.max_rows, a.max_len, a.window, a.heads, c.kv_heads, c.hd);
  const unsigned heads = (unsigned)(c.kv_heads * t.group_tiles);
  const unsigned n = (unsigned)attn_workgroups(t, c.kv_heads);
  if (t.listed) {
    hipLaunchKernelGGL(attention_kv8_pieces_kernel, dim3(1), dim3(1024), 0, s, b, a, t);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  switch (c.hd / 32) {
    case 1: launch_attention_hd<1>(b, c, a, t, n, s); break;
    case 2: launch_attention_hd<2>(b, c, a, t, n, s); break;
    case 3: launch_attention_hd<3>(b, c, a, t, n, s); break;
    case 4: launch_attention_hd<4>(b, c, a, t, n, s); break;
    case 5: launch_attention_hd<5>(b, c, a, t, n, s); break;
    case 6: launch_attention_hd<6>(b, c, a, t, n, s); break;
    case 7: launch_attention_hd<7>(b, c, a, t, n, s); break;
    default: launch_attention_hd<8>(b, c, a, t, n, s); break;
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || t.splits == 1) return e;
  if (t.splits <= kJoinFew) {
    hipLaunchKernelGGL(attention_kv8_join_few_kernel, dim3((unsigned)t.units, heads), dim3(256), 0, s, b, c, a, t);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(attention_kv8_join_kernel, dim3((unsigned)t.units, heads, (unsigned)t.used), dim3(256), 0, s, b, c, a,
                     t);
  return hipGetLastError();
}

}  // namespace rehip
