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

namespace rehip {

__device__ __forceinline__ int k_byte(int token, int dim) {
  return 16 * (16 * (dim >> 3) + (token & 15)) + 8 * (token >> 4) + (dim & 7);
}
__device__ __forceinline__ int v_byte(int token, int dim) {
  return 16 * (16 * ((token >> 2) & 3) + (dim & 15)) + 8 * (dim >> 4) + 4 * (token >> 4) + (token & 3);
}

// ---- append --------------------------------------------------------------------------------------
// A page and head's scale s is the largest finite magnitude of what it holds / 127 (0 below the smallest normal
// float: such values are stored as 0), a value's code round(x / s), ties to even. Rows that raise the scale of a
// page with earlier rows in it round those rows' codes to the new one: round(c * (s_old / s_new)). Infinities
// are stored as +-127 and NaN as 0, so that one bad value does not reach the page's other tokens.
__device__ __forceinline__ int code_of(float x, float s) {
  const float r = rintf(x / s);
  return x != x || s == 0.0f ? 0 : (int)fminf(fmaxf(r, -127.0f), 127.0f);
}

// One workgroup per (run of one request's new rows inside one page, head, K or V).
__global__ __launch_bounds__(256) void kv8_append_kernel(PagedBatch b, Kv8Cache c, const float* __restrict__ k,
                                                         size_t ldk, const float* __restrict__ v, size_t ldv) {
  __shared__ unsigned red[4];
  const int u = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  const bool is_v = blockIdx.z != 0;
  const int r = request_of_unit<256>(u, b.start, b.requests, b.rows, b.page, 2);
  if (r < 0) return;
  const int row0 = min(max(b.start[r], 0), b.rows);
  const int n = min(max(b.count[r], 0), b.rows - row0);
  const int len = b.len[r], first = len - n;
  if (n == 0 || first < 0 || len > b.table_ld * b.page) return;
  const int pi = first / b.page + (u - (row0 / b.page + 2 * r));
  const int lo = max(pi * b.page, first), hi = min((pi + 1) * b.page, len);   // positions
  if (lo >= hi) return;
  const int pid = b.table[(size_t)r * b.table_ld + pi];
  if (pid < 0 || pid >= b.n_pages) return;
  const int o0 = lo - pi * b.page, o1 = hi - pi * b.page, hd = c.hd;
  const size_t ld = is_v ? ldv : ldk;
  const float* x = (is_v ? v : k) + (size_t)(row0 + lo - first) * ld + (size_t)head * hd;
  int8_t* codes = (is_v ? c.v : c.k) + ((size_t)pid * c.kv_heads + head) * b.page * hd;
  float* scale = (is_v ? c.vs : c.ks) + (size_t)pid * c.kv_heads + head;
  const float s_old = o0 > 0 ? *scale : 0.0f;
  unsigned a = 0;
  for (int e = tid; e < (o1 - o0) * hd; e += 256) {
    const unsigned bits = __float_as_uint(x[(size_t)(e / hd) * ld + e % hd]) & 0x7fffffffu;
    if (bits < 0x7f800000u) a = max(a, bits);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) a = max(a, (unsigned)__shfl_xor((int)a, off, 64));
  if ((tid & 63) == 0) red[tid >> 6] = a;
  __syncthreads();
  a = max(max(red[0], red[1]), max(red[2], red[3]));
  float s = __uint_as_float(a) * (1.0f / 127.0f);
  if (s < 1.17549435e-38f) s = 0.0f;
  s = fmaxf(s, s_old);
  const float ratio = s > s_old ? s_old / s : 1.0f;
  const int t0 = ratio != 1.0f ? 0 : o0;       // old codes are touched only if the scale grew
  for (int e = t0 * hd + tid; e < o1 * hd; e += 256) {
    const int tok = e / hd, d = e % hd;
    int8_t* p = codes + (size_t)((tok >> 5) * (hd >> 5) + (d >> 5)) * 1024 +
                (is_v ? v_byte(tok & 31, d & 31) : k_byte(tok & 31, d & 31));
    *p = (int8_t)(tok < o0 ? (int)rintf((float)*p * ratio) : code_of(x[(size_t)(tok - o0) * ld + d], s));
  }
  if (tid == 0) *scale = s;
}

hipError_t launch_kv8_append(const PagedBatch& b, const Kv8Cache& c, const float* k, size_t ldk, const float* v,
                             size_t ldv, hipStream_t s) {
  const dim3 grid((unsigned)(b.rows / b.page + 2 * b.requests), (unsigned)c.kv_heads, 2);
  hipLaunchKernelGGL(kv8_append_kernel, grid, dim3(256), 0, s, b, c, k, ldk, v, ldv);
  return hipGetLastError();
}

// ---- attention -----------------------------------------------------------------------------------
// Row i of request r stands at position p = len - count + i and sees the keys max(0, p - window + 1) .. p that lie
// in a page: softmax over scale * q . k, then the weighted values. A row that sees no key gets zeros.
// One workgroup per (row, head): 256 keys at a time, a key per thread for the scores, a dimension per thread for the
// values.
__global__ __launch_bounds__(256) void attention_kv8_rows_kernel(PagedBatch b, Kv8Cache c, Attn8Args a) {
  __shared__ float qs[256], ps[256], red[4];
  __shared__ int pages[256];
  const int u = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, hd = c.hd;
  const int r = request_of_unit<256>(u, b.start, b.requests, b.rows, 1, 1);
  if (r < 0) return;
  const int row0 = min(max(b.start[r], 0), b.rows);
  const int n = min(max(b.count[r], 0), min(b.rows - row0, a.max_rows));
  const int i = u - (row0 + r);
  if (i < 0 || i >= n) return;
  const int len = min(max(b.len[r], 0), b.table_ld * b.page);
  const int p = len - min(max(b.count[r], 0), b.rows - row0) + i;
  const int head = h / (a.heads / c.kv_heads);
  if (tid < hd) qs[tid] = a.q[(size_t)(row0 + i) * a.ldq + (size_t)h * hd + tid];
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  const int first = a.window > 0 ? max(0, p - a.window + 1) : 0;
  for (int j0 = first; j0 <= p; j0 += 256) {
    const int j = j0 + tid;
    int pid = -1;
    if (j <= p) pid = b.table[(size_t)r * b.table_ld + j / b.page];
    if (pid < 0 || pid >= b.n_pages) pid = -1;
    __syncthreads();
    pages[tid] = pid;
    float s = -INFINITY;
    if (pid >= 0) {
      const int tok = j % b.page;
      const int8_t* kc = c.k + ((size_t)pid * c.kv_heads + head) * b.page * hd + (size_t)(tok >> 5) * (hd >> 5) * 1024;
      s = 0.0f;
      for (int d = 0; d < hd; ++d) s += qs[d] * (float)kc[(d >> 5) * 1024 + k_byte(tok & 31, d & 31)];
      s *= c.ks[(size_t)pid * c.kv_heads + head] * a.scale;
    }
    float mx = s;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float y = __shfl_xor(mx, off, 64);
      mx = y > mx || y != y ? y : mx;
    }
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    float mn = m;
#pragma unroll
    for (int w = 0; w < 4; ++w) mn = red[w] > mn || red[w] != red[w] ? red[w] : mn;
    const float alpha = m == mn ? 1.0f : expf(m - mn);
    const float e = pid < 0 ? 0.0f : expf(s - mn);
    ps[tid] = e;
    float sum = e;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    l = l * alpha + ((red[0] + red[1]) + (red[2] + red[3]));
    m = mn;
    o *= alpha;
    if (tid < hd) {
      const int d = tid;
      for (int t = 0; t < 256 && j0 + t <= p; ++t) {
        const int pg = pages[t];
        if (pg < 0) continue;
        const int tok = (j0 + t) % b.page;
        const int8_t* vc = c.v + ((size_t)pg * c.kv_heads + head) * b.page * hd;
        const float x = (float)vc[(size_t)((tok >> 5) * (hd >> 5) + (d >> 5)) * 1024 + v_byte(tok & 31, d & 31)];
        o += ps[t] * (x * c.vs[(size_t)pg * c.kv_heads + head]);
      }
    }
  }
  if (tid < hd) a.ctx[((size_t)(row0 + i) * a.heads + h) * hd + tid] = l == 0.0f ? 0.0f : o / l;
}

size_t attention_kv8_work_floats(int, int, int, int, int, int, int) { return 0; }

hipError_t launch_attention_kv8(const PagedBatch& b, const Kv8Cache& c, const Attn8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)(b.rows + b.requests), (unsigned)a.heads);
  hipLaunchKernelGGL(attention_kv8_rows_kernel, grid, dim3(256), 0, s, b, c, a);
  return hipGetLastError();
}

}  // namespace rehip
