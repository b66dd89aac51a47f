// What a cache of int8 pages is cut by: the weight that attention gives each token, added up over steps, and the move of the
// tokens that stay to fresh pages. The codes' layout is kv8.hip's.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv8.hpp"
#include "serve.hpp"
#include "wave.hpp"

namespace rehip {

// ---- weights of a step -----------------------------------------------------------------------------
// Key j of a request and KV head gets sum over its rows and the heads of the group of exp(scale q . k_j - lse), lse the log of
// the row's sum of exponentials as attention left it, over the rows that see the key. Products as in attention: codes exact in
// f16, q in two f16 parts, f32 sums. A key belongs to one wave, so its sum is taken in one order.
//
// A workgroup of four waves holds 128 KS keys of one head as f16 operands in registers, KS steps of 32 for each wave, and
// walks the query vectors that see some of them, 64 at a time (a tile of 16 for each wave to split, all four tiles for every
// wave to multiply). Sums over the 16 vectors of a tile stay in the lanes until the end.
struct MassCut {
  int chunks;                            // workgroups of a request and head
};

template <int NB, int KS>
__global__ __launch_bounds__(256) void kv8_mass_kernel(PagedBatch b, Kv8Cache c, MassArgs a, MassCut t) {
  constexpr int HD = 32 * NB, kKeys = 128 * KS;
  __shared__ __attribute__((aligned(16))) char big[4 * NB * 2 * 1024];
  h8* const qf = reinterpret_cast<h8*>(big);                       // [tile][NB][hi, lo][lane]
  __shared__ float qss[4][16], cut[4][16];                         // a vector's factor, its lse in powers of 2
  const int head = blockIdx.x % c.kv_heads, rest = blockIdx.x / c.kv_heads;
  const int req = rest / t.chunks;
  const RequestRows q = request_rows(req, b.start[req], b.count[req], b.len[req], b.rows);
  const int n = min(q.count, a.max_rows);
  if (n <= 0) return;
  const int grp = a.heads / c.kv_heads, p0 = max(q.len, 0) - q.count;
  const int last = min(p0 + n, b.table_ld * b.page) - 1;           // (no key behind the table)
  if (last < 0) return;
  const int lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
  const int sink_chunks = a.window > 0 ? (min(a.sinks, last + 1) + kKeys - 1) / kKeys : 0;
  const int first = max(lo / kKeys, sink_chunks), all = sink_chunks + max(last / kKeys - first + 1, 0);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4, page_steps = b.page >> 5;
  float minus_one = -1.0f;
  asm volatile("" : "+v"(minus_one));
  for (int ch = rest % t.chunks; ch < all; ch += t.chunks) {
    const int k0 = (ch < sink_chunks ? ch : ch - sink_chunks + first) * kKeys;
    // this wave's keys
    int pid[KS], in_page[KS];
    u32x4 kc[KS][NB];
    float ks[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int step = (k0 >> 5) + w * KS + s, pg = step / page_steps;
      in_page[s] = step - pg * page_steps;
      int p = -1;
      if (32 * step <= last) p = b.table[(size_t)req * b.table_ld + pg];
      pid[s] = __builtin_amdgcn_readfirstlane(p >= 0 && p < b.n_pages ? p : -1);
      const int8_t* at = c.k + ((size_t)max(pid[s], 0) * c.kv_heads + head) * ((size_t)b.page * HD) + in_page[s] * (NB * 1024);
#pragma unroll
      for (int k = 0; k < NB; ++k) kc[s][k] = *reinterpret_cast<const u32x4*>(at + 1024 * k + 16 * lane);
      ks[s] = c.ks[(size_t)max(pid[s], 0) * c.kv_heads + head];
    }
    f32x4 sum[KS][2] = {};
    // rows that see some key of the workgroup's
    const int i0 = max(0, k0 - p0);
    const int i1 = a.window > 0 && k0 >= a.sinks ? (int)min((long long)n, (long long)k0 + kKeys - 1 + a.window - p0) : n;
    const int tile1 = (i1 * grp + 15) >> 4;
    for (int t0 = (i0 * grp) >> 4; t0 < tile1; t0 += 4) {
      __syncthreads();                   // the tiles before have been read
      if (t0 + w < tile1) {
        const int vec = 16 * (t0 + w) + col, row = vec / grp, hq = head * grp + vec - row * grp;
        const bool live = row < n;
        const float* at = a.q + (size_t)(q.row0 + (live ? row : 0)) * a.ldq + (size_t)(live ? hq : 0) * HD + 8 * g;
        const float lse = live ? a.lse[(size_t)(q.row0 + row) * a.heads + hq] : INFINITY;
        float x[NB][8];
        unsigned top = 0;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          *reinterpret_cast<float4*>(&x[k][0]) = *reinterpret_cast<const float4*>(at + 32 * k);
          *reinterpret_cast<float4*>(&x[k][4]) = *reinterpret_cast<const float4*>(at + 32 * k + 4);
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[k][j]) & 0x7fffffffu);
        }
        top = max(top, lane_xor_u32<16>(top));
        top = max(top, lane_xor_u32<32>(top));
        const int e = (int)(top >> 23), f = min(267 - e, 253);     // 2^13 <= largest * 2^(f - 127) < 2^14
        // (a row that is not there, sees nothing or is not finite gives no weight: q = 0, lse = inf)
        const bool ok = e != 255 && fabsf(lse) < INFINITY;
        const float up = ok ? copysignf(__uint_as_float((unsigned)f << 23), a.scale) : 0.0f;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[k][j] = ok ? x[k][j] * up : 0.0f;
          h8 hi, lo8;
          split8(x[k], minus_one, hi, lo8);
          qf[((w * NB + k) * 2 + 0) * 64 + lane] = hi;
          qf[((w * NB + k) * 2 + 1) * 64 + lane] = lo8;
        }
        if (g == 0) {
          qss[w][col] = ok ? __uint_as_float((unsigned)(254 - f) << 23) * (fabsf(a.scale) * 1.4426950408889634f) : 0.0f;
          cut[w][col] = ok ? lse * 1.4426950408889634f : INFINITY;
        }
      }
      __syncthreads();
      for (int u = 0; u < 4 && t0 + u < tile1; ++u) {
        const float qs = qss[u][col], m = cut[u][col];
        const int low_row = 16 * (t0 + u) / grp, pos = p0 + (16 * (t0 + u) + col) / grp;
        const int pos_low = p0 + low_row, pos_high = p0 + (16 * (t0 + u) + 15) / grp;
        f32x4 st[KS][2] = {};
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const h8 hi = qf[((u * NB + k) * 2 + 0) * 64 + lane], lo8 = qf[((u * NB + k) * 2 + 1) * 64 + lane];
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const h8 a0 = codes8(kc[s][k][0], kc[s][k][1]), a1 = codes8(kc[s][k][2], kc[s][k][3]);
            st[s][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, hi, st[s][0], 0, 0, 0);
            st[s][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, hi, st[s][1], 0, 0, 0);
            st[s][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, lo8, st[s][0], 0, 0, 0);
            st[s][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, lo8, st[s][1], 0, 0, 0);
          }
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int key0 = k0 + 32 * (w * KS + s);
          const float f = ks[s] * qs;
          const bool hides = key0 + 31 > pos_low || (a.window > 0 && key0 <= pos_high - a.window && key0 + 31 >= a.sinks);
          const int low = a.window > 0 ? pos - a.window + 1 : 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float p = pow2(__builtin_fmaf(st[s][e >> 2][e & 3], f, -m));
            if (hides) {
              const int j = key0 + 16 * (e >> 2) + 4 * g + (e & 3);
              if (j > pos || (j < low && j >= a.sinks)) p = 0.0f;
            }
            sum[s][e >> 2][e & 3] += p;
          }
        }
      }
    }
    // over the 16 vectors of the tiles' columns; a step's own tokens start from nothing
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int key0 = k0 + 32 * (w * KS + s);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = sum[s][h][i];
          v += lane_xor<8>(v);
          v += lane_xor<4>(v);
          v += lane_xor<2>(v);
          y[i] = v + lane_xor<1>(v);
        }
        const int j = key0 + 16 * h + 4 * g;
        if (pid[s] < 0 || j > last || col != 0) continue;
        float4* const at = reinterpret_cast<float4*>(
            a.mass + ((size_t)pid[s] * c.kv_heads + head) * b.page + 32 * in_page[s] + 16 * h + 4 * g);
        const float4 was = *at;
        float z[4] = {was.x, was.y, was.z, was.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j + i <= last) z[i] = j + i >= p0 ? y[i] : z[i] + y[i];
        *at = make_float4(z[0], z[1], z[2], z[3]);
      }
    }
  }
}

template <int NB>
static void launch_mass(const PagedBatch& b, const Kv8Cache& c, const MassArgs& a, hipStream_t s) {
  constexpr int KS = 2, kKeys = 128 * KS;
  long chunks = (std::max(a.max_len, 1) + kKeys - 1) / kKeys;
  if (a.window > 0)
    chunks = std::min(chunks, (long)(a.sinks + kKeys - 1) / kKeys + ((long)a.window + a.max_rows - 2) / kKeys + 2);
  const size_t heads = (size_t)b.requests * c.kv_heads;
  chunks = std::max(1L, std::min(chunks, (long)(kMassMaxWorkgroups / heads)));
  hipLaunchKernelGGL((kv8_mass_kernel<NB, KS>), dim3((unsigned)(heads * chunks)), dim3(256), 0, s, b, c, a,
                     MassCut{(int)chunks});
}

hipError_t launch_kv8_mass(const PagedBatch& b, const Kv8Cache& c, const MassArgs& a, hipStream_t s) {
  switch (c.hd / 32) {
    case 1: launch_mass<1>(b, c, a, s); break;
    case 2: launch_mass<2>(b, c, a, s); break;
    case 3: launch_mass<3>(b, c, a, s); break;
    case 4: launch_mass<4>(b, c, a, s); break;
    case 5: launch_mass<5>(b, c, a, s); break;
    case 6: launch_mass<6>(b, c, a, s); break;
    case 7: launch_mass<7>(b, c, a, s); break;
    default: launch_mass<8>(b, c, a, s); break;
  }
  return hipGetLastError();
}

// ---- which tokens stay -----------------------------------------------------------------------------
// Of T tokens `keep` stay: the first `first`, the last `recent`, and of the N between them the M = keep - first - recent of
// the largest mass, ties to the lower. A mass is a 32-bit key in order of the values (NaN as -inf, a token without a page
// below that). The M-th largest key is found by its digits, 11, 11 and 10 bits from the top: a histogram of those whose
// higher digits are the ones found so far, and a scan of it from the top. Then a token stays if its key is larger, or equal
// and among the first of those.
constexpr int kPickMost = 16;            // tokens of a thread at a time
constexpr int kPickBins = 2048;

__device__ __forceinline__ unsigned mass_key(float x) {
  const unsigned u = __float_as_uint(x != x ? -INFINITY : x + 0.0f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

// One workgroup per (request, head). A thread has up to kPickMost tokens that follow one another, by fours: a page's places
// come in fours that lie together.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv8_evict_pick_kernel(EvictArgs a, int kv_heads) {
  __shared__ int bins[kPickBins];
  __shared__ int found_bin, found_above, found_in;
  const int req = blockIdx.x / kv_heads, head = blockIdx.x % kv_heads, tid = threadIdx.x;
  const int T = a.from_len[req];
  if (T <= a.keep || T > a.table_ld * a.page) return;
  int* const kept = a.kept + (size_t)blockIdx.x * a.keep;
  const int* const table = a.from_table + (size_t)req * a.table_ld;
  const int M = a.keep - a.first - a.recent, end = T - a.recent;   // M of the tokens first .. end - 1
  for (int i = tid; i < a.first; i += THREADS) kept[i] = i;
  for (int i = tid; i < a.recent; i += THREADS) kept[a.keep - a.recent + i] = end + i;
  if (M == 0) return;
  const int per = min(kPickMost, ((end + THREADS - 1) / THREADS + 3) & ~3), block = THREADS * per;
  // tokens at .. at + per - 1 (those behind the middle: some of its own)
  auto load = [&](int at, unsigned (&key)[kPickMost]) {
    float4 x[kPickMost / 4];
    int pid[kPickMost / 4];
#pragma unroll
    for (int e = 0; e < kPickMost / 4; ++e) pid[e] = table[min(at + min(4 * e, per - 4), end - 1) / a.page];
#pragma unroll
    for (int e = 0; e < kPickMost / 4; ++e) {
      const int t = min(at + min(4 * e, per - 4), (end - 1) & ~3);
      const bool there = pid[e] >= 0 && pid[e] < a.n_pages;
      x[e] = *reinterpret_cast<const float4*>(a.mass + ((size_t)(there ? pid[e] : 0) * kv_heads + head) * a.page + t % a.page);
      if (!there) pid[e] = -1;
    }
#pragma unroll
    for (int e = 0; e < kPickMost; ++e) key[e] = pid[e / 4] >= 0 ? mass_key((&x[e / 4].x)[e & 3]) : 0;
  };
  unsigned key[kPickMost];
  const bool once = end <= block;
  auto middle = [&](int at, int e) { return e < per && at + e >= a.first && at + e < end; };
  if (once) load(tid * per, key);
  unsigned high = 0;                     // the digits found, and what of M is left below the larger ones
  int want = M, shift = 32;
  constexpr int kBits[3] = {11, 11, 10};
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    const int size = 1 << kBits[d], below = shift - kBits[d];
    for (int i = tid; i < size; i += THREADS) bins[i] = 0;
    __syncthreads();
    for (int base = 0; base < end; base += block) {
      const int at = base + tid * per;
      if (!once) load(at, key);
#pragma unroll
      for (int e = 0; e < kPickMost; ++e) {
        const bool same = d == 0 || (key[e] >> shift) == (high >> shift);
        if (middle(at, e) && same) atomicAdd(&bins[(key[e] >> below) & (size - 1)], 1);
      }
    }
    __syncthreads();
    // a thread has bins that follow one another, from the top down
    constexpr int kOwn = kPickBins / THREADS;
    const int own = size / THREADS, top = size - 1 - own * tid;
    int mine[kOwn], sum = 0, before;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      mine[i] = i < own ? bins[top - i] : 0;
      sum += mine[i];
    }
    scan_block<THREADS / 64>(sum, before);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (before < want && before + mine[i] >= want) {
        found_bin = top - i;
        found_above = before;
        found_in = mine[i];
      }
      before += mine[i];
    }
    __syncthreads();
    high |= (unsigned)found_bin << below;
    want -= found_above;
    shift = below;
    if (found_in == want) break;         // all of them stay: what their lower digits are does not matter
    __syncthreads();
  }
  // keys above `high` (in their digits down to `shift`) stay, and the first `want` of those equal to it
  high >>= shift;
  int at_kept = a.first, equals = 0;
  for (int base = 0; base < end; base += block) {
    const int at = base + tid * per;
    if (!once) load(at, key);
    int more = 0, same = 0, before;
#pragma unroll
    for (int e = 0; e < kPickMost; ++e) {
      more += middle(at, e) && (key[e] >> shift) > high;
      same += middle(at, e) && (key[e] >> shift) == high;
    }
    // (both counts in one sum: of at most 2^14 tokens)
    const int all = scan_block<THREADS / 64>(more | same << 16, before);
    int s = equals + (before >> 16), o = at_kept + (before & 0xffff) + min(s, want) - min(equals, want);
#pragma unroll
    for (int e = 0; e < kPickMost; ++e) {
      const bool in = middle(at, e), equal = in && (key[e] >> shift) == high;
      if ((in && (key[e] >> shift) > high) || (equal && s < want)) kept[o++] = at + e;
      s += equal;
    }
    at_kept += (all & 0xffff) + min(equals + (all >> 16), want) - min(equals, want);
    equals += all >> 16;
  }
}

// ---- the move --------------------------------------------------------------------------------------
// Place o of new page p holds token kept[p * page + o]; the page's scale is the largest among the pages that its tokens come
// from, so that no code grows, a code round(c * (s_old / s_new)), ties to even. Places behind the last token get code 0 and
// mass 0.
//
// One workgroup for each new page and head, K or V. A lane makes 16 bytes of a block of 32 tokens x 32 dimensions: K's are
// two tokens' 8 dimensions, two loads of 8 bytes; V's are 8 tokens' 2 dimensions, and of each of them the 16 old bytes
// that hold them with 7 neighbours are loaded. Where a lane's tokens lie is found once for all blocks of dimensions.
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// the code in byte i of x, rounded to another scale: q + 1.5 2^23 rounds q to an integer, whose low byte is the code
__device__ __forceinline__ unsigned moved(unsigned x, int i, float r) {
  const float q = (float)((int)(x << (24 - 8 * i)) >> 24) * r;
  return __float_as_uint(q + 12582912.0f);
}
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

template <bool IS_V>
__device__ __forceinline__ void move_page(const EvictArgs& a, const Kv8Cache& c, int req, int p, int pid, int head) {
  __shared__ const int8_t* src[256];     // the old page's first block of the token's 32
  __shared__ int place[256];             // .. and the token's place in it
  __shared__ float ratio[256], red[4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nb = c.hd >> 5, m = lane & 15, g = lane >> 4;
  int8_t* const codes = IS_V ? c.v : c.k;
  float* const scales = IS_V ? c.vs : c.ks;
  const int T = a.from_len[req], count = min(a.page, a.keep - p * a.page);
  const size_t head_bytes = (size_t)a.page * c.hd, mine = (size_t)pid * c.kv_heads + head;
  int from = -1, at = 0;
  float s = 0.0f;
  if (tid < count) {
    const int t = a.kept[((size_t)req * c.kv_heads + head) * a.keep + p * a.page + tid];
    if (t >= 0 && t < T) {
      const int pg = t / a.page, id = a.from_table[(size_t)req * a.table_ld + pg];
      at = t - pg * a.page;
      if (id >= 0 && id < a.n_pages) {
        from = id;
        s = scales[(size_t)id * c.kv_heads + head];
      }
    }
  }
  const float mass = !IS_V && a.mass && from >= 0 ? a.mass[((size_t)from * c.kv_heads + head) * a.page + at] : 0.0f;
  float top = wave_max(s);
  if (lane == 0) red[w] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  if (tid < a.page) {                    // (a place without a token: its own page, times 0)
    ratio[tid] = from >= 0 && top > 0.0f ? s / top : 0.0f;
    src[tid] = codes + (from >= 0 ? (size_t)from * c.kv_heads + head : mine) * head_bytes + (size_t)(at >> 5) * (nb * 1024);
    place[tid] = at & 31;
    if (!IS_V && a.mass) a.mass[mine * a.page + tid] = mass;
  }
  if (tid == 0) scales[mine] = top;
  __syncthreads();
  // waves: blocks of tokens, and where there are fewer than four, every so-manieth block of dimensions
  const int tokens = a.page >> 5, step = tokens >= 4 ? 1 : 4 / tokens;
  for (int tb = w / step; tb < tokens; tb += 4) {
    int8_t* const out = codes + mine * head_bytes + (size_t)tb * (nb * 1024) + 16 * lane;
    if constexpr (IS_V) {
      const u32x4* at8[8];
      int shift[8];
      float r[8];
      bool later[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int o = 32 * tb + 16 * (e >> 2) + 4 * g + (e & 3), x = place[o];
        at8[e] = reinterpret_cast<const u32x4*>(src[o] + 256 * (x >> 2 & 3) + 16 * m);
        shift[e] = x & 3;
        later[e] = x & 16;
        r[e] = ratio[o];
      }
      for (int d = w % step; d < nb; d += step) {
        u32x4 x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = at8[e][64 * d];
        unsigned y[2][8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int b = 0; b < 2; ++b) y[b][e] = moved(later[e] ? x[e][2 * b + 1] : x[e][2 * b], shift[e], r[e]);
        *reinterpret_cast<u32x4*>(out + 1024 * d) =
            u32x4{low_bytes(y[0][0], y[0][1], y[0][2], y[0][3]), low_bytes(y[0][4], y[0][5], y[0][6], y[0][7]),
                  low_bytes(y[1][0], y[1][1], y[1][2], y[1][3]), low_bytes(y[1][4], y[1][5], y[1][6], y[1][7])};
      }
    } else {
      const u32x2* at8[2];
      float r[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int o = 32 * tb + 16 * t + m, x = place[o];
        at8[t] = reinterpret_cast<const u32x2*>(src[o] + 256 * g + 16 * (x & 15) + 8 * (x >> 4));
        r[t] = ratio[o];
      }
#pragma unroll 4
      for (int d = w % step; d < nb; d += step) {
        u32x4 z;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const u32x2 x = at8[t][128 * d];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            z[2 * t + h] = low_bytes(moved(x[h], 0, r[t]), moved(x[h], 1, r[t]), moved(x[h], 2, r[t]), moved(x[h], 3, r[t]));
        }
        *reinterpret_cast<u32x4*>(out + 1024 * d) = z;
      }
    }
  }
}

__global__ __launch_bounds__(256) void kv8_evict_move_kernel(EvictArgs a, Kv8Cache c, long units) {
  const int fresh = (a.keep + a.page - 1) / a.page;
  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    const long page = u >> 1;
    const int head = (int)(page % c.kv_heads), p = (int)(page / c.kv_heads % fresh), req = (int)(page / c.kv_heads / fresh);
    const int T = a.from_len[req];
    if (T <= a.keep || T > a.table_ld * a.page) continue;
    const int pid = a.table[(size_t)req * a.table_ld + p];
    if (pid < 0 || pid >= a.n_pages) continue;
    if (u & 1) move_page<true>(a, c, req, p, pid, head);
    else move_page<false>(a, c, req, p, pid, head);
    __syncthreads();
  }
}

hipError_t launch_kv8_evict(const EvictArgs& a, const Kv8Cache& c, hipStream_t s) {
  const dim3 picks((unsigned)(a.requests * c.kv_heads));
  // the fewest waves that hold a request's tokens at once: their barriers are shorter
  if (a.max_len <= 256 * kPickMost) hipLaunchKernelGGL(kv8_evict_pick_kernel<256>, picks, dim3(256), 0, s, a, c.kv_heads);
  else if (a.max_len <= 512 * kPickMost) hipLaunchKernelGGL(kv8_evict_pick_kernel<512>, picks, dim3(512), 0, s, a, c.kv_heads);
  else hipLaunchKernelGGL(kv8_evict_pick_kernel<1024>, picks, dim3(1024), 0, s, a, c.kv_heads);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const long units = 2L * a.requests * c.kv_heads * ((a.keep + a.page - 1) / a.page);
  hipLaunchKernelGGL(kv8_evict_move_kernel, dim3((unsigned)std::min(units, 1L << 22)), dim3(256), 0, s, a, c, units);
  return hipGetLastError();
}

}  // namespace rehip
