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
// f16, q in two f16 parts, f32 sums. A key belongs to one wave or workgroup, so its sum is taken in one order.
//
// A piece is 32 KS keys of one request and head, held as f16 operands in registers; tiles of 16 query vectors that see some of
// them go past, each split by the wave that multiplies it (the matrix operand's lanes are those that load it), the next
// one on its way meanwhile. Sums over a tile's vectors stay in the lanes until the end. Steps of few vectors: a wave takes a
// piece alone (W = 1). Prompts: the four waves of a workgroup share a piece and take every fourth tile (W = 4). The launch has as
// many waves as run at once, and each takes every so-manieth piece of the whole batch, found from the lengths: a piece for each
// wave of the longest request's would leave most of a ragged batch's waves without any.
#ifndef MWG
#define MWG 1024
#endif
constexpr int kMassWorkgroups = MWG;
struct MassCut {
  int chunks;                            // pieces of a request and head, of the longest planned
  int mode;                              // how a piece is found: below
};
constexpr int kMassLanes = 0, kMassListed = 1, kMassEven = 2;      // requests a lane each; listed in LDS; chunks of each
constexpr int kMassList = 1024;

// A request's pieces: those of the sinks, then those from `first` on that some row sees; n rows from position p0 to `last`.
struct MassPlace {
  int n, p0, last, sinks, first, all;
};
__device__ __forceinline__ MassPlace mass_place(const PagedBatch& b, const MassArgs& a, const RequestRows& q, int keys) {
  MassPlace o;
  o.n = min(q.count, a.max_rows);
  o.p0 = max(q.len, 0) - q.count;
  o.last = min(o.p0 + o.n, b.table_ld * b.page) - 1;               // (no key behind the table)
  const int lo = a.window > 0 ? max(0, o.p0 - a.window + 1) : 0;
  o.sinks = a.window > 0 ? (min(a.sinks, o.last + 1) + keys - 1) / keys : 0;
  o.first = max(lo / keys, o.sinks);
  o.all = o.n <= 0 || o.last < 0 ? 0 : o.sinks + max(o.last / keys - o.first + 1, 0);
  return o;
}

template <int NB, int W>
__global__ __launch_bounds__(256, 2) void kv8_mass_kernel(PagedBatch b, Kv8Cache c, MassArgs a, MassCut t) {
  constexpr int HD = 32 * NB, KS = NB <= 2 ? 4 : NB <= 4 ? 2 : 1, kKeys = 32 * KS;
  __shared__ float4 red[W > 1 ? W - 1 : 1][2 * KS][4];
  __shared__ int at[kMassList];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4, page_steps = b.page >> 5, grp = a.heads / c.kv_heads;
  float minus_one = -1.0f;
  asm volatile("" : "+v"(minus_one));

  auto piece = [&](int req, int row0, const MassPlace& o, int ch, int head) {
    const int k0 = (ch < o.sinks ? ch : ch - o.sinks + o.first) * kKeys;
    int pid[KS], in_page[KS];
    u32x4 kc[KS][NB];
    float ks[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int step = (k0 >> 5) + s, pg = step / page_steps;
      in_page[s] = step - pg * page_steps;
      pid[s] = b.table[(size_t)req * b.table_ld + min(pg, b.table_ld - 1)];
      if (32 * step > o.last || pid[s] >= b.n_pages) pid[s] = -1;
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      pid[s] = __builtin_amdgcn_readfirstlane(pid[s]);
      const int8_t* p = c.k + ((size_t)max(pid[s], 0) * c.kv_heads + head) * ((size_t)b.page * HD) + in_page[s] * (NB * 1024);
#pragma unroll
      for (int k = 0; k < NB; ++k) kc[s][k] = *reinterpret_cast<const u32x4*>(p + 1024 * k + 16 * lane);
      ks[s] = c.ks[(size_t)max(pid[s], 0) * c.kv_heads + head];
    }
    // this lane's four places of each half step, and what is there already
    float4* place[KS][2];
    float4 was[KS][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        place[s][h] = reinterpret_cast<float4*>(a.mass + ((size_t)max(pid[s], 0) * c.kv_heads + head) * b.page +
                                                32 * in_page[s] + 16 * h + 4 * g);
        if (W == 1) was[s][h] = *place[s][h];
      }
    // tiles of the vectors that see some key of the piece
    const int i0 = max(0, k0 - o.p0);
    const int i1 = a.window > 0 && k0 >= a.sinks ? (int)min((long long)o.n, (long long)k0 + kKeys - 1 + a.window - o.p0) : o.n;
    const int tile1 = (i1 * grp + 15) >> 4;
    int tile = ((i0 * grp) >> 4) + (W > 1 ? w : 0);
    float x[NB][8], lse;
    int row;
    auto load_q = [&](int tile, float (&x)[NB][8], float& lse, int& row) {
      const int vec = 16 * tile + col;
      row = vec / grp;
      const int r = row0 + min(row, o.n - 1), hq = head * grp + vec - row * grp;
      const float* p = a.q + (size_t)r * a.ldq + (size_t)hq * HD + 8 * g;
      lse = a.lse[(size_t)r * a.heads + hq];
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        *reinterpret_cast<float4*>(&x[k][0]) = *reinterpret_cast<const float4*>(p + 32 * k);
        *reinterpret_cast<float4*>(&x[k][4]) = *reinterpret_cast<const float4*>(p + 32 * k + 4);
      }
    };
    f32x4 sum[KS][2] = {};
    if (tile < tile1) load_q(tile, x, lse, row);
    h8 kf[KS][NB][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        kf[s][k][0] = codes8(kc[s][k][0], kc[s][k][1]);
        kf[s][k][1] = codes8(kc[s][k][2], kc[s][k][3]);
      }
    for (; tile < tile1; tile += W) {
      unsigned top = 0;
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[k][j]) & 0x7fffffffu);
      top = max(top, lane_xor_u32<16>(top));
      top = max(top, lane_xor_u32<32>(top));
      const int e = (int)(top >> 23), f = min(267 - e, 253);       // 2^13 <= largest * 2^(f - 127) < 2^14
      // (a row that is not there, sees nothing or is not finite gives no weight: q = 0, lse = inf)
      const bool ok = e != 255 && row < o.n && fabsf(lse) < INFINITY;
      const float up = copysignf(__uint_as_float((unsigned)f << 23), a.scale);
      const float qs = ok ? __uint_as_float((unsigned)(254 - f) << 23) * (fabsf(a.scale) * 1.4426950408889634f) : 0.0f;
      const float m = ok ? lse * 1.4426950408889634f : INFINITY;
      h8 qh[NB], ql[NB];
#pragma unroll
      for (int k = 0; k < NB; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[k][j] = ok ? x[k][j] * up : 0.0f;
        split8(x[k], minus_one, qh[k], ql[k]);
      }
      const int pos = o.p0 + row;
      const int pos_low = __builtin_amdgcn_readlane(pos, 0), pos_high = __builtin_amdgcn_readlane(pos, 15);
      load_q(tile + W < tile1 ? tile + W : tile, x, lse, row);     // (on its way while this one is multiplied)
      f32x4 st[KS][2] = {};
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          st[s][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[s][k][0], qh[k], st[s][0], 0, 0, 0);
          st[s][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[s][k][1], qh[k], st[s][1], 0, 0, 0);
          st[s][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[s][k][0], ql[k], st[s][0], 0, 0, 0);
          st[s][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[s][k][1], ql[k], st[s][1], 0, 0, 0);
        }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int key0 = k0 + 32 * s;
        const float factor = ks[s] * qs;
        const bool hides = key0 + 31 > pos_low || (a.window > 0 && key0 <= pos_high - a.window && key0 + 31 >= a.sinks);
        const int low = a.window > 0 ? pos - a.window + 1 : 0;
#pragma unroll
        for (int e8 = 0; e8 < 8; ++e8) {
          float p = pow2(__builtin_fmaf(st[s][e8 >> 2][e8 & 3], factor, -m));
          if (hides) {
            const int j = key0 + 16 * (e8 >> 2) + 4 * g + (e8 & 3);
            if (j > pos || (j < low && j >= a.sinks)) p = 0.0f;
          }
          sum[s][e8 >> 2][e8 & 3] += p;
        }
      }
    }
    // over the 16 vectors of the tiles' columns, and the waves; a step's own tokens start from nothing
    float4 y[KS][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = sum[s][h][i];
          v += lane_xor<8>(v);
          v += lane_xor<4>(v);
          v += lane_xor<2>(v);
          (&y[s][h].x)[i] = v + lane_xor<1>(v);
        }
    if constexpr (W > 1) {
      __syncthreads();                   // the piece before has been read
      if (w > 0 && col == 0) {
#pragma unroll
        for (int s = 0; s < 2 * KS; ++s) red[w - 1][s][g] = y[s >> 1][s & 1];
      }
      __syncthreads();
      if (w > 0) return;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          was[s][h] = *place[s][h];
#pragma unroll
          for (int i = 0; i < W - 1; ++i) {
            const float4 z = red[i][2 * s + h][g];
            y[s][h] = make_float4(y[s][h].x + z.x, y[s][h].y + z.y, y[s][h].z + z.z, y[s][h].w + z.w);
          }
        }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = k0 + 32 * s + 16 * h + 4 * g;
        if (pid[s] < 0 || j > o.last || col != 0) continue;
        float z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float old = (&was[s][h].x)[i], add = (&y[s][h].x)[i];
          z[i] = j + i > o.last ? old : j + i >= o.p0 ? add : old + add;
        }
        *place[s][h] = make_float4(z[0], z[1], z[2], z[3]);
      }
  };

  const int first = W > 1 ? blockIdx.x : 4 * blockIdx.x + w, stride = W > 1 ? gridDim.x : 4 * gridDim.x;
  if (t.mode == kMassLanes) {
    const int i = min(lane, b.requests - 1);
    const RequestRows q = request_rows(i, b.start[i], b.count[i], b.len[i], b.rows);
    const MassPlace o = mass_place(b, a, q, kKeys);
    const int mine = lane < b.requests ? o.all : 0, upto = wave_scan(mine);
    const int total = __builtin_amdgcn_readlane(upto, 63) * c.kv_heads;
    for (int u = first; u < total; u += stride) {
      const int ch = u / c.kv_heads, l = __ffsll(__ballot(ch < upto)) - 1;
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      piece(l, of(q.row0), MassPlace{of(o.n), of(o.p0), of(o.last), of(o.sinks), of(o.first), of(o.all)}, ch - of(upto - mine),
            u - ch * c.kv_heads);
    }
    return;
  }
  if (t.mode == kMassListed) {
    constexpr int kOwn = kMassList / 256;
    int mine[kOwn], sum = 0, before;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int r = kOwn * threadIdx.x + i, in = min(r, b.requests - 1);
      const MassPlace o = mass_place(b, a, request_rows(in, b.start[in], b.count[in], b.len[in], b.rows), kKeys);
      mine[i] = r < b.requests ? o.all : 0;
      sum += mine[i];
    }
    const int total = scan_block<4>(sum, before) * c.kv_heads;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      at[kOwn * threadIdx.x + i] = before;
      before += mine[i];
    }
    __syncthreads();
    for (int u = first; u < total; u += stride) {
      const int ch = u / c.kv_heads, r = last_at_most(at, b.requests, ch);
      const RequestRows q = request_rows(r, b.start[r], b.count[r], b.len[r], b.rows);
      piece(r, q.row0, mass_place(b, a, q, kKeys), ch - at[r], u - ch * c.kv_heads);
    }
    return;
  }
  const long long all = (long long)b.requests * t.chunks * c.kv_heads;
  for (long long u = first; u < all; u += stride) {
    const int head = (int)(u % c.kv_heads), r = (int)(u / c.kv_heads / t.chunks);
    const RequestRows q = request_rows(r, b.start[r], b.count[r], b.len[r], b.rows);
    const MassPlace o = mass_place(b, a, q, kKeys);
    for (int ch = (int)(u / c.kv_heads % t.chunks); ch < o.all; ch += t.chunks) piece(r, q.row0, o, ch, head);
  }
}

template <int NB, int W>
static void launch_mass_as(const PagedBatch& b, const Kv8Cache& c, const MassArgs& a, hipStream_t s) {
  constexpr int kKeys = 32 * (NB <= 2 ? 4 : NB <= 4 ? 2 : 1);
  long chunks = (std::max(a.max_len, 1) + kKeys - 1) / kKeys;
  if (a.window > 0)
    chunks = std::min(chunks, (long)(a.sinks + kKeys - 1) / kKeys + ((long)a.window + a.max_rows - 2) / kKeys + 2);
  const int mode = b.requests <= 64 ? kMassLanes : b.requests <= kMassList ? kMassListed : kMassEven;
  if (mode == kMassEven) chunks = std::min(chunks, 16L);           // (a longer request's waves take several)
  const long waves = (long)b.requests * c.kv_heads * chunks;
  const long groups = std::min(W > 1 ? waves : (waves + 3) / 4, (long)kMassWorkgroups);
  hipLaunchKernelGGL((kv8_mass_kernel<NB, W>), dim3((unsigned)groups), dim3(256), 0, s, b, c, a, MassCut{(int)chunks, mode});
}
template <int NB>
static void launch_mass(const PagedBatch& b, const Kv8Cache& c, const MassArgs& a, hipStream_t s) {
  if ((long)a.max_rows * (a.heads / c.kv_heads) > 64) launch_mass_as<NB, 4>(b, c, a, s);
  else launch_mass_as<NB, 1>(b, c, a, s);
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
