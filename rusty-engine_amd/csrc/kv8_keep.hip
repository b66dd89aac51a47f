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
// them go past, each split by the wave that multiplies it, the next one on its way meanwhile. Sums over a tile's vectors stay in
// the lanes until the end, and are then taken by halves, so that every lane ends with a key or two of its own. Steps of few vectors:
// a wave takes a piece alone (W = 1). Prompts: a workgroup's W waves share a piece and take every W-th tile. The launch has about
// as many workgroups as run at once, and each takes every so-manieth piece of the whole batch, found from the lengths: with a piece
// for each of the longest request's, most workgroups of a ragged batch would find nothing (64 requests of up to 8192 tokens 32 us,
// where these took 17, before q went through LDS).
//
// 64 requests of up to 8192 tokens, 32 heads in 4 of 128, 36 MB: 14.6 us, 2.4 TB/s: two pieces a wave, one after the other, four
// trips to memory each. Two prompts of up to 1000 rows behind up to 5000 tokens, 16 heads in 8 of 64, 9.7 GFLOP and as many of low
// parts: 47 us: exponentials, the split of q (each vector for every 128 keys) and few pieces of unequal length (the first keys
// are seen by every row), two waves on a SIMD half of the time waiting. One prompt of 961 rows, 32 heads in 4 of 128: 71 us, the
// workgroups of the first keys, which every row sees, with the split of q for each 32.
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

// f(request, its first row, its place, piece, head) for every `stride`-th piece of the batch from `u` on. `at`: kMassList places in
// LDS. All threads of the workgroup call it.
template <int WAVES, class F>
__device__ __forceinline__ void mass_pieces(const PagedBatch& b, const MassArgs& a, const MassCut& t, int kv_heads, int keys,
                                            int u, int stride, int* at, F f) {
  const int lane = threadIdx.x & 63, i = min(lane, b.requests - 1);
  RequestRows q{};
  MassPlace mine{};
  int upto = 0;
  long long total = (long long)b.requests * t.chunks * kv_heads;
  if (t.mode == kMassLanes) {
    q = request_rows(i, b.start[i], b.count[i], b.len[i], b.rows);
    mine = mass_place(b, a, q, keys);
    if (lane >= b.requests) mine.all = 0;
    upto = wave_scan(mine.all);
    total = (long long)__builtin_amdgcn_readlane(upto, 63) * kv_heads;
  } else if (t.mode == kMassListed) {
    constexpr int kOwn = kMassList / (64 * WAVES);
    int n[kOwn], sum = 0, before;
#pragma unroll
    for (int e = 0; e < kOwn; ++e) {
      const int r = kOwn * threadIdx.x + e, in = min(r, b.requests - 1);
      const MassPlace o = mass_place(b, a, request_rows(in, b.start[in], b.count[in], b.len[in], b.rows), keys);
      n[e] = r < b.requests ? o.all : 0;
      sum += n[e];
    }
    total = (long long)scan_block<WAVES>(sum, before) * kv_heads;
#pragma unroll
    for (int e = 0; e < kOwn; ++e) {
      at[kOwn * threadIdx.x + e] = before;
      before += n[e];
    }
    __syncthreads();
  }
  for (long long v = u; v < total; v += stride) {
    const int c = (int)(v / kv_heads), head = (int)(v - (long long)c * kv_heads);
    int r, row0, ch, step = 0x40000000;
    MassPlace o;
    if (t.mode == kMassLanes) {
      r = __ffsll(__ballot(c < upto)) - 1;
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, r); };
      row0 = of(q.row0);
      o = {of(mine.n), of(mine.p0), of(mine.last), of(mine.sinks), of(mine.first), of(mine.all)};
      ch = c - of(upto - mine.all);
    } else {
      if (t.mode == kMassListed) {
        r = __builtin_amdgcn_readfirstlane(last_at_most(at, b.requests, c));
        ch = c - at[r];
      } else {
        r = c / t.chunks;
        ch = c - r * t.chunks;
        step = t.chunks;
      }
      const RequestRows y = request_rows(r, b.start[r], b.count[r], b.len[r], b.rows);
      o = mass_place(b, a, y, keys);
      row0 = y.row0;
    }
    for (; ch < o.all; ch += step) f(r, row0, o, ch, head);
  }
}

// A tile of 16 vectors. The matrix operand's lane m + 16 g has vector m, dimensions 32 k + 8 g .. . Loaded by those lanes (DIRECT) every
// lane of an instruction meets a line of its own, and the CU's load unit, a line a clock, bounds pieces of few keys whatever the
// waves: so four lanes next to one another load 128 bytes of one vector (lane l: vector l / 4, dimensions 32 k + 8 (l % 4) ..) and split
// them, and what a lane then holds, 16 bytes of each part, is what one lane of the operand needs: they change places in the
// wave's own LDS (us of direct / this: a step of 64 requests, 4 heads of 128 16.0 / 14.8, 4000 vectors of two requests of up to 5000, 4 of
// 256 291 / 182; but pieces of 128 keys of 64, 16 heads in 8, 46.5 / 51.6).
constexpr int kMassSlots = 68;           // 64 lanes' 16 bytes and a slot behind every 16, so that both orders meet all banks
__device__ __forceinline__ int mass_slot(int i) { return i + (i >> 4); }
template <int NB, bool DIRECT>
struct MassVector {
  float x[NB][8], lse;
  int row;                               // of the operand's vector
  __device__ __forceinline__ void load(const MassArgs& a, const MassPlace& o, int row0, int grp, int head, int tile) {
    const int lane = threadIdx.x & 63, vec = 16 * tile + (lane & 15), from = DIRECT ? vec : 16 * tile + (lane >> 2);
    const int at = from / grp, part = DIRECT ? lane >> 4 : lane & 3;
    row = vec / grp;
    const float* p = a.q + (size_t)(row0 + min(at, o.n - 1)) * a.ldq + (size_t)(head * grp + from - at * grp) * (32 * NB) + 8 * part;
    lse = a.lse[(size_t)(row0 + min(row, o.n - 1)) * a.heads + head * grp + vec - row * grp];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      *reinterpret_cast<float4*>(&x[k][0]) = *reinterpret_cast<const float4*>(p + 32 * k);
      *reinterpret_cast<float4*>(&x[k][4]) = *reinterpret_cast<const float4*>(p + 32 * k + 4);
    }
  }
  // the operand's two f16 parts, scaled by the power of two that takes the largest element to 2^13 .. 2^14; the factor of its
  // products and its lse, in powers of 2. A row that is not there, sees nothing or is not finite gives no weight: lse = inf, and q = 0
  // if it is not finite. `swap`: the wave's LDS
  __device__ __forceinline__ float2 split(const MassArgs& a, const MassPlace& o, float minus_one, h8* swap, h8 (&hi)[NB], h8 (&lo)[NB]) {
    const int lane = threadIdx.x & 63;
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[k][j]) & 0x7fffffffu);
    top = max(top, lane_xor_u32<DIRECT ? 16 : 1>(top));
    top = max(top, lane_xor_u32<DIRECT ? 32 : 2>(top));
    const int e = (int)(top >> 23);
    int f = min(267 - e, 253);
    const float up = copysignf(__uint_as_float((unsigned)f << 23), a.scale);
    if (e == 255) f = -1;
    if (__ballot(f < 0) != 0) {
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[k][j] = f < 0 ? 0.0f : x[k][j];
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[k][j] *= up;
      split8(x[k], minus_one, hi[k], lo[k]);
    }
    if constexpr (!DIRECT) {
      const int to = mass_slot(lane), from = mass_slot(4 * (lane & 15) + (lane >> 4));
      wave_sync();                       // (the tile before has been read)
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        swap[2 * k * kMassSlots + to] = hi[k];
        swap[(2 * k + 1) * kMassSlots + to] = lo[k];
      }
      f = __shfl(f, 4 * (lane & 15), 64);
      wave_sync();
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        hi[k] = swap[2 * k * kMassSlots + from];
        lo[k] = swap[(2 * k + 1) * kMassSlots + from];
      }
    }
    const bool ok = f >= 0 && row < o.n && fabsf(lse) < INFINITY;
    return ok ? make_float2(__uint_as_float((unsigned)(254 - f) << 23) * (fabsf(a.scale) * 1.4426950408889634f),
                            lse * 1.4426950408889634f)
              : make_float2(0.0f, INFINITY);
  }
};

// A wave's keys, from k0 on, and their sums.
template <int NB, int KS>
struct MassKeys {
  u32x4 raw[KS][NB];
  float scale[KS];
  int k0;
  f32x4 sum[KS][2];
  // a lane's own keys (KS = 1: of every other lane), -1 where there is none, their places and what is there
  static constexpr int kLeft = KS > 1 ? KS / 2 : 1;
  int mine[kLeft];
  float* place[kLeft];
  float was[kLeft];
  __device__ __forceinline__ void load(const PagedBatch& b, const Kv8Cache& c, const MassArgs& a, const MassPlace& o, int req, int head,
                                       int from) {
    const int page_steps = b.page >> 5, lane = threadIdx.x & 63, col = lane & 15;
    k0 = from;
    int pid[KS], in_page[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int step = (k0 >> 5) + s, pg = step / page_steps;
      in_page[s] = step - pg * page_steps;
      const int id = b.table[(size_t)req * b.table_ld + min(pg, b.table_ld - 1)];
      pid[s] = 32 * step > o.last || id >= b.n_pages ? -1 : id;
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      pid[s] = __builtin_amdgcn_readfirstlane(pid[s]);
      const size_t page = (size_t)max(pid[s], 0) * c.kv_heads + head;
      const int8_t* p = c.k + page * ((size_t)b.page * (32 * NB)) + in_page[s] * (NB * 1024) + 16 * lane;
#pragma unroll
      for (int k = 0; k < NB; ++k) raw[s][k] = *reinterpret_cast<const u32x4*>(p + 1024 * k);
      scale[s] = c.ks[page];
      sum[s][0] = sum[s][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int e = 0; e < kLeft; ++e) {
      const int i = KS > 1 ? kLeft * col + e : col >> 1, s = i >> 3;                // its number: 8 step + 4 half + place
      int page = 0, step = 0;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        page = k == s ? pid[k] : page;
        step = k == s ? in_page[k] : step;
      }
      const int in = 16 * (i >> 2 & 1) + 4 * (lane >> 4) + (i & 3), key = k0 + 32 * s + in;
      mine[e] = page >= 0 && key <= o.last && (KS > 1 || (col & 1) == 0) ? key : -1;
      place[e] = a.mass + ((size_t)max(page, 0) * c.kv_heads + head) * b.page + 32 * step + in;
      was[e] = *place[e];
    }
  }
  // adds the weights of a tile of 16 vectors; st: their products, v: factor and lse, pos: positions (low, high: of the tile's
  // first and last)
  __device__ __forceinline__ void add(const MassArgs& a, const f32x4 (&st)[KS][2], float2 v, int pos, int low, int high) {
    const int g = (threadIdx.x & 63) >> 4, from = a.window > 0 ? pos - a.window + 1 : 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int key0 = k0 + 32 * s;
      const float f = scale[s] * v.x;
      const bool hides = key0 + 31 > low || (a.window > 0 && key0 <= high - a.window && key0 + 31 >= a.sinks);
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = pow2(__builtin_fmaf(st[s][e >> 2][e & 3], f, -v.y));
      if (hides) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = key0 + 16 * (e >> 2) + 4 * g + (e & 3);
          if (j > pos || (j < from && j >= a.sinks)) p[e] = 0.0f;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[s][e >> 2][e & 3] += p[e];
    }
  }
  // The sums over the 16 lanes that share keys, by halves: a lane ends with those of its own kLeft keys. v[0 .. N - 1]: what is
  // left, over the lanes xor X, X / 2, .., 1.
  template <int N, int X>
  static __device__ __forceinline__ void halve(float (&v)[8 * KS]) {
    if constexpr (N == 1) {
      v[0] += lane_xor<X>(v[0]);
    } else {
      const bool upper = threadIdx.x & X;
#pragma unroll
      for (int k = 0; k < N / 2; ++k) {
        const float keep = upper ? v[k + N / 2] : v[k], give = upper ? v[k] : v[k + N / 2];
        v[k] = keep + lane_xor<X>(give);
      }
    }
    if constexpr (X > 1) halve<(N > 1 ? N / 2 : 1), X / 2>(v);
  }
  __device__ __forceinline__ void reduce(float (&out)[kLeft]) const {
    float v[8 * KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[8 * s + 4 * h + i] = sum[s][h][i];
    halve<8 * KS, 8>(v);
#pragma unroll
    for (int e = 0; e < kLeft; ++e) out[e] = v[e];
  }
  // .. added to what the keys have; a step's own tokens start from nothing
  __device__ __forceinline__ void write(const MassPlace& o, const float (&v)[kLeft]) const {
#pragma unroll
    for (int e = 0; e < kLeft; ++e)
      if (mine[e] >= 0) *place[e] = mine[e] >= o.p0 ? v[e] : was[e] + v[e];
  }
};

// tiles of the vectors that see some of `keys` keys from k0 on
__device__ __forceinline__ int2 mass_tiles(const MassArgs& a, const MassPlace& o, int grp, int k0, int keys) {
  const int i0 = max(0, k0 - o.p0);
  const int i1 = a.window > 0 && k0 >= a.sinks ? (int)min((long long)o.n, (long long)k0 + keys - 1 + a.window - o.p0) : o.n;
  return make_int2((i0 * grp) >> 4, (i1 * grp + 15) >> 4);
}
__device__ __forceinline__ int piece_key(const MassPlace& o, int ch, int keys) {
  return (ch < o.sinks ? ch : ch - o.sinks + o.first) * keys;
}

// W = 1: a wave for each piece. Else a workgroup for each, whose W waves take every W-th tile.
// Steps of a piece: as many as leave a SIMD two waves (us of 1 / 2 for a wave alone: 64 requests of up to 8192 tokens, 4 heads of
// 128 20.9 / 16.8; of 2 / 4 for prompts of 8 heads of 64 62 / 48).
constexpr int mass_steps(int nb, int w) { return w == 4 && nb <= 2 ? 4 : nb <= 4 && w < 16 ? 2 : 1; }
template <int NB, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W, W < 16 ? 2 : 4) void kv8_mass_kernel(PagedBatch b, Kv8Cache c, MassArgs a, MassCut t) {
  constexpr int KS = mass_steps(NB, W), kKeys = 32 * KS, kLeft = MassKeys<NB, KS>::kLeft;
  constexpr bool kDirect = KS == 4;
  __shared__ float red[W > 1 ? W - 1 : 1][kLeft][64];
  __shared__ int at[kMassList];
  __shared__ h8 swap[kDirect ? 1 : W == 1 ? 4 : W][2 * NB * kMassSlots];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grp = a.heads / c.kv_heads;
  float minus_one = -1.0f;
  asm volatile("" : "+v"(minus_one));
  mass_pieces<W == 1 ? 4 : W>(b, a, t, c.kv_heads, kKeys, W == 1 ? 4 * blockIdx.x + w : blockIdx.x, W == 1 ? 4 * gridDim.x : gridDim.x,
                              at, [&](int req, int row0, const MassPlace& o, int ch, int head) {
    const int k0 = piece_key(o, ch, kKeys);
    MassKeys<NB, KS> keys;
    keys.load(b, c, a, o, req, head, k0);
    const int2 tiles = mass_tiles(a, o, grp, k0, kKeys);
    int tile = tiles.x + (W == 1 ? 0 : w);
    MassVector<NB, kDirect> q;
    if (tile < tiles.y) q.load(a, o, row0, grp, head, tile);
    h8 kf[KS][NB][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        kf[s][k][0] = codes8(keys.raw[s][k][0], keys.raw[s][k][1]);
        kf[s][k][1] = codes8(keys.raw[s][k][2], keys.raw[s][k][3]);
      }
    for (; tile < tiles.y; tile += W) {
      h8 hi[NB], lo[NB];
      const float2 v = q.split(a, o, minus_one, swap[kDirect ? 0 : w], hi, lo);
      const int pos = o.p0 + q.row;
      q.load(a, o, row0, grp, head, tile + W < tiles.y ? tile + W : tile);          // (on its way meanwhile)
      f32x4 st[KS][2] = {};
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              st[s][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[s][k][h], part ? lo[k] : hi[k], st[s][h], 0, 0, 0);
      keys.add(a, st, v, pos, __builtin_amdgcn_readlane(pos, 0), __builtin_amdgcn_readlane(pos, 15));
    }
    float sums[kLeft];
    keys.reduce(sums);
    if constexpr (W > 1) {               // the waves' sums, in their order
      __syncthreads();                   // (those of the piece before have been read)
#pragma unroll
      for (int e = 0; e < kLeft; ++e)
        if (w > 0) red[w - 1][e][lane] = sums[e];
      __syncthreads();
      if (w > 0) return;
#pragma unroll
      for (int i = 0; i < W - 1; ++i)
#pragma unroll
        for (int e = 0; e < kLeft; ++e) sums[e] += red[i][e][lane];
    }
    keys.write(o, sums);
  });
}

static MassCut mass_cut(const PagedBatch& b, const MassArgs& a, int keys) {
  long chunks = (std::max(a.max_len, 1) + keys - 1) / keys;
  if (a.window > 0) chunks = std::min(chunks, (long)(a.sinks + keys - 1) / keys + ((long)a.window + a.max_rows - 2) / keys + 2);
  const int mode = b.requests <= 64 ? kMassLanes : b.requests <= kMassList ? kMassListed : kMassEven;
  return {(int)(mode == kMassEven ? std::min(chunks, 16L) : chunks), mode};        // (a longer request's waves take several)
}

template <int NB, int W>
static long mass_count(const PagedBatch& b, const Kv8Cache& c, const MassArgs& a) {
  return (long)b.requests * c.kv_heads * mass_cut(b, a, 32 * mass_steps(NB, W)).chunks;
}
template <int NB, int W>
static void launch_mass_as(const PagedBatch& b, const Kv8Cache& c, const MassArgs& a, hipStream_t s) {
  const long pieces = mass_count<NB, W>(b, c, a);
  const long groups = W == 1 ? std::min((pieces + 3) / 4, 512L) : std::min(pieces, 4096L / W);
  hipLaunchKernelGGL((kv8_mass_kernel<NB, W>), dim3((unsigned)groups), dim3(W == 1 ? 256 : 64 * W), 0, s, b, c, a,
                     mass_cut(b, a, 32 * mass_steps(NB, W)));
}
// Eight and sixteen waves of a piece have a CU each, so they pay if the launch's work is no more than a round of 256: the pieces of
// all keys by how much of the rows they see on average (the first keys are seen by every row, the last by one), of several requests
// of which about half are that long.
template <int NB, int W>
static bool one_round(const PagedBatch& b, const Kv8Cache& c, const MassArgs& a) {
  const long keys = 32 * mass_steps(NB, W), rows = std::min(a.max_rows, a.max_len);
  long span = a.max_len - rows / 2;
  if (a.window > 0) span = std::min(span, (long)std::max(a.max_rows, a.window) + a.sinks);
  return (span + keys - 1) / keys * c.kv_heads * ((b.requests + 1) / 2) <= 256;
}
// Waves of a piece, us of each:
//   one up to four tiles of vectors (1 / 2 / 4: 64 vectors of one request of 1000 tokens, 2 heads of 64 7.5 / 8.7 / 8.5, of 64 of up to 2000,
//     8 of 64 13.6 / 15.8 / 20.2; but 128 of one of 1000 10.4 / 8.7 / 8.5), of heads beyond 128 up to one tile unless their pieces are many;
//   two for a few more vectors of so many pieces that they fill the card by themselves (2 / 4: 128 vectors of 64 requests of up to
//     2000, 8 of 64 21.4 / 26.8, of 128 31.1 / 38.5, 256 vectors 49.4 / 57.4; but 512, 8 of 64 72 / 66, and 256, 2 of 64 15.9 / 14.4);
//   sixteen of 32 keys for prompts of so few that all have a CU (4 / 8 / 16: 1000 tokens, 4000 vectors, 2 of 64 62 / 38 / 28, 4 of 128
//     75 / 55 / 41; but three of 475, 8 of 128 32 / 31 / 35);
//   eight of 64 (32 of heads beyond 128) if one round does (4 / 8: 2048 vectors of two requests of up to 5000, a window of 1000, 8
//     of 64 52 / 30, of 128 49 / 36; 500 rows of one of 2500, 8 of 128 53 / 57, 1000 78 / 68);
//   else four, of 128 keys of heads up to 64.
template <int NB>
static void launch_mass(const PagedBatch& b, const Kv8Cache& c, const MassArgs& a, hipStream_t s) {
  const long vectors = (long)a.max_rows * (a.heads / c.kv_heads);
  const bool alone = NB <= 4 || vectors <= 16 || mass_count<NB, 1>(b, c, a) > 1024;
  if (vectors <= 64 && alone) launch_mass_as<NB, 1>(b, c, a, s);
  else if (vectors <= 64 || (vectors <= 256 && mass_count<NB, 2>(b, c, a) > 4096)) launch_mass_as<NB, 2>(b, c, a, s);
  else if (NB <= 4 && vectors > 128 && mass_count<NB, 16>(b, c, a) <= 256) launch_mass_as<NB, NB <= 4 ? 16 : 8>(b, c, a, s);
  else if (vectors > 128 && one_round<NB, 8>(b, c, a)) launch_mass_as<NB, 8>(b, c, a, s);
  else launch_mass_as<NB, 4>(b, c, a, s);
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
//
// 32 requests of 8 heads and up to 8192 tokens, 8 MB of masses: 13.7 us (2101 tokens, two heads: 10.2), not bandwidth but a chain:
// lengths, table, masses (held in registers after that), then for each digit zeros, counts in LDS, a scan, four barriers, and a last
// scan for the places. The search ends at the first digit whose bin stays whole. Not kept: scans by every wave for itself, one
// barrier a digit (14.4, and 10.9); tokens in turn of one bin counted at once (1 us more, though 15 less where all masses are equal,
// whose counts wait for one another).
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
  const int M = a.keep - a.first - a.recent, end = T - a.recent;   // M > 0 of the tokens first .. end - 1
  for (int i = tid; i < a.first; i += THREADS) kept[i] = i;
  for (int i = tid; i < a.recent; i += THREADS) kept[a.keep - a.recent + i] = end + i;
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
// Where the first and the last tokens are all that stay, which they are is plain: no launch has picked any, and K's workgroups
// write them down (one request of 2101 tokens 12.4 us of both calls, 15.4 with a launch that picks nothing; another kernel, since the
// picked tokens' moves lose 5 % by the condition).
//
// One workgroup for each new page and head, K or V. A lane makes 16 bytes of a block of 32 tokens x 32 dimensions: K's are
// two tokens' 8 dimensions, two loads of 8 bytes; V's are 8 tokens' 2 dimensions, and of each of them the 16 old bytes
// that hold them with 7 neighbours are loaded. Where a lane's tokens lie is found once for all blocks of dimensions.
//
// 27 requests cut to 2048 tokens, 8 heads of 128: 96 us. 236 MB are read and written, but a token's codes lie in 8 and 16 byte
// pieces among its neighbours': with every fourth token kept or more nearly every line of the old pages is fetched, 417 MB,
// 4.3 TB/s. Blocks taken whole to LDS and scattered from there, each line fetched once for sure: 167 us (the scatter writes
// single bytes).
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// the code in byte i of x, rounded to another scale: q + 1.5 2^23 rounds q to an integer, whose low byte is the code (q is a
// rounded product: fused with the sum, codes next to a half would go the other way)
__device__ __forceinline__ unsigned moved(unsigned x, int i, float r) {
#pragma clang fp contract(off)
  const float q = (float)((int)(x << (24 - 8 * i)) >> 24) * r;
  return __float_as_uint(q + 12582912.0f);
}
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// token i of those that stay where the first and the last are all of them
__device__ __forceinline__ int end_token(const EvictArgs& a, int T, int i) { return i < a.first ? i : T - a.keep + i; }

template <bool IS_V, bool ENDS>
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
    const int t = ENDS ? end_token(a, T, p * a.page + tid) : a.kept[((size_t)req * c.kv_heads + head) * a.keep + p * a.page + tid];
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

template <bool ENDS>
__global__ __launch_bounds__(256) void kv8_evict_move_kernel(EvictArgs a, Kv8Cache c, long units) {
  const int fresh = (a.keep + a.page - 1) / a.page;
  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    const long page = u >> 1;
    const int head = (int)(page % c.kv_heads), p = (int)(page / c.kv_heads % fresh), req = (int)(page / c.kv_heads / fresh);
    const int T = a.from_len[req];
    if (T <= a.keep || T > a.table_ld * a.page) continue;
    if (ENDS && (u & 1) == 0) {
      const int i = p * a.page + threadIdx.x;
      if ((int)threadIdx.x < a.page && i < a.keep) a.kept[((size_t)req * c.kv_heads + head) * a.keep + i] = end_token(a, T, i);
    }
    const int pid = a.table[(size_t)req * a.table_ld + p];
    if (pid < 0 || pid >= a.n_pages) continue;
    if (u & 1) move_page<true, ENDS>(a, c, req, p, pid, head);
    else move_page<false, ENDS>(a, c, req, p, pid, head);
    __syncthreads();
  }
}

hipError_t launch_kv8_evict(const EvictArgs& a, const Kv8Cache& c, hipStream_t s) {
  const dim3 picks((unsigned)(a.requests * c.kv_heads));
  const bool ends = a.first + a.recent == a.keep;
  if (!ends) {
    // the fewest waves that hold a request's tokens at once: their barriers are shorter (us of the kernel with 1024 threads / these:
    // one request of 2101 tokens 14.8 / 10.4, 32 of up to 8192 17.2 / 13.6)
    if (a.max_len <= 256 * kPickMost) hipLaunchKernelGGL(kv8_evict_pick_kernel<256>, picks, dim3(256), 0, s, a, c.kv_heads);
    else if (a.max_len <= 512 * kPickMost) hipLaunchKernelGGL(kv8_evict_pick_kernel<512>, picks, dim3(512), 0, s, a, c.kv_heads);
    else hipLaunchKernelGGL(kv8_evict_pick_kernel<1024>, picks, dim3(1024), 0, s, a, c.kv_heads);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const long units = 2L * a.requests * c.kv_heads * ((a.keep + a.page - 1) / a.page);
  hipLaunchKernelGGL(ends ? kv8_evict_move_kernel<true> : kv8_evict_move_kernel<false>, dim3((unsigned)std::min(units, 1L << 22)), dim3(256), 0, s, a, c, units);
  return hipGetLastError();
}

}  // namespace rehip
