// Argument blocks and host-side launchers of the batched serving step (serve.hip, kv8.hip), shared with
// their C ABI (serve_api.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <cstddef>
#include <cstdint>

namespace rehip {

// A ragged batch over pages: request b's rows are start[b] .. start[b] + count[b] - 1 of the row arrays
// (start ascending, ranges disjoint), its last row is position len[b] - 1, and token t of it lies in page
// table[b * table_ld + t / page] at place t % page. Entries outside 0 .. n_pages - 1 hold no page.
struct PagedBatch {
  const int* start;
  const int* count;
  const int* len;
  const int* table;
  int requests, rows, table_ld, page, n_pages;
};

// The int8 pages and their scales (n_pages x kv_heads each): codes of one page and head are
// [page / 32][hd / 32] blocks of 1 KiB in fragment order (kv8.hip).
struct Kv8Cache {
  int8_t* k;
  int8_t* v;
  float* ks;
  float* vs;
  int kv_heads, hd;
};

struct PlanArgs {
  const int* new_len;
  const int* len;
  int* table;
  int* free_pages;
  const int* n_free;
  int* len_out;
  int* n_free_out;
  int* start;
  int* count;
  int* seq;
  int* pos;
  int* slot;
  int* status;
  int requests, page, table_ld, n_pages, cap;
};

constexpr int kPlanMaxRequests = 4096;
constexpr int kPlanMaxNew = 1 << 18;       // new tokens of one request (the sum over all stays below 2^31)

struct RopeArgs {
  const float* x;
  float* out;
  const double* freqs;
  const int* pos;
  size_t ldx, ldo;
  float mscale;
  int rows, heads, hd, rot, interleaved;
};

struct LogprobArgs {
  const float* x;
  const int* targets;
  float* logprob;
  float* entropy;
  int* ids;
  float* top;
  float* work;
  size_t ld;
  int rows, vocab, k;
};

constexpr int kLogprobsMaxTop = 64;

struct Attn8Args {
  const float* q;
  float* ctx;
  float* work;
  size_t ldq;
  float scale;
  int window, heads, max_rows, max_len;
};

hipError_t launch_kv_plan(const PlanArgs& a, hipStream_t s);
hipError_t launch_rope_rows(const RopeArgs& a, hipStream_t s);
size_t logprobs_work_floats(int rows, int vocab, int k);
hipError_t launch_logprobs(const LogprobArgs& a, hipStream_t s);
hipError_t launch_kv8_append(const PagedBatch& b, const Kv8Cache& c, const float* k, int ldk, const float* v, int ldv,
                             hipStream_t s);
// workgroups of the call's first launch: at most kAttnMaxWorkgroups are taken (a launch has fewer than 2^32 threads)
constexpr size_t kAttnMaxWorkgroups = (size_t)1 << 23;
size_t attention_kv8_workgroups(int rows, int requests, int max_rows, int max_len, int heads, int kv_heads, int hd);
size_t attention_kv8_work_floats(int rows, int requests, int max_rows, int max_len, int heads, int kv_heads, int hd);
hipError_t launch_attention_kv8(const PagedBatch& b, const Kv8Cache& c, const Attn8Args& a, hipStream_t s);

// A request's place in the batch, in bounds whatever the arrays hold: rows row0 .. row0 + count - 1, tokens len.
struct RequestRows {
  int req, row0, count, len;
};
__device__ __forceinline__ RequestRows request_rows(int r, int start, int count, int len, int rows) {
  const int row0 = min(max(start, 0), rows);
  return {r, row0, min(max(count, 0), rows - row0), len};
}

// lane l's of a wave, in every lane (l the same in all of them)
__device__ __forceinline__ RequestRows lane_rows(const RequestRows& q, int l) {
  return {__builtin_amdgcn_readlane(q.req, l), __builtin_amdgcn_readlane(q.row0, l), __builtin_amdgcn_readlane(q.count, l),
          __builtin_amdgcn_readlane(q.len, l)};
}

// Request of unit u, where request b owns the units from start[b] / div + mult * b on: the last one whose first unit is
// at most u (req -1: none; of starts that do not ascend, any one). Every wave looks at 64 requests at a time, a lane each,
// spread over the range that is left: one trip to memory up to 64 requests, two up to 4096, and nothing goes through LDS.
__device__ __forceinline__ RequestRows request_of_unit(int u, const PagedBatch& b, int div, int mult) {
  const int lane = threadIdx.x & 63;
  int base = 0, n = b.requests;
  while (n > 64) {
    const int step = (n + 63) >> 6, i = base + lane * step;
    const int row0 = min(max(b.start[min(i, b.requests - 1)], 0), b.rows);
    const int k = __popcll(__ballot(lane * step < n && row0 / div + mult * i <= u));
    if (k == 0) return {-1, 0, 0, 0};
    base += (k - 1) * step;
    n = min(step, n - (k - 1) * step);
  }
  const int r = base + min(lane, n - 1);
  const RequestRows q = request_rows(r, b.start[r], b.count[r], b.len[r], b.rows);
  const int k = __popcll(__ballot(lane < n && q.row0 / div + mult * r <= u));
  return k == 0 ? RequestRows{-1, 0, 0, 0} : lane_rows(q, k - 1);
}

}  // namespace rehip
