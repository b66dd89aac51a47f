// C ABI of the batched serving step (include/rehip.h): argument checks, then the launchers of serve.hip, kv8.hip,
// kv8_keep.hip, kv_pages.hip and draft.hip. Nothing here allocates, so every call may be captured into a graph.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/rehip.h"
#include "serve.hpp"

namespace rehip {
int report_error(int code, const char* fmt, ...);
}

using namespace rehip;

namespace {

#define HIP_TRY(expr)                                                                              \
  do {                                                                                             \
    hipError_t e_ = (expr);                                                                        \
    if (e_ != hipSuccess) return report_error(RE_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
  } while (0)

bool a16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// the batch and the cache that append and attention share
int paged_args(size_t rows, size_t requests, const int* start, const int* count, const int* len, const int* table,
               size_t table_ld, size_t page, size_t n_pages, const int8_t* k, const int8_t* v, const float* ks,
               const float* vs, size_t kv_heads, size_t hd) {
  if (!start || !count || !len || !table || !k || !v || !ks || !vs) return report_error(RE_ERR_ARG, "null pointer");
  if (rows > (1u << 22) || requests > (1u << 16))
    return report_error(RE_ERR_SIZE, "batch of %zu rows, %zu requests (up to 4194304, 65536)", rows, requests);
  if (page == 0 || page % 32 || page > 256 || hd == 0 || hd % 32 || hd > 256)
    return report_error(RE_ERR_SIZE, "page %zu and head_dim %zu: multiples of 32 up to 256", page, hd);
  if (kv_heads == 0 || kv_heads > 1024) return report_error(RE_ERR_SIZE, "%zu KV heads (1 .. 1024)", kv_heads);
  if (table_ld == 0 || table_ld * page > (1u << 30) || n_pages == 0 || n_pages > (1u << 30) / page)
    return report_error(RE_ERR_SIZE, "table of %zu columns, %zu pages of %zu tokens (tokens up to 2^30)", table_ld,
                        n_pages, page);
  if (!a16(k) || !a16(v)) return report_error(RE_ERR_ARG, "codes must be 16-byte aligned");
  return RE_OK;
}

// pages, tables and the stack of free pages, of up to kPlanMaxRequests requests
int pool_args(size_t requests, size_t page, size_t table_ld, size_t n_pages) {
  if (requests == 0 || requests > (size_t)kPlanMaxRequests)
    return report_error(RE_ERR_SIZE, "pages of %zu requests (1 .. %d)", requests, kPlanMaxRequests);
  if (page == 0 || page > (1u << 16) || table_ld == 0 || table_ld > (1u << 30) / page || n_pages == 0 ||
      n_pages > (1u << 30) / page)
    return report_error(RE_ERR_SIZE, "table of %zu columns, %zu pages of %zu tokens (tokens up to 2^30)", table_ld,
                        n_pages, page);
  if (requests * table_ld > (1u << 30))
    return report_error(RE_ERR_SIZE, "table of %zu x %zu entries (up to 2^30)", requests, table_ld);
  return RE_OK;
}

// causal attention over the pages, with sinks and the rows' sums of exponentials where they are asked for
int attention_kv8(const float* d_q, size_t ldq, size_t rows, size_t requests, const int* d_row_start,
                  const int* d_row_count, const int* d_kv_len, const int* d_table, size_t table_ld, size_t page,
                  size_t n_pages, const int8_t* d_kcodes, const int8_t* d_vcodes, const float* d_kscale,
                  const float* d_vscale, size_t max_rows, size_t max_len, size_t n_heads, size_t n_kv_heads,
                  size_t head_dim, float scale, size_t window, size_t sinks, float* d_ctx, float* d_lse, void* d_work,
                  size_t work_bytes, void* stream) {
  if (!d_q || !d_ctx) return report_error(RE_ERR_ARG, "null pointer");
  int rc = paged_args(rows, requests, d_row_start, d_row_count, d_kv_len, d_table, table_ld, page, n_pages, d_kcodes,
                      d_vcodes, d_kscale, d_vscale, n_kv_heads, head_dim);
  if (rc) return rc;
  if (n_heads == 0 || n_heads % n_kv_heads || n_heads > 8192 || ldq < n_heads * head_dim || ldq % 4 ||
      ldq > (1u << 30))
    return report_error(RE_ERR_SIZE, "attention heads %zu/%zu of %zu, q stride %zu (a multiple of 4)", n_heads,
                        n_kv_heads, head_dim, ldq);
  if (!std::isfinite(scale)) return report_error(RE_ERR_ARG, "attention scale %g", (double)scale);
  if (sinks > kAttnMaxSinks) return report_error(RE_ERR_SIZE, "%zu sinks (up to %zu)", sinks, kAttnMaxSinks);
  if (!a16(d_q) || !a16(d_ctx) || !a16(d_work))
    return report_error(RE_ERR_ARG, "q, ctx and workspace must be 16-byte aligned");
  if (rows == 0 || requests == 0) return RE_OK;
  if (max_rows == 0) return report_error(RE_ERR_SIZE, "max_rows 0 for %zu rows", rows);
  const size_t ml = max_len < (1u << 30) ? max_len : (1u << 30), mr = max_rows < rows ? max_rows : rows;
  if (attention_kv8_workgroups((int)rows, (int)requests, (int)mr, (int)ml, (int)n_heads, (int)n_kv_heads,
                               (int)head_dim) > kAttnMaxWorkgroups)
    return report_error(RE_ERR_SIZE, "attention of %zu rows and %zu requests with %zu heads is too large for one call",
                        rows, requests, n_heads);
  const size_t need = re_attention_kv8_work_bytes(rows, requests, max_rows, max_len, n_heads, n_kv_heads, head_dim);
  if (need && !d_work) return report_error(RE_ERR_ARG, "null workspace, need %zu bytes", need);
  if (work_bytes < need) return report_error(RE_ERR_SIZE, "attention workspace of %zu bytes, need %zu", work_bytes, need);
  const PagedBatch b{d_row_start, d_row_count, d_kv_len, d_table, (int)requests, (int)rows, (int)table_ld, (int)page,
                     (int)n_pages};
  const Kv8Cache c{const_cast<int8_t*>(d_kcodes), const_cast<int8_t*>(d_vcodes), const_cast<float*>(d_kscale),
                   const_cast<float*>(d_vscale), (int)n_kv_heads, (int)head_dim};
  const Attn8Args a{d_q, d_ctx, (float*)d_work, ldq, scale, (int)(window < (1u << 30) ? window : (1u << 30)),
                    (int)n_heads, (int)mr, (int)ml, (int)sinks, d_lse};
  HIP_TRY(launch_attention_kv8(b, c, a, (hipStream_t)stream));
  return RE_OK;
}

}  // namespace

extern "C" {

int re_kv_plan_dev(size_t requests, size_t page, const int* d_new_len, const int* d_kv_len, int* d_table,
                   size_t table_ld, int* d_free, size_t n_pages, const int* d_n_free, int* d_kv_len_out,
                   int* d_n_free_out, int* d_row_start, int* d_row_count, size_t row_cap, int* d_row_seq,
                   int* d_row_pos, int* d_row_slot, int* d_status, void* stream) {
  if (!d_new_len || !d_kv_len || !d_table || !d_free || !d_n_free || !d_kv_len_out || !d_n_free_out || !d_row_start ||
      !d_row_count || !d_status || (row_cap && (!d_row_seq || !d_row_pos || !d_row_slot)))
    return report_error(RE_ERR_ARG, "null pointer");
  if (requests == 0 || requests > (size_t)kPlanMaxRequests || row_cap > (1u << 22))
    return report_error(RE_ERR_SIZE, "plan of %zu requests, %zu rows (1 .. %d, up to 4194304)", requests, row_cap,
                        kPlanMaxRequests);
  if (page == 0 || page > (1u << 16) || table_ld == 0 || table_ld > (1u << 30) / page || n_pages == 0 ||
      n_pages > (1u << 30) / page)
    return report_error(RE_ERR_SIZE, "table of %zu columns, %zu pages of %zu tokens (tokens up to 2^30)", table_ld,
                        n_pages, page);
  if (requests * table_ld > (1u << 30))
    return report_error(RE_ERR_SIZE, "table of %zu x %zu entries (up to 2^30)", requests, table_ld);
  const PlanArgs a{d_new_len,   d_kv_len,  d_table,   d_free,     d_n_free, d_kv_len_out, d_n_free_out,
                   d_row_start, d_row_count, d_row_seq, d_row_pos, d_row_slot, d_status, (int)requests,
                   (int)page,   (int)table_ld, (int)n_pages, (int)row_cap};
  HIP_TRY(launch_kv_plan(a, (hipStream_t)stream));
  return RE_OK;
}

int re_rope_freqs(double theta, size_t rot_dim, int scaling, double factor, double trained_len, double p0, double p1,
                  double* freqs, float* mscale) {
  if (!freqs || !mscale) return report_error(RE_ERR_ARG, "null pointer");
  if (rot_dim == 0 || rot_dim % 2 || rot_dim > 256)
    return report_error(RE_ERR_SIZE, "rotary size %zu: even, up to 256", rot_dim);
  if (!(theta > 1.0) || !std::isfinite(theta)) return report_error(RE_ERR_ARG, "rotary base %g", theta);
  if (scaling != RE_ROPE_NONE && (!(factor >= 1.0) || !std::isfinite(factor)))
    return report_error(RE_ERR_ARG, "rotary scaling factor %g", factor);
  if ((scaling == RE_ROPE_YARN || scaling == RE_ROPE_BANDS) &&
      (!(trained_len > 0.0) || !std::isfinite(trained_len) || !(p0 > 0.0) || !(p1 > 0.0) || !std::isfinite(p0) ||
       !std::isfinite(p1)))
    return report_error(RE_ERR_ARG, "rotary scaling over %g positions, %g and %g turns", trained_len, p0, p1);
  if (scaling == RE_ROPE_BANDS && !(p0 < p1))
    return report_error(RE_ERR_ARG, "rotary bands: %g turns must be below %g", p0, p1);
  if (scaling == RE_ROPE_NTK && rot_dim == 2) return report_error(RE_ERR_SIZE, "rotary base scaling needs 2 pairs");
  const double pi2 = 6.283185307179586477, d = (double)rot_dim;
  float m = 1.0f;
  double low = 0.0, high = 0.0;
  switch (scaling) {
    case RE_ROPE_NONE:
    case RE_ROPE_LINEAR:
    case RE_ROPE_BANDS:
      break;
    case RE_ROPE_NTK:
      theta *= std::pow(factor, d / (d - 2.0));
      break;
    case RE_ROPE_YARN: {
      // the pairs that make p0 (fast) and p1 (slow) turns over the trained positions
      auto pair_at = [&](double turns) { return d * std::log(trained_len / (turns * pi2)) / (2.0 * std::log(theta)); };
      low = std::fmax(std::floor(pair_at(p0)), 0.0);
      high = std::fmin(std::ceil(pair_at(p1)), d - 1.0);
      m = (float)(0.1 * std::log(factor) + 1.0);
      break;
    }
    default:
      return report_error(RE_ERR_ARG, "unknown rotary scaling %d", scaling);
  }
  for (size_t i = 0; i < rot_dim / 2; ++i) {
    double f = std::pow(theta, -2.0 * (double)i / d);
    if (scaling == RE_ROPE_LINEAR) f /= factor;
    if (scaling == RE_ROPE_YARN) {
      const double ramp = std::fmin(std::fmax(((double)i - low) / std::fmax(high - low, 1e-3), 0.0), 1.0);
      f = f * (1.0 - ramp) + f / factor * ramp;
    }
    if (scaling == RE_ROPE_BANDS) {
      const double keep = std::fmin(std::fmax((trained_len * f / pi2 - p0) / (p1 - p0), 0.0), 1.0);
      f = f * keep + f / factor * (1.0 - keep);
    }
    freqs[i] = f;
  }
  *mscale = m;
  return RE_OK;
}

int re_rope_rows_dev(const float* d_x, size_t ldx, size_t rows, size_t heads, size_t head_dim, size_t rot_dim,
                     int layout, const double* d_freqs, float mscale, const int* d_pos, float* d_out, size_t ldo,
                     void* stream) {
  if (!d_x || !d_freqs || !d_pos || !d_out) return report_error(RE_ERR_ARG, "null pointer");
  if (layout != RE_ROPE_HALF && layout != RE_ROPE_INTERLEAVED)
    return report_error(RE_ERR_ARG, "unknown rotary layout %d", layout);
  if (rows == 0 || heads == 0) return RE_OK;
  if (rows > (1u << 22) || heads > 65535 || head_dim == 0 || head_dim > 256 || rot_dim == 0 || rot_dim % 2 ||
      rot_dim > head_dim || ldx < heads * head_dim || ldo < heads * head_dim || ldx > (1u << 30) || ldo > (1u << 30))
    return report_error(RE_ERR_SIZE, "rope shape rows %zu heads %zu head_dim %zu (up to 256) rotary %zu (even) strides "
                        "%zu/%zu", rows, heads, head_dim, rot_dim, ldx, ldo);
  if (d_x == d_out && ldx != ldo) return report_error(RE_ERR_ARG, "rope in place needs one stride, not %zu and %zu", ldx, ldo);
  const RopeArgs a{d_x, d_out, d_freqs, d_pos, ldx, ldo, mscale, (int)rows, (int)heads, (int)head_dim, (int)rot_dim,
                   layout == RE_ROPE_INTERLEAVED};
  HIP_TRY(launch_rope_rows(a, (hipStream_t)stream));
  return RE_OK;
}

int re_kv8_append_dev(const float* d_k, size_t ldk, const float* d_v, size_t ldv, size_t rows, size_t requests,
                      const int* d_row_start, const int* d_row_count, const int* d_kv_len, const int* d_table,
                      size_t table_ld, size_t page, size_t n_pages, int8_t* d_kcodes, int8_t* d_vcodes,
                      float* d_kscale, float* d_vscale, size_t n_kv_heads, size_t head_dim, void* stream) {
  if (!d_k || !d_v) return report_error(RE_ERR_ARG, "null pointer");
  int rc = paged_args(rows, requests, d_row_start, d_row_count, d_kv_len, d_table, table_ld, page, n_pages, d_kcodes,
                      d_vcodes, d_kscale, d_vscale, n_kv_heads, head_dim);
  if (rc) return rc;
  if (ldk < n_kv_heads * head_dim || ldv < n_kv_heads * head_dim || ldk % 4 || ldv % 4 || ldk > (1u << 22) ||
      ldv > (1u << 22))
    return report_error(RE_ERR_SIZE, "append strides %zu/%zu (multiples of 4, %zu .. 4194304)", ldk, ldv,
                        n_kv_heads * head_dim);
  if (!a16(d_k) || !a16(d_v)) return report_error(RE_ERR_ARG, "k and v must be 16-byte aligned");
  if (rows == 0 || requests == 0) return RE_OK;
  const PagedBatch b{d_row_start, d_row_count, d_kv_len, d_table, (int)requests, (int)rows, (int)table_ld, (int)page,
                     (int)n_pages};
  const Kv8Cache c{d_kcodes, d_vcodes, d_kscale, d_vscale, (int)n_kv_heads, (int)head_dim};
  HIP_TRY(launch_kv8_append(b, c, d_k, (int)ldk, d_v, (int)ldv, (hipStream_t)stream));
  return RE_OK;
}

size_t re_attention_kv8_work_bytes(size_t rows, size_t requests, size_t max_rows, size_t max_len, size_t n_heads,
                                   size_t n_kv_heads, size_t head_dim) {
  if (rows == 0 || requests == 0 || max_rows == 0 || n_heads == 0 || n_kv_heads == 0 || n_heads % n_kv_heads ||
      rows > (1u << 22) || requests > (1u << 16) || n_heads > 8192 || head_dim > 256)
    return 0;
  const size_t mr = max_rows < rows ? max_rows : rows, ml = max_len < (1u << 30) ? max_len : (1u << 30);
  return attention_kv8_work_floats((int)rows, (int)requests, (int)mr, (int)ml, (int)n_heads, (int)n_kv_heads,
                                   (int)head_dim) * sizeof(float);
}

int re_attention_kv8_dev(const float* d_q, size_t ldq, size_t rows, size_t requests, const int* d_row_start,
                         const int* d_row_count, const int* d_kv_len, const int* d_table, size_t table_ld, size_t page,
                         size_t n_pages, const int8_t* d_kcodes, const int8_t* d_vcodes, const float* d_kscale,
                         const float* d_vscale, size_t max_rows, size_t max_len, size_t n_heads, size_t n_kv_heads,
                         size_t head_dim, float scale, size_t window, float* d_ctx, void* d_work, size_t work_bytes,
                         void* stream) {
  return attention_kv8(d_q, ldq, rows, requests, d_row_start, d_row_count, d_kv_len, d_table, table_ld, page, n_pages,
                       d_kcodes, d_vcodes, d_kscale, d_vscale, max_rows, max_len, n_heads, n_kv_heads, head_dim, scale,
                       window, 0, d_ctx, nullptr, d_work, work_bytes, stream);
}

int re_attention_kv8_sinks_dev(const float* d_q, size_t ldq, size_t rows, size_t requests, const int* d_row_start,
                               const int* d_row_count, const int* d_kv_len, const int* d_table, size_t table_ld,
                               size_t page, size_t n_pages, const int8_t* d_kcodes, const int8_t* d_vcodes,
                               const float* d_kscale, const float* d_vscale, size_t max_rows, size_t max_len,
                               size_t n_heads, size_t n_kv_heads, size_t head_dim, float scale, size_t window,
                               size_t sinks, float* d_ctx, float* d_lse, void* d_work, size_t work_bytes, void* stream) {
  return attention_kv8(d_q, ldq, rows, requests, d_row_start, d_row_count, d_kv_len, d_table, table_ld, page, n_pages,
                       d_kcodes, d_vcodes, d_kscale, d_vscale, max_rows, max_len, n_heads, n_kv_heads, head_dim, scale,
                       window, sinks, d_ctx, d_lse, d_work, work_bytes, stream);
}

int re_kv8_mass_dev(const float* d_q, size_t ldq, const float* d_lse, size_t rows, size_t requests,
                    const int* d_row_start, const int* d_row_count, const int* d_kv_len, const int* d_table,
                    size_t table_ld, size_t page, size_t n_pages, const int8_t* d_kcodes, const float* d_kscale,
                    size_t max_rows, size_t max_len, size_t n_heads, size_t n_kv_heads, size_t head_dim, float scale,
                    size_t window, size_t sinks, float* d_mass, void* stream) {
  if (!d_q || !d_lse || !d_mass) return report_error(RE_ERR_ARG, "null pointer");
  int rc = paged_args(rows, requests, d_row_start, d_row_count, d_kv_len, d_table, table_ld, page, n_pages, d_kcodes,
                      d_kcodes, d_kscale, d_kscale, n_kv_heads, head_dim);
  if (rc) return rc;
  if (n_heads == 0 || n_heads % n_kv_heads || n_heads > 8192 || ldq < n_heads * head_dim || ldq % 4 ||
      ldq > (1u << 30))
    return report_error(RE_ERR_SIZE, "attention heads %zu/%zu of %zu, q stride %zu (a multiple of 4)", n_heads,
                        n_kv_heads, head_dim, ldq);
  if (!std::isfinite(scale)) return report_error(RE_ERR_ARG, "attention scale %g", (double)scale);
  if (sinks > kAttnMaxSinks) return report_error(RE_ERR_SIZE, "%zu sinks (up to %zu)", sinks, kAttnMaxSinks);
  if (!a16(d_q) || !a16(d_mass)) return report_error(RE_ERR_ARG, "q and masses must be 16-byte aligned");
  if (rows == 0 || requests == 0) return RE_OK;
  if (max_rows == 0) return report_error(RE_ERR_SIZE, "max_rows 0 for %zu rows", rows);
  const size_t ml = max_len < (1u << 30) ? max_len : (1u << 30), mr = max_rows < rows ? max_rows : rows;
  if (mr * (n_heads / n_kv_heads) > (1u << 30) || requests * n_kv_heads > kMassMaxWorkgroups)
    return report_error(RE_ERR_SIZE, "weights of %zu rows and %zu requests with %zu heads are too many for one call", rows,
                        requests, n_heads);
  const PagedBatch b{d_row_start, d_row_count, d_kv_len, d_table, (int)requests, (int)rows, (int)table_ld, (int)page,
                     (int)n_pages};
  const Kv8Cache c{const_cast<int8_t*>(d_kcodes), nullptr, const_cast<float*>(d_kscale), nullptr, (int)n_kv_heads,
                   (int)head_dim};
  const MassArgs a{d_q, d_lse, d_mass, ldq, scale, (int)(window < (1u << 30) ? window : (1u << 30)), (int)sinks,
                   (int)n_heads, (int)mr, (int)ml};
  HIP_TRY(launch_kv8_mass(b, c, a, (hipStream_t)stream));
  return RE_OK;
}

int re_kv_evict_plan_dev(size_t requests, size_t page, size_t limit, size_t keep, const int* d_kv_len,
                         const int* d_table, size_t table_ld, const int* d_free, size_t n_pages, const int* d_n_free,
                         int* d_kv_len_out, int* d_table_out, int* d_free_out, int* d_n_free_out, int* d_from_len,
                         int* d_from_table, int* d_dropped, int* d_status, void* stream) {
  if (!d_kv_len || !d_table || !d_free || !d_n_free || !d_kv_len_out || !d_table_out || !d_free_out || !d_n_free_out ||
      !d_from_len || !d_from_table || !d_status)
    return report_error(RE_ERR_ARG, "null pointer");
  int rc = pool_args(requests, page, table_ld, n_pages);
  if (rc) return rc;
  if (keep == 0 || keep > limit || keep > (1u << 30))
    return report_error(RE_ERR_SIZE, "%zu of %zu tokens to keep (1 .. that, up to 2^30)", keep, limit);
  if (d_table_out == d_from_table)
    return report_error(RE_ERR_ARG, "the old table and the new one must be two buffers");
  if (d_from_len == d_kv_len || d_from_len == d_kv_len_out)
    return report_error(RE_ERR_ARG, "the cut requests' old lengths must be a buffer of their own");
  const EvictPlanArgs a{d_kv_len, d_table, d_free, d_n_free, d_kv_len_out, d_table_out, d_free_out, d_n_free_out,
                        d_from_len, d_from_table, d_dropped, d_status, (int)requests, (int)page, (int)table_ld,
                        (int)n_pages, (int)(limit < (1u << 30) ? limit : (1u << 30)), (int)keep};
  HIP_TRY(launch_kv_evict_plan(a, (hipStream_t)stream));
  return RE_OK;
}

int re_kv8_evict_dev(size_t requests, const int* d_from_len, const int* d_from_table, const int* d_table,
                     size_t table_ld, size_t page, size_t n_pages, int8_t* d_kcodes, int8_t* d_vcodes, float* d_kscale,
                     float* d_vscale, float* d_mass, size_t n_kv_heads, size_t head_dim, size_t keep, size_t first,
                     size_t recent, size_t max_len, int* d_kept, void* stream) {
  if (!d_kept) return report_error(RE_ERR_ARG, "null pointer");
  int rc = paged_args(0, requests, d_from_len, d_from_len, d_from_table, d_table, table_ld, page, n_pages, d_kcodes,
                      d_vcodes, d_kscale, d_vscale, n_kv_heads, head_dim);
  if (rc) return rc;
  rc = pool_args(requests, page, table_ld, n_pages);
  if (rc) return rc;
  if (d_table == d_from_table) return report_error(RE_ERR_ARG, "the old table and the new one must be two buffers");
  if (keep == 0 || keep > (1u << 30) || first > keep || recent > keep - first)
    return report_error(RE_ERR_SIZE, "%zu first and %zu last tokens of %zu to keep (up to 2^30)", first, recent, keep);
  if (!a16(d_mass)) return report_error(RE_ERR_ARG, "masses must be 16-byte aligned");
  if (!d_mass && first + recent < keep)
    return report_error(RE_ERR_ARG, "without masses the first and last tokens must be all of the %zu to keep", keep);
  const size_t pages = (keep + page - 1) / page;
  if (requests * n_kv_heads > (1u << 21) || requests * n_kv_heads > (1u << 30) / pages)
    return report_error(RE_ERR_SIZE, "%zu requests of %zu KV heads and %zu tokens are too many for one call", requests,
                        n_kv_heads, keep);
  const Kv8Cache c{d_kcodes, d_vcodes, d_kscale, d_vscale, (int)n_kv_heads, (int)head_dim};
  const EvictArgs a{d_from_len, d_from_table, d_table, d_mass, d_kept, (int)requests, (int)table_ld, (int)page,
                    (int)n_pages, (int)keep, (int)first, (int)recent, (int)(max_len < (1u << 30) ? max_len : (1u << 30))};
  HIP_TRY(launch_kv8_evict(a, c, (hipStream_t)stream));
  return RE_OK;
}

int re_kv_rewind_dev(size_t requests, size_t page, const int* d_back, const int* d_kv_len, const int* d_table,
                     size_t table_ld, int* d_free, size_t n_pages, const int* d_n_free, int* d_kv_len_out,
                     int* d_n_free_out, void* stream) {
  if (!d_back || !d_kv_len || !d_table || !d_free || !d_n_free || !d_kv_len_out || !d_n_free_out)
    return report_error(RE_ERR_ARG, "null pointer");
  int rc = pool_args(requests, page, table_ld, n_pages);
  if (rc) return rc;
  const RewindArgs a{d_back, d_kv_len, d_table, d_free, d_n_free, d_kv_len_out, d_n_free_out, (int)requests, (int)page,
                     (int)table_ld, (int)n_pages};
  HIP_TRY(launch_kv_rewind(a, (hipStream_t)stream));
  return RE_OK;
}

int re_kv_positions_dev(size_t rows, const int* d_row_seq, const int* d_row_pos, size_t requests, const int* d_dropped,
                        int* d_out, void* stream) {
  if (!d_row_seq || !d_row_pos || !d_dropped || !d_out) return report_error(RE_ERR_ARG, "null pointer");
  if (rows > (1u << 22) || requests == 0 || requests > (1u << 16))
    return report_error(RE_ERR_SIZE, "positions of %zu rows, %zu requests (up to 4194304, 1 .. 65536)", rows, requests);
  if (rows == 0) return RE_OK;
  HIP_TRY(launch_kv_positions(d_row_seq, d_row_pos, (int)rows, d_dropped, (int)requests, d_out, (hipStream_t)stream));
  return RE_OK;
}

size_t re_draft_verify_work_bytes(size_t rows, size_t requests, size_t vocab) {
  if (rows == 0 || requests == 0 || vocab == 0 || rows > (1u << 22) || requests > (1u << 16) || vocab > (1u << 24)) return 0;
  return verify_work_bytes((int)rows, (int)requests, (int)vocab);
}

int re_draft_verify_dev(const float* d_logits, size_t ld, size_t rows, size_t vocab, size_t requests,
                        const int* d_row_start, const int* d_row_count, const int* d_tokens, const float* d_probs,
                        size_t ldp, const float* d_temperature, const float* d_accept_u, const float* d_sample_u,
                        int* d_accepted, int* d_back, int* d_out_tokens, void* d_work, size_t work_bytes, void* stream) {
  if (!d_logits || !d_row_start || !d_row_count || !d_tokens || !d_accept_u || !d_sample_u || !d_accepted || !d_back ||
      !d_out_tokens)
    return report_error(RE_ERR_ARG, "null pointer");
  if (vocab == 0 || vocab > (1u << 24) || ld < vocab || ld > (1u << 30) || rows > (1u << 22) || requests > (1u << 16))
    return report_error(RE_ERR_SIZE, "drafts of %zu requests over %zu rows of %zu logits, stride %zu", requests, rows, vocab,
                        ld);
  if (d_probs && (ldp < vocab || ldp > (1u << 30)))
    return report_error(RE_ERR_SIZE, "drafts' probabilities of %zu tokens, stride %zu", vocab, ldp);
  if (!a16(d_work)) return report_error(RE_ERR_ARG, "workspace must be 16-byte aligned");
  if (requests == 0) return RE_OK;
  if (rows == 0) return report_error(RE_ERR_SIZE, "no rows for %zu requests", requests);
  const size_t need = re_draft_verify_work_bytes(rows, requests, vocab);
  if (!d_work) return report_error(RE_ERR_ARG, "null workspace, need %zu bytes", need);
  if (work_bytes < need) return report_error(RE_ERR_SIZE, "draft workspace of %zu bytes, need %zu", work_bytes, need);
  if (d_out_tokens < d_tokens + rows && d_tokens < d_out_tokens + rows)
    return report_error(RE_ERR_ARG, "the tokens that come out must be a buffer apart from the drafted ones");
  const VerifyArgs a{d_logits, d_row_start, d_row_count, d_tokens, d_probs, d_temperature, d_accept_u, d_sample_u,
                     d_accepted, d_back, d_out_tokens, d_work, ld, ldp, (int)rows, (int)vocab, (int)requests};
  HIP_TRY(launch_verify(a, (hipStream_t)stream));
  return RE_OK;
}

size_t re_logprobs_work_bytes(size_t rows, size_t vocab, size_t top_k) {
  if (rows == 0 || vocab == 0 || rows > (1u << 22) || vocab > (1u << 24) || top_k > (size_t)kLogprobsMaxTop) return 0;
  return logprobs_work_floats((int)rows, (int)vocab, (int)top_k) * sizeof(float);
}

int re_logprobs_dev(const float* d_logits, size_t ld, size_t rows, size_t vocab, const int* d_targets, size_t top_k,
                    float* d_logprob, float* d_entropy, int* d_top_ids, float* d_top_logprobs, void* d_work,
                    size_t work_bytes, void* stream) {
  if (!d_logits || (d_logprob && !d_targets) || (top_k && (!d_top_ids || !d_top_logprobs)))
    return report_error(RE_ERR_ARG, "null pointer");
  if (vocab == 0 || vocab > (1u << 24) || ld < vocab || ld > (1u << 30) || rows > (1u << 22))
    return report_error(RE_ERR_SIZE, "log probabilities of %zu rows of %zu logits, stride %zu", rows, vocab, ld);
  if (top_k > (size_t)kLogprobsMaxTop || top_k > vocab)
    return report_error(RE_ERR_SIZE, "top %zu of %zu logits (up to %d)", top_k, vocab, kLogprobsMaxTop);
  if (!a16(d_work)) return report_error(RE_ERR_ARG, "workspace must be 16-byte aligned");
  if (rows == 0) return RE_OK;
  const size_t need = re_logprobs_work_bytes(rows, vocab, top_k);
  if (need && !d_work) return report_error(RE_ERR_ARG, "null workspace, need %zu bytes", need);
  if (work_bytes < need)
    return report_error(RE_ERR_SIZE, "log probability workspace of %zu bytes, need %zu", work_bytes, need);
  const LogprobArgs a{d_logits, d_targets, d_logprob, d_entropy, d_top_ids, d_top_logprobs, (float*)d_work, ld,
                      (int)rows, (int)vocab, (int)top_k};
  HIP_TRY(launch_logprobs(a, (hipStream_t)stream));
  return RE_OK;
}

}  // extern "C"
