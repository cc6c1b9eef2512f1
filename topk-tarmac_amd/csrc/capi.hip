// extern "C" boundary of libtarmac.so: argument validation, launch-shape
// policy, error reporting. Declarations and reference citations: include/tarmac.h.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/tarmac.h"
#include "tarmac_internal.hpp"

namespace {

thread_local std::string g_last_error;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

int ok() {
  g_last_error.clear();
  return TARMAC_OK;
}

int hip_status(hipError_t e, const char* what) {
  if (e != hipSuccess) return fail(TARMAC_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  return ok();
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

constexpr size_t kLdsBudget = 64 * 1024;
constexpr size_t kBf16TopkLds = 49 * 1024;
// Head width 128: a 64-key block of fp32 keys and transposed values takes
// 69 KB, so those rows may use up to 80 KB (two workgroups per CU; gfx950
// has 160 KB of LDS per CU).
size_t lds_budget(int d) { return d > 64 ? 80 * 1024 : kLdsBudget; }
// Dense rows staged whole take the fixed exponent offset (no running
// maximum), so the dense kernel may use 80 KB (two workgroups per CU): rows
// of 512 keys at d = 32 then fit one chunk (bf16 B=4096 N=512: 334 -> 242
// us). At d = 64 the 256-key rows that would then fit ran slower at
// B >= 1024 (156 -> 163 us) than two chunks at 64 KB.
size_t dense_lds_budget(int d) { return d == 64 ? kLdsBudget : 80 * 1024; }
constexpr int kZorderMaxN = 4096;  // agents per row the Morton selector sorts
constexpr size_t kZorderLds = 160 * 1024;  // LDS per workgroup on gfx950

float inv_sqrt(int d) { return static_cast<float>(1.0 / std::sqrt(static_cast<double>(d))); }

int check_core(const void* q, const void* k, const void* v, const void* out, int B, int N, int d,
               int dtype, const char* fn) {
  if (!q || !k || !v || !out) return fail(TARMAC_ERR_INVALID, "%s: null tensor pointer", fn);
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
    return fail(TARMAC_ERR_INVALID, "%s: q, k, v and out must be 16-byte aligned", fn);
  if (B < 1 || N < 2)
    return fail(TARMAC_ERR_INVALID, "%s: need B >= 1 and N >= 2 (got B=%d, N=%d)", fn, B, N);
  if (dtype == tarmac::kF32) {
    if (d != 8 && d != 16 && d != 32 && d != 64 && d != 128)
      return fail(TARMAC_ERR_UNSUPPORTED, "%s: fp32 head dim must be 8, 16, 32, 64 or 128 (got %d)",
                  fn, d);
  } else if (dtype == tarmac::kBf16) {
    if (d != 16 && d != 32 && d != 64 && d != 128)
      return fail(TARMAC_ERR_UNSUPPORTED, "%s: bf16 head dim must be 16, 32, 64 or 128 (got %d)",
                  fn, d);
  } else {
    return fail(TARMAC_ERR_INVALID, "%s: unknown dtype %d", fn, dtype);
  }
  if (static_cast<long long>(B) * N * d >= (1ll << 40))
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: tensor too large", fn);
  return TARMAC_OK;
}

// Largest multiple of 64 keys whose padded LDS copy fits the budget.
int max_topk_chunk(int dtype, int d) {
  int kc = 64;
  while (tarmac::topk_lds_bytes(dtype, d, kc + 64) <= lds_budget(d)) kc += 64;
  return kc;
}

int topk_common(const void* q, const void* k, const void* v, void* out, int32_t* idx_out, int B,
                int N, int d, int topk, int dtype, int key_chunk, void* stream, const char* fn) {
  int rc = check_core(q, k, v, out, B, N, d, dtype, fn);
  if (rc) return rc;
  if (topk < 1 || topk > N - 1)
    return fail(TARMAC_ERR_INVALID, "%s: need 1 <= topk <= N-1 (got topk=%d, N=%d)", fn, topk, N);
  if (idx_out && !aligned(idx_out, 4)) return fail(TARMAC_ERR_INVALID, "%s: idx_out misaligned", fn);
  if (topk > tarmac::kTopkSmallMax && N + topk > 16384)
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: topk > 8 needs N + topk <= 16384", fn);
  const int kmax = max_topk_chunk(dtype, d);
  const int n64 = (N + 63) / 64 * 64;
  int kc;
  if (key_chunk <= 0) {
    kc = n64 < kmax ? n64 : kmax;
    // bf16: keep the key copy within 49 KiB so three workgroups share a CU
    // (a whole 512-key row at d = 64 would allow two; a whole 1024-key row
    // at d = 16, 48 KiB of rows, runs 1.2x faster than 832-key chunks)
    if (dtype == tarmac::kBf16)
      while (kc > 64 && tarmac::topk_lds_bytes(dtype, d, kc) > kBf16TopkLds) kc -= 64;
  } else {
    if (key_chunk % 16 != 0)
      return fail(TARMAC_ERR_INVALID, "%s: key_chunk must be a multiple of 16 (got %d)", fn, key_chunk);
    if (tarmac::topk_lds_bytes(dtype, d, key_chunk) > lds_budget(d))
      return fail(TARMAC_ERR_UNSUPPORTED, "%s: key_chunk %d exceeds the LDS budget (max %d at d=%d)",
                  fn, key_chunk, kmax, d);
    kc = key_chunk;
  }
  // a chunk beyond the row is the resident row: LDS is sized for the row, not
  // the chunk (a larger allocation only costs workgroups per CU)
  if (kc > n64) kc = n64;
  tarmac::TopkArgs a{q, k, v, out, idx_out, B, N, d, topk, dtype, kc, inv_sqrt(d), stream};
  return hip_status(tarmac::run_topk(a), fn);
}

}  // namespace

extern "C" {

int tarmac_abi_version(void) { return 1; }

const char* tarmac_last_error(void) { return g_last_error.c_str(); }

namespace {

int dense_common(const void* q, const void* k, const void* v, void* out, float* stats, int B,
                 int N, int d, int dtype, int key_chunk, void* stream, const char* fn) {
  int rc = check_core(q, k, v, out, B, N, d, dtype, fn);
  if (rc) return rc;
  int kc = key_chunk;
  if (kc <= 0) {
    kc = (N + 63) / 64 * 64;
    while (kc > 64 && tarmac::dense_lds_bytes(dtype, d, kc) > dense_lds_budget(d)) kc -= 64;
    // a row in several chunks takes equal ones (N = 1024 as 512 + 512, not
    // 960 + 64): the same rounds, less LDS per workgroup
    const int nch = (N + kc - 1) / kc;
    if (nch > 1) kc = ((N + nch - 1) / nch + 63) / 64 * 64;
  } else if (kc % 16 != 0) {
    return fail(TARMAC_ERR_INVALID, "%s: key_chunk must be a multiple of 16 (got %d)", fn, kc);
  }
  if (tarmac::dense_lds_bytes(dtype, d, kc) > dense_lds_budget(d))
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: key_chunk %d exceeds the LDS budget at d=%d", fn, kc, d);
  tarmac::DenseArgs a{q, k, v, out, B, N, d, dtype, kc, inv_sqrt(d), stream, stats};
  a.chunk_given = key_chunk > 0;
  return hip_status(tarmac::run_dense(a), fn);
}

}  // namespace

int tarmac_dense_fwd(const void* q, const void* k, const void* v, void* out, int B, int N, int d,
                     int dtype, int key_chunk, void* stream) {
  return dense_common(q, k, v, out, nullptr, B, N, d, dtype, key_chunk, stream,
                      "tarmac_dense_fwd");
}

int tarmac_dense_fwd_stats(const float* q, const float* k, const float* v, float* out,
                           float* stats, int B, int N, int d, void* stream) {
  const char* fn = "tarmac_dense_fwd_stats";
  if (!stats || !aligned(stats, 8)) return fail(TARMAC_ERR_INVALID, "%s: stats null or misaligned", fn);
  return dense_common(q, k, v, out, stats, B, N, d, TARMAC_DTYPE_F32, 0, stream, fn);
}

int tarmac_topk_fused_fwd(const void* q, const void* k, const void* v, void* out, int32_t* idx_out,
                          int B, int N, int d, int topk, int dtype, void* stream) {
  return topk_common(q, k, v, out, idx_out, B, N, d, topk, dtype, 0, stream, "tarmac_topk_fused_fwd");
}

int tarmac_topk_stream_fwd(const void* q, const void* k, const void* v, void* out,
                           int32_t* idx_out, int B, int N, int d, int topk, int dtype,
                           int key_chunk, void* stream) {
  const char* fn = "tarmac_topk_stream_fwd";
  const int kmax = max_topk_chunk(dtype, d);
  if (key_chunk <= 0) key_chunk = kmax;
  if (key_chunk > kmax) key_chunk = kmax;
  return topk_common(q, k, v, out, idx_out, B, N, d, topk, dtype, key_chunk, stream, fn);
}

int tarmac_topk_variant_fwd(const void* q, const void* k, const void* v, void* out,
                            int32_t* idx_out, int B, int N, int d, int topk, int variant, int bisect,
                            int dtype, void* stream) {
  const char* fn = "tarmac_topk_variant_fwd";
  int rc = check_core(q, k, v, out, B, N, d, dtype, fn);
  if (rc) return rc;
  if (variant != TARMAC_VARIANT_MASKED && variant != TARMAC_VARIANT_SORT)
    return fail(TARMAC_ERR_INVALID, "%s: variant must be %d (masked) or %d (sort) (got %d)", fn,
                TARMAC_VARIANT_MASKED, TARMAC_VARIANT_SORT, variant);
  if (topk < 1 || topk > N - 1)
    return fail(TARMAC_ERR_INVALID, "%s: need 1 <= topk <= N-1 (got topk=%d, N=%d)", fn, topk, N);
  if (bisect < 0) return fail(TARMAC_ERR_INVALID, "%s: bisect must be >= 0 (got %d)", fn, bisect);
  if (variant == TARMAC_VARIANT_MASKED && idx_out)
    return fail(TARMAC_ERR_INVALID, "%s: the masked variant keeps a variable number of peers; "
                "idx_out must be NULL", fn);
  if (idx_out && !aligned(idx_out, 4)) return fail(TARMAC_ERR_INVALID, "%s: idx_out misaligned", fn);
  // key chunk of the register-list kernel, which serves fp32 k <= 8 (the
  // wide kernels ignore it): the whole row when it fits
  const int n64 = (N + 63) / 64 * 64, kmax = max_topk_chunk(dtype, d);
  tarmac::TopkArgs a{q, k, v, out, idx_out, B, N, d, topk, dtype, n64 < kmax ? n64 : kmax,
                     inv_sqrt(d), stream};
  a.select = variant == TARMAC_VARIANT_MASKED ? tarmac::kSelMasked : tarmac::kSelSort;
  a.bisect = bisect;
  if (static_cast<size_t>(N + tarmac::wide_cap(a)) * 4 > kLdsBudget)
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: N=%d too large for one score row in LDS", fn, N);
  return hip_status(tarmac::run_topk(a), fn);
}

int tarmac_fixedset_fwd(const void* q, const void* k, const void* v, const void* idx,
                        int idx_dtype, int kk, void* out, int B, int N, int d, int dtype,
                        void* stream) {
  const char* fn = "tarmac_fixedset_fwd";
  int rc = check_core(q, k, v, out, B, N, d, dtype, fn);
  if (rc) return rc;
  if (kk < 1) return fail(TARMAC_ERR_INVALID, "%s: need kk >= 1 (got %d)", fn, kk);
  if (!idx) return fail(TARMAC_ERR_INVALID, "%s: null idx", fn);
  if (idx_dtype != TARMAC_IDX_I32 && idx_dtype != TARMAC_IDX_I64)
    return fail(TARMAC_ERR_INVALID, "%s: unknown idx dtype %d", fn, idx_dtype);
  if (!aligned(idx, idx_dtype == TARMAC_IDX_I64 ? 8 : 4))
    return fail(TARMAC_ERR_INVALID, "%s: idx misaligned", fn);
  tarmac::FixedsetArgs a{q, k, v, idx, idx_dtype == TARMAC_IDX_I64, out, B, N, d, kk, dtype,
                         inv_sqrt(d), stream};
  return hip_status(tarmac::run_fixedset(a), fn);
}

int tarmac_morton_window(const float* pos, void* idx_out, int idx_dtype, int64_t* codes_out,
                         int B, int N, int k, int bits, void* stream) {
  const char* fn = "tarmac_morton_window";
  if (!pos) return fail(TARMAC_ERR_INVALID, "%s: null pos", fn);
  if (!aligned(pos, 8)) return fail(TARMAC_ERR_INVALID, "%s: pos must be 8-byte aligned", fn);
  if (B < 1 || N < 2) return fail(TARMAC_ERR_INVALID, "%s: need B >= 1 and N >= 2", fn);
  if (bits < 1 || bits > 16) return fail(TARMAC_ERR_INVALID, "%s: bits must be 1..16 (got %d)", fn, bits);
  if (idx_out) {
    if (k < 1 || k > N - 1)
      return fail(TARMAC_ERR_INVALID, "%s: need 1 <= k <= N-1 (got k=%d, N=%d)", fn, k, N);
    if (idx_dtype != TARMAC_IDX_I32 && idx_dtype != TARMAC_IDX_I64)
      return fail(TARMAC_ERR_INVALID, "%s: unknown idx dtype %d", fn, idx_dtype);
    if (!aligned(idx_out, idx_dtype == TARMAC_IDX_I64 ? 8 : 4))
      return fail(TARMAC_ERR_INVALID, "%s: idx_out misaligned", fn);
  }
  if (codes_out && !aligned(codes_out, 8)) return fail(TARMAC_ERR_INVALID, "%s: codes_out misaligned", fn);
  if (N > kZorderMaxN || tarmac::zorder_lds_bytes(N) > kZorderLds)
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: N=%d exceeds the per-row sort capacity (%d)", fn, N,
                kZorderMaxN);
  tarmac::MortonArgs a{pos, idx_out, idx_dtype == TARMAC_IDX_I64, codes_out, B, N, k, bits, stream};
  return hip_status(tarmac::run_morton_window(a), fn);
}

namespace {

int knn_common(const float* pos, void* idx_out, int idx_dtype, int B, int N, int k, int grid,
               void* stream, const char* fn) {
  if (!pos || !idx_out) return fail(TARMAC_ERR_INVALID, "%s: null pos or idx_out", fn);
  if (!aligned(pos, 8)) return fail(TARMAC_ERR_INVALID, "%s: pos must be 8-byte aligned", fn);
  if (B < 1 || N < 2) return fail(TARMAC_ERR_INVALID, "%s: need B >= 1 and N >= 2", fn);
  if (k < 1 || k > N - 1)
    return fail(TARMAC_ERR_INVALID, "%s: need 1 <= k <= N-1 (got k=%d, N=%d)", fn, k, N);
  if (idx_dtype != TARMAC_IDX_I32 && idx_dtype != TARMAC_IDX_I64)
    return fail(TARMAC_ERR_INVALID, "%s: unknown idx dtype %d", fn, idx_dtype);
  if (!aligned(idx_out, idx_dtype == TARMAC_IDX_I64 ? 8 : 4))
    return fail(TARMAC_ERR_INVALID, "%s: idx_out misaligned", fn);
  if (static_cast<long long>(B) * N * k >= (1ll << 40))
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: tensor too large", fn);
  tarmac::KnnArgs a{pos, idx_out, idx_dtype == TARMAC_IDX_I64, B, N, k, 0, 0, 0, stream};
  if (grid) {
    int G = 0, M = 0;
    tarmac::grid_knn_shape(N, k, &G, &M);
    // the reference's own route: all pairs when the 3x3 block would hold N or more
    if (9ll * M < N) {
      a.grid = 1;
      a.G = G;
      a.L = 3 * M;
      if (tarmac::knn_grid_lds_bytes(N, G, tarmac::knn_grid_threads(N)) > kLdsBudget)
        return fail(TARMAC_ERR_UNSUPPORTED, "%s: N=%d exceeds the per-row grid capacity", fn, N);
    }
  }
  if (!a.grid && tarmac::knn_radius_lds_bytes(N) > kLdsBudget)
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: N=%d exceeds the per-row position capacity", fn, N);
  return hip_status(tarmac::run_knn(a), fn);
}

}  // namespace

int tarmac_knn_radius(const float* pos, void* idx_out, int idx_dtype, int B, int N, int k,
                      void* stream) {
  return knn_common(pos, idx_out, idx_dtype, B, N, k, 0, stream, "tarmac_knn_radius");
}

int tarmac_knn_grid(const float* pos, void* idx_out, int idx_dtype, int B, int N, int k,
                    void* stream) {
  return knn_common(pos, idx_out, idx_dtype, B, N, k, 1, stream, "tarmac_knn_grid");
}

int tarmac_grid_knn_shape(int N, int k, int* G, int* M) {
  if (!G || !M) return fail(TARMAC_ERR_INVALID, "tarmac_grid_knn_shape: null output");
  if (N < 1 || k < 1) return fail(TARMAC_ERR_INVALID, "tarmac_grid_knn_shape: need N >= 1, k >= 1");
  tarmac::grid_knn_shape(N, k, G, M);
  return ok();
}

int tarmac_zorder_fwd(const void* q, const void* k, const void* v, const float* pos, void* out,
                      int32_t* idx_out, int B, int N, int d, int topk, int bits, int dtype,
                      void* stream) {
  const char* fn = "tarmac_zorder_fwd";
  int rc = check_core(q, k, v, out, B, N, d, dtype, fn);
  if (rc) return rc;
  if (!pos || !aligned(pos, 8)) return fail(TARMAC_ERR_INVALID, "%s: pos null or misaligned", fn);
  if (topk < 1 || topk > N - 1)
    return fail(TARMAC_ERR_INVALID, "%s: need 1 <= topk <= N-1 (got topk=%d, N=%d)", fn, topk, N);
  if (bits < 1 || bits > 16) return fail(TARMAC_ERR_INVALID, "%s: bits must be 1..16 (got %d)", fn, bits);
  if (idx_out && !aligned(idx_out, 4)) return fail(TARMAC_ERR_INVALID, "%s: idx_out misaligned", fn);
  if (N > kZorderMaxN || tarmac::zorder_lds_bytes(N) > kZorderLds)
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: N=%d exceeds the per-row sort capacity (%d)", fn, N,
                kZorderMaxN);
  tarmac::ZorderArgs a{q, k, v, pos, out, idx_out, B, N, d, topk, bits, dtype, inv_sqrt(d), stream};
  return hip_status(tarmac::run_zorder(a), fn);
}

int tarmac_fixedset_bwd(const float* q, const float* k, const float* v, const float* dout,
                        const void* idx, int idx_dtype, int kk, float* dq, float* dk, float* dv,
                        int B, int N, int d, void* stream) {
  const char* fn = "tarmac_fixedset_bwd";
  int rc = check_core(q, k, v, dout, B, N, d, TARMAC_DTYPE_F32, fn);
  if (rc) return rc;
  if (!idx || !dq || !dk || !dv) return fail(TARMAC_ERR_INVALID, "%s: null pointer", fn);
  if (!aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16))
    return fail(TARMAC_ERR_INVALID, "%s: gradient buffers must be 16-byte aligned", fn);
  if (idx_dtype != TARMAC_IDX_I32 && idx_dtype != TARMAC_IDX_I64)
    return fail(TARMAC_ERR_INVALID, "%s: idx_dtype must be TARMAC_IDX_I32 or TARMAC_IDX_I64", fn);
  if (kk < 1) return fail(TARMAC_ERR_INVALID, "%s: kk must be >= 1 (got %d)", fn, kk);
  tarmac::FixedsetBwdArgs a{q, k, v, dout, idx, idx_dtype == TARMAC_IDX_I64, dq, dk, dv,
                            B, N, d, kk, inv_sqrt(d), stream};
  return hip_status(tarmac::run_fixedset_bwd(a), fn);
}

int tarmac_dense_bwd(const float* q, const float* k, const float* v, const float* out,
                     const float* dout, float* dq, float* dk, float* dv, float* stats,
                     int stats_ready, int B, int N, int d, void* stream) {
  const char* fn = "tarmac_dense_bwd";
  int rc = check_core(q, k, v, out, B, N, d, TARMAC_DTYPE_F32, fn);
  if (rc) return rc;
  if (!dout || !dq || !dk || !dv || !stats) return fail(TARMAC_ERR_INVALID, "%s: null pointer", fn);
  if (!aligned(dout, 16) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16) ||
      !aligned(stats, 8))
    return fail(TARMAC_ERR_INVALID, "%s: misaligned buffer", fn);
  if (stats_ready != 0 && stats_ready != 1)
    return fail(TARMAC_ERR_INVALID, "%s: stats_ready must be 0 or 1", fn);
  tarmac::DenseBwdArgs a{q, k, v, out, dout, dq, dk, dv, stats, stats_ready, B, N, d,
                         inv_sqrt(d), stream};
  return hip_status(tarmac::run_dense_bwd(a), fn);
}

int tarmac_dense_bwd_noalloc(const float* q, const float* k, const float* v, const float* out,
                             const float* dout, float* dq, float* dk, float* dv, int B, int N,
                             int d, void* stream) {
  const char* fn = "tarmac_dense_bwd_noalloc";
  int rc = check_core(q, k, v, out, B, N, d, TARMAC_DTYPE_F32, fn);
  if (rc) return rc;
  if (!dout || !dq || !dk || !dv) return fail(TARMAC_ERR_INVALID, "%s: null pointer", fn);
  if (!aligned(dout, 16) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16))
    return fail(TARMAC_ERR_INVALID, "%s: misaligned buffer", fn);
  const size_t need = size_t(2) * size_t(B) * size_t(N) * sizeof(float);
  if (need > tarmac::kScratchBytes)
    return fail(TARMAC_ERR_UNSUPPORTED,
                "%s: the [B, 2, N] statistics need %zu bytes, more than the library's %zu-byte "
                "scratch (B * N <= %zu); use tarmac_dense_bwd with a caller workspace",
                fn, need, tarmac::kScratchBytes, tarmac::kScratchBytes / (2 * sizeof(float)));
  void* ws = nullptr;
  hipError_t e = tarmac::scratch_address(&ws);
  if (e != hipSuccess) return hip_status(e, fn);
  // every statistic is written by the first pass before the second reads it:
  // nothing in the scratch needs clearing
  tarmac::DenseBwdArgs a{q, k, v, out, dout, dq, dk, dv, static_cast<float*>(ws), 0, B, N, d,
                         inv_sqrt(d), stream};
  return hip_status(tarmac::run_dense_bwd(a), fn);
}

int tarmac_set_topk_filter(int mode) {
  if (mode < tarmac::kFilterOff || mode > tarmac::kFilterSplit32) {
    fail(TARMAC_ERR_INVALID, "tarmac_set_topk_filter: mode must be 0 to 5 (got %d)", mode);
    return -1;
  }
  return tarmac::set_topk_filter_mode(mode);
}

int tarmac_set_query_tiles(int mode) {
  if (mode < tarmac::kTilesAuto || mode > tarmac::kTilesTwo) {
    fail(TARMAC_ERR_INVALID, "tarmac_set_query_tiles: mode must be 0 to 2 (got %d)", mode);
    return -1;
  }
  return tarmac::set_query_tiles_mode(mode);
}

int tarmac_mfma_bf16_probe(const void* a, const void* b, float* out, int tiles, int chain,
                           int shape, void* stream) {
  const char* fn = "tarmac_mfma_bf16_probe";
  if (!a || !b || !out) return fail(TARMAC_ERR_INVALID, "%s: null pointer", fn);
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(out, 16))
    return fail(TARMAC_ERR_INVALID, "%s: operands must be 16-byte aligned", fn);
  if (tiles < 1 || chain < 1 || chain > 64)
    return fail(TARMAC_ERR_INVALID, "%s: need tiles >= 1 and 1 <= chain <= 64", fn);
  if (shape != 16 && shape != 32) return fail(TARMAC_ERR_INVALID, "%s: shape must be 16 or 32", fn);
  return hip_status(tarmac::run_mfma_bf16_probe(a, b, out, tiles, chain, shape, stream), fn);
}

// -- attention over heads -----------------------------------------------------

namespace {

int64_t elem_size(int dtype) { return dtype == TARMAC_DTYPE_F32 ? 4 : 2; }

// A tensor of heads: present, and every row's start on 16 bytes.
int check_heads(const tarmac_heads& t, int dtype, const char* name, const char* fn) {
  if (!t.data) return fail(TARMAC_ERR_INVALID, "%s: null %s", fn, name);
  const int64_t per = 16 / elem_size(dtype);
  if (!aligned(t.data, 16) || t.stride_b % per || t.stride_n % per || t.stride_h % per)
    return fail(TARMAC_ERR_INVALID, "%s: %s must be 16-byte aligned, in its strides too", fn, name);
  // tiles of up to 64 rows are addressed by 32-bit offsets
  if (t.stride_n < 0 || t.stride_n * elem_size(dtype) >= (int64_t(1) << 25))
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: stride_n of %s must be from 0 to below 32 MiB", fn, name);
  return TARMAC_OK;
}

int check_width(int d, int dtype, const char* fn) {
  if (dtype != TARMAC_DTYPE_F32 && dtype != TARMAC_DTYPE_BF16 && dtype != TARMAC_DTYPE_F16)
    return fail(TARMAC_ERR_INVALID, "%s: unknown dtype %d", fn, dtype);
  if (d < 8 || d > 128 || d % 8)
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: head width must be a multiple of 8 up to 128 (got %d)", fn, d);
  return TARMAC_OK;
}

tarmac::HeadsView view(const tarmac_heads& t) { return {t.data, t.stride_b, t.stride_n, t.stride_h}; }

tarmac::MhaArgs mha_args(const tarmac_mha* m, void* stream) {
  return {view(m->q), view(m->k), view(m->v), view(m->out), view(m->dout), view(m->dq), view(m->dk), view(m->dv),
          m->lse, m->workspace, m->workspace_bytes, m->lengths, m->q_lengths, m->q_start,
          m->B, m->Nq, m->Nk, m->Hq, m->Hkv, m->d, m->dtype, m->causal != 0, m->exclude_self != 0, m->scale, stream};
}

// Everything but the tensors: sizes, type, scale.
int mha_sizes(const tarmac_mha* m, const char* fn) {
  if (!m || m->size != static_cast<int64_t>(sizeof(tarmac_mha)))
    return fail(TARMAC_ERR_INVALID, "%s: null call, or not a tarmac_mha of this header", fn);
  if (m->B < 1 || m->Nq < 1 || m->Nk < 1 || m->Hq < 1 || m->Hkv < 1)
    return fail(TARMAC_ERR_INVALID, "%s: need B, Nq, Nk, Hq, Hkv >= 1 (got %d, %d, %d, %d, %d)", fn, m->B, m->Nq,
                m->Nk, m->Hq, m->Hkv);
  if (m->Hq % m->Hkv)
    return fail(TARMAC_ERR_INVALID, "%s: Hkv must divide Hq (got %d, %d)", fn, m->Hkv, m->Hq);
  const int rc = check_width(m->d, m->dtype, fn);
  if (rc) return rc;
  const int64_t longest = m->Nq > m->Nk ? m->Nq : m->Nk;
  // (a last tile's rows end up to 127 behind the last row, in 32 bits)
  if (static_cast<double>(m->B) * m->Hq * longest >= 2147483648.0 - 256 || longest > (int64_t(1) << 29))
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: B * Hq * max(Nq, Nk) must stay below 2^31 - 256, Nq and Nk up to 2^29", fn);
  if (!(m->scale > 0.f) || std::isinf(m->scale))
    return fail(TARMAC_ERR_INVALID, "%s: scale must be positive and finite", fn);
  if ((m->lengths && !aligned(m->lengths, 4)) || (m->q_lengths && !aligned(m->q_lengths, 4)) ||
      (m->q_start && !aligned(m->q_start, 4)))
    return fail(TARMAC_ERR_INVALID, "%s: lengths, q_lengths or q_start misaligned", fn);
  if (tarmac::mha_threads(mha_args(m, nullptr)) >> 32)
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: %d x %d key heads of %d queries and %d keys are more than one launch holds",
                fn, m->B, m->Hkv, m->Nq, m->Nk);
  return TARMAC_OK;
}

int check_workspace(void* ws, int64_t have, int64_t need, const char* fn) {
  if (need > 0 && (!ws || !aligned(ws, 16) || have < need))
    return fail(TARMAC_ERR_INVALID, "%s: needs a 16-byte aligned workspace of %lld bytes (got %lld)", fn,
                static_cast<long long>(need), static_cast<long long>(ws ? have : 0));
  return TARMAC_OK;
}

tarmac::RopeArgs rope_args(const tarmac_qk_rope* r, void* stream) {
  return {view(r->q), view(r->k), view(r->q_out), view(r->k_out), view(r->dq), view(r->dk), r->wq, r->wk, r->table,
          r->positions, r->dwq, r->dwk, r->workspace, r->workspace_bytes, r->table_rows, r->B, r->N, r->Hq, r->Hkv,
          r->d, r->table ? r->rot : 0, r->dtype, r->w_dtype == TARMAC_DTYPE_F32, r->pos_dtype == TARMAC_IDX_I64,
          r->eps, stream};
}

int rope_sizes(const tarmac_qk_rope* r, const char* fn) {
  if (!r || r->size != static_cast<int64_t>(sizeof(tarmac_qk_rope)))
    return fail(TARMAC_ERR_INVALID, "%s: null call, or not a tarmac_qk_rope of this header", fn);
  if (r->B < 1 || r->N < 1 || r->Hq < 1 || r->Hkv < 1)
    return fail(TARMAC_ERR_INVALID, "%s: need B, N, Hq, Hkv >= 1 (got %d, %d, %d, %d)", fn, r->B, r->N, r->Hq, r->Hkv);
  const int rc = check_width(r->d, r->dtype, fn);
  if (rc) return rc;
  if (static_cast<double>(r->B) * r->N * (static_cast<double>(r->Hq) + r->Hkv) >= 2147483648.0)
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: B * N * (Hq + Hkv) must stay below 2^31", fn);
  if (!r->table && !r->wq && !r->wk)
    return fail(TARMAC_ERR_INVALID, "%s: neither weights nor a table: nothing to do", fn);
  if (r->table && (r->rot < 8 || r->rot > r->d || r->rot % 8 || r->table_rows < 1 || !aligned(r->table, 16)))
    return fail(TARMAC_ERR_INVALID,
                "%s: the table needs rows of a multiple of 8 columns up to the head width, 16-byte aligned "
                "(got %lld rows of %d at width %d)",
                fn, static_cast<long long>(r->table_rows), r->rot, r->d);
  if ((r->wq && !aligned(r->wq, 16)) || (r->wk && !aligned(r->wk, 16)))
    return fail(TARMAC_ERR_INVALID, "%s: weights must be 16-byte aligned", fn);
  if (r->w_dtype != TARMAC_DTYPE_F32 && r->w_dtype != r->dtype)
    return fail(TARMAC_ERR_INVALID, "%s: weights must be fp32 or of the heads' type", fn);
  if (r->pos_dtype != TARMAC_IDX_I32 && r->pos_dtype != TARMAC_IDX_I64)
    return fail(TARMAC_ERR_INVALID, "%s: pos_dtype must be TARMAC_IDX_I32 or TARMAC_IDX_I64", fn);
  if (r->positions && !aligned(r->positions, r->pos_dtype == TARMAC_IDX_I64 ? 8 : 4))
    return fail(TARMAC_ERR_INVALID, "%s: positions misaligned", fn);
  if (!(r->eps >= 0.f) || std::isinf(r->eps))
    return fail(TARMAC_ERR_INVALID, "%s: eps must be finite and not negative", fn);
  if (tarmac::qk_rope_threads(rope_args(r, nullptr)) >> 32)
    return fail(TARMAC_ERR_UNSUPPORTED, "%s: %d x %d tokens of %d and %d heads are more than one launch holds", fn, r->B,
                r->N, r->Hq, r->Hkv);
  return TARMAC_OK;
}

}  // namespace

int64_t tarmac_mha_fwd_workspace(const tarmac_mha* m) {
  if (mha_sizes(m, "tarmac_mha_fwd_workspace")) return -1;
  return tarmac::mha_fwd_workspace(mha_args(m, nullptr));
}

int64_t tarmac_mha_bwd_workspace(const tarmac_mha* m) {
  if (mha_sizes(m, "tarmac_mha_bwd_workspace")) return -1;
  return tarmac::mha_bwd_workspace(mha_args(m, nullptr));
}

int tarmac_mha_fwd(const tarmac_mha* m, void* stream) {
  const char* fn = "tarmac_mha_fwd";
  int rc = mha_sizes(m, fn);
  if (rc) return rc;
  if ((rc = check_heads(m->q, m->dtype, "q", fn)) || (rc = check_heads(m->k, m->dtype, "k", fn)) ||
      (rc = check_heads(m->v, m->dtype, "v", fn)) || (rc = check_heads(m->out, m->dtype, "out", fn)))
    return rc;
  if (!m->lse || !aligned(m->lse, 4)) return fail(TARMAC_ERR_INVALID, "%s: lse null or misaligned", fn);
  const tarmac::MhaArgs a = mha_args(m, stream);
  if ((rc = check_workspace(m->workspace, m->workspace_bytes, tarmac::mha_fwd_workspace(a), fn))) return rc;
  return hip_status(m->dtype == TARMAC_DTYPE_F32    ? tarmac::run_mha_fwd_f32(a)
                    : m->dtype == TARMAC_DTYPE_BF16 ? tarmac::run_mha_fwd_bf16(a)
                                                    : tarmac::run_mha_fwd_f16(a),
                    fn);
}

int tarmac_mha_bwd(const tarmac_mha* m, void* stream) {
  const char* fn = "tarmac_mha_bwd";
  int rc = mha_sizes(m, fn);
  if (rc) return rc;
  const struct { const tarmac_heads& t; const char* name; } all[] = {
      {m->q, "q"}, {m->k, "k"}, {m->v, "v"}, {m->out, "out"}, {m->dout, "dout"}, {m->dq, "dq"}, {m->dk, "dk"}, {m->dv, "dv"}};
  for (const auto& x : all)
    if ((rc = check_heads(x.t, m->dtype, x.name, fn))) return rc;
  if (!m->lse || !aligned(m->lse, 4)) return fail(TARMAC_ERR_INVALID, "%s: lse null or misaligned", fn);
  const tarmac::MhaArgs a = mha_args(m, stream);
  if ((rc = check_workspace(m->workspace, m->workspace_bytes, tarmac::mha_bwd_workspace(a), fn))) return rc;
  return hip_status(m->dtype == TARMAC_DTYPE_F32    ? tarmac::run_mha_bwd_f32(a)
                    : m->dtype == TARMAC_DTYPE_BF16 ? tarmac::run_mha_bwd_bf16(a)
                                                    : tarmac::run_mha_bwd_f16(a),
                    fn);
}

int64_t tarmac_qk_rope_bwd_workspace(const tarmac_qk_rope* r) {
  if (rope_sizes(r, "tarmac_qk_rope_bwd_workspace")) return -1;
  return tarmac::qk_rope_bwd_workspace(rope_args(r, nullptr));
}

int tarmac_qk_rope_fwd(const tarmac_qk_rope* r, void* stream) {
  const char* fn = "tarmac_qk_rope_fwd";
  int rc = rope_sizes(r, fn);
  if (rc) return rc;
  if ((rc = check_heads(r->q, r->dtype, "q", fn)) || (rc = check_heads(r->k, r->dtype, "k", fn)) ||
      (rc = check_heads(r->q_out, r->dtype, "q_out", fn)) || (rc = check_heads(r->k_out, r->dtype, "k_out", fn)))
    return rc;
  return hip_status(tarmac::run_qk_rope(rope_args(r, stream), false), fn);
}

int tarmac_qk_rope_bwd(const tarmac_qk_rope* r, void* stream) {
  const char* fn = "tarmac_qk_rope_bwd";
  int rc = rope_sizes(r, fn);
  if (rc) return rc;
  if ((rc = check_heads(r->q, r->dtype, "q", fn)) || (rc = check_heads(r->k, r->dtype, "k", fn)) ||
      (rc = check_heads(r->q_out, r->dtype, "q_out", fn)) || (rc = check_heads(r->k_out, r->dtype, "k_out", fn)) ||
      (rc = check_heads(r->dq, r->dtype, "dq", fn)) || (rc = check_heads(r->dk, r->dtype, "dk", fn)))
    return rc;
  if ((r->wq != nullptr) != (r->dwq != nullptr) || (r->wk != nullptr) != (r->dwk != nullptr))
    return fail(TARMAC_ERR_INVALID, "%s: a weight and its gradient come together", fn);
  if ((rc = check_workspace(r->workspace, r->workspace_bytes, tarmac::qk_rope_bwd_workspace(rope_args(r, nullptr)), fn)))
    return rc;
  return hip_status(tarmac::run_qk_rope(rope_args(r, stream), true), fn);
}

int tarmac_noop(float* out, void* stream) {
  if (!out) return fail(TARMAC_ERR_INVALID, "tarmac_noop: null out");
  return hip_status(tarmac::run_noop(out, stream), "tarmac_noop");
}

}  // extern "C"
