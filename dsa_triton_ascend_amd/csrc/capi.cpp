// C ABI of libdsa_mi355x.so: argument validation, error reporting, dispatch.
//
// Validation mirrors the ValueError conditions of the reference operators
// (lightning_indexer_triton.py:501-502, :524-525; sparse_flash_attention_triton.py
// :1341-1351, :1377-1378, :1391-1398) so a bad call fails here with a message
// instead of reaching a kernel; the Python layer raises the same conditions first.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "../../include/dsa_mi355x.h"
#include "dsa_common.hpp"

bool li_score_supported_d(int d);

namespace {
thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int hip_status(hipError_t e, const char* what) {
  if (e == hipSuccess) {
    g_err[0] = 0;
    return DSA_OK;
  }
  return fail(DSA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool is16(int dt) { return dt == DSA_DTYPE_BF16 || dt == DSA_DTYPE_F16; }

// A call's length and offset arrays travel as kernel arguments. A copy from pageable memory made the
// host wait for the stream (four of them a call: about 20 us in which the GPU idled between calls).
constexpr int UPLOAD_MAX = 8192;   // ints per call
template <int N> struct UploadArgs { int32_t v[N]; };

template <int N>
__global__ __launch_bounds__(256) void upload_i32_kernel(UploadArgs<N> a, int n, int32_t* dst, uint4* zero, int n16) {
  for (int i = threadIdx.x; i < n; i += 256) dst[i] = a.v[i];
  for (int i = threadIdx.x; i < n16; i += 256) zero[i] = make_uint4(0, 0, 0, 0);
}

template <int N>
void launch_upload(const int32_t* host, int n, int32_t* dst, void* zero, int n16, hipStream_t s) {
  UploadArgs<N> a;
  std::memcpy(a.v, host, sizeof(int32_t) * (size_t)n);
  hipLaunchKernelGGL(upload_i32_kernel<N>, dim3(1), dim3(256), 0, s, a, n, dst, reinterpret_cast<uint4*>(zero), n16);
}
}  // namespace

extern "C" {

int dsa_abi_version(void) { return 1; }

const char* dsa_last_error(void) { return g_err; }

int dsa_upload_i32(const int32_t* host, int n, int32_t* dst, void* zero_dst, size_t zero_bytes, void* stream) {
  if (n < 0 || (n > 0 && (!host || !dst)))
    return fail(DSA_ERR_INVALID, "dsa_upload_i32: null pointer argument or negative count");
  if (n > UPLOAD_MAX) return fail(DSA_ERR_UNSUPPORTED, "dsa_upload_i32: n=%d > %d", n, UPLOAD_MAX);
  if (!zero_dst) zero_bytes = 0;
  if (zero_bytes % 16 != 0 || zero_bytes > (1 << 20) || ((uintptr_t)zero_dst & 15) != 0)
    return fail(DSA_ERR_INVALID, "dsa_upload_i32: zero_dst / zero_bytes must be multiples of 16, at most 1 MiB");
  const hipStream_t s = (hipStream_t)stream;
  const int n16 = (int)(zero_bytes / 16);
  if (n == 0 && n16 == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  // kernel arguments are limited to 4 KiB; most calls fit the small form
  constexpr int SMALL = 56, LARGE = 960;
  if (n <= SMALL) {
    launch_upload<SMALL>(host, n, dst, zero_dst, n16, s);
  } else {
    for (int i = 0; i < n; i += LARGE)
      launch_upload<LARGE>(host + i, n - i < LARGE ? n - i : LARGE, dst + i, zero_dst, i == 0 ? n16 : 0, s);
  }
  return hip_status(hipGetLastError(), "dsa_upload_i32 launch");
}

int dsa_li_score(const void* query, const void* key, const void* weights, int io_dtype,
                 int w_dtype, const int32_t* row_start, const int32_t* key_start,
                 const int32_t* act_q, const int32_t* act_k, int batch, int total_rows, int n1,
                 int n2, int d, int s2, int max_rows_per_batch, int max_kv, int sparse_mode,
                 uint16_t* scores, int64_t score_ld, void* stream) {
  if (!query || !key || !weights || !row_start || !key_start || !act_q || !act_k || !scores)
    return fail(DSA_ERR_INVALID, "dsa_li_score: null pointer argument");
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "dsa_li_score: io_dtype must be fp16 or bf16");
  if (!is16(w_dtype) && w_dtype != DSA_DTYPE_F32)
    return fail(DSA_ERR_INVALID, "dsa_li_score: weights dtype must be fp16, bf16 or fp32");
  if (batch <= 0 || total_rows < 0 || n1 <= 0 || n2 <= 0 || s2 < 0 || max_rows_per_batch < 0)
    return fail(DSA_ERR_INVALID, "dsa_li_score: non-positive shape");
  if (n1 % n2 != 0) return fail(DSA_ERR_INVALID, "N1(%d) must be divisible by N2(%d)", n1, n2);
  if (n1 / n2 > 128) return fail(DSA_ERR_UNSUPPORTED, "dsa_li_score: group size N1/N2=%d > 128", n1 / n2);
  if (!li_score_supported_d(d))
    return fail(DSA_ERR_UNSUPPORTED, "dsa_li_score: D=%d not in {64, 96, 128, 256, 512}", d);
  if (sparse_mode != 0 && sparse_mode != 3)
    return fail(DSA_ERR_INVALID, "dsa_li_score: sparse_mode must be 0 or 3");
  if (score_ld < s2) return fail(DSA_ERR_INVALID, "dsa_li_score: score_ld < S2");
  if (batch > 65535 || n2 > 65535) return fail(DSA_ERR_UNSUPPORTED, "dsa_li_score: batch or N2 > 65535");
  LiScoreArgs a{query, key, weights, io_dtype, w_dtype, row_start, key_start, act_q, act_k,
                batch, total_rows, n1, n2, d, s2, max_rows_per_batch, max_kv, sparse_mode,
                scores, score_ld};
  return hip_status(launch_li_score(a, (hipStream_t)stream), "dsa_li_score launch");
}

int dsa_li_score_paged(const void* query, const void* key_cache, const void* weights, int io_dtype,
                       int w_dtype, const int32_t* row_start, const int32_t* block_table,
                       int max_blocks, int page_block_size, int64_t key_rows, const int32_t* act_q,
                       const int32_t* act_k, int batch, int total_rows, int n1, int n2, int d,
                       int max_rows_per_batch, int max_kv, int sparse_mode, uint16_t* scores,
                       int64_t score_ld, void* stream) {
  if (!query || !key_cache || !weights || !row_start || !block_table || !act_q || !act_k || !scores)
    return fail(DSA_ERR_INVALID, "dsa_li_score_paged: null pointer argument");
  if (max_blocks <= 0 || page_block_size <= 0 || key_rows <= 0)
    return fail(DSA_ERR_INVALID, "dsa_li_score_paged: max_blocks, page_block_size and key_rows must be positive");
  if (max_blocks > LI_MAX_BLOCKS)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_li_score_paged: max_blocks=%d > %d", max_blocks, LI_MAX_BLOCKS);
  const int64_t s2 = (int64_t)max_blocks * page_block_size;
  if (s2 > INT_MAX) return fail(DSA_ERR_UNSUPPORTED, "dsa_li_score_paged: max_blocks*block_size > 2^31-1");
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "dsa_li_score_paged: io_dtype must be fp16 or bf16");
  if (!is16(w_dtype) && w_dtype != DSA_DTYPE_F32)
    return fail(DSA_ERR_INVALID, "dsa_li_score_paged: weights dtype must be fp16, bf16 or fp32");
  if (batch <= 0 || total_rows < 0 || n1 <= 0 || n2 <= 0 || max_rows_per_batch < 0)
    return fail(DSA_ERR_INVALID, "dsa_li_score_paged: non-positive shape");
  if (n1 % n2 != 0) return fail(DSA_ERR_INVALID, "N1(%d) must be divisible by N2(%d)", n1, n2);
  if (n1 / n2 > 128) return fail(DSA_ERR_UNSUPPORTED, "dsa_li_score_paged: group size N1/N2=%d > 128", n1 / n2);
  if (!li_score_supported_d(d))
    return fail(DSA_ERR_UNSUPPORTED, "dsa_li_score_paged: D=%d not in {64, 96, 128, 256, 512}", d);
  if (sparse_mode != 0 && sparse_mode != 3)
    return fail(DSA_ERR_INVALID, "dsa_li_score_paged: sparse_mode must be 0 or 3");
  if (score_ld < s2) return fail(DSA_ERR_INVALID, "dsa_li_score_paged: score_ld < max_blocks*block_size");
  if (batch > 65535 || n2 > 65535) return fail(DSA_ERR_UNSUPPORTED, "dsa_li_score_paged: batch or N2 > 65535");
  LiScoreArgs a{query, key_cache, weights, io_dtype, w_dtype, row_start, act_q, act_q, act_k,
                batch, total_rows, n1, n2, d, (int)s2, max_rows_per_batch, max_kv, sparse_mode,
                scores, score_ld};
  a.block_table = block_table;
  a.max_blocks = max_blocks;
  a.page_bs = page_block_size;
  a.key_rows = key_rows;
  return hip_status(launch_li_score(a, (hipStream_t)stream), "dsa_li_score_paged launch");
}

namespace {
// Argument checks of dsa_li_topk / dsa_li_topk_ws; DSA_OK when the call may proceed.
int check_li_topk(const char* fn, const uint16_t* scores, int64_t score_ld, int io_dtype,
                  const int32_t* row_start, const int32_t* act_q, const int32_t* act_k, int batch,
                  int total_rows, int n2, int s2, int sparse_mode, int sparse_count, const int32_t* indices) {
  if (!scores || !row_start || !act_q || !act_k || !indices)
    return fail(DSA_ERR_INVALID, "%s: null pointer argument", fn);
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "%s: io_dtype must be fp16 or bf16", fn);
  if (batch <= 0 || total_rows < 0 || n2 <= 0 || s2 < 0)
    return fail(DSA_ERR_INVALID, "%s: non-positive shape", fn);
  if (sparse_count <= 0) return fail(DSA_ERR_INVALID, "%s: sparse_count must be positive", fn);
  if (sparse_mode != 0 && sparse_mode != 3)
    return fail(DSA_ERR_INVALID, "%s: sparse_mode must be 0 or 3", fn);
  if (score_ld < s2) return fail(DSA_ERR_INVALID, "%s: score_ld < S2", fn);
  return DSA_OK;
}
}  // namespace

int dsa_li_topk(const uint16_t* scores, int64_t score_ld, int io_dtype, const int32_t* row_start,
                const int32_t* act_q, const int32_t* act_k, int batch, int total_rows, int n2,
                int s2, int sparse_mode, int sparse_count, int32_t* indices, uint16_t* values,
                void* stream) {
  const int st = check_li_topk("dsa_li_topk", scores, score_ld, io_dtype, row_start, act_q, act_k, batch,
                               total_rows, n2, s2, sparse_mode, sparse_count, indices);
  if (st != DSA_OK) return st;
  if (sparse_count > LI_TOPK_MAX_K)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_li_topk: sparse_count=%d > %d (use dsa_li_topk_ws)", sparse_count,
                LI_TOPK_MAX_K);
  LiTopkArgs a{scores, score_ld, io_dtype, row_start, act_q, act_k, batch, total_rows, n2, s2,
               sparse_mode, sparse_count, indices, values};
  return hip_status(launch_li_topk(a, (hipStream_t)stream), "dsa_li_topk launch");
}

int dsa_li_topk_kv(const uint16_t* scores, int64_t score_ld, int io_dtype, const int32_t* row_start,
                   const int32_t* act_q, const int32_t* act_k, int batch, int total_rows, int n2,
                   int s2, int max_kv, int sparse_mode, int sparse_count, int32_t* indices,
                   uint16_t* values, void* stream) {
  const int st = check_li_topk("dsa_li_topk_kv", scores, score_ld, io_dtype, row_start, act_q, act_k, batch,
                               total_rows, n2, s2, sparse_mode, sparse_count, indices);
  if (st != DSA_OK) return st;
  if (max_kv < 0) return fail(DSA_ERR_INVALID, "dsa_li_topk_kv: negative max_kv");
  if (sparse_count > LI_TOPK_MAX_K)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_li_topk_kv: sparse_count=%d > %d (use dsa_li_topk_ws)", sparse_count,
                LI_TOPK_MAX_K);
  LiTopkArgs a{scores, score_ld, io_dtype, row_start, act_q, act_k, batch, total_rows, n2, s2,
               sparse_mode, sparse_count, indices, values, max_kv};
  return hip_status(launch_li_topk(a, (hipStream_t)stream), "dsa_li_topk_kv launch");
}

size_t dsa_li_topk_workspace_bytes(int total_rows, int n2, int s2, int sparse_count) {
  return li_topk_workspace_bytes(total_rows, n2, s2, sparse_count);
}

int dsa_li_topk_ws(const uint16_t* scores, int64_t score_ld, int io_dtype, const int32_t* row_start,
                   const int32_t* act_q, const int32_t* act_k, int batch, int total_rows, int n2,
                   int s2, int sparse_mode, int sparse_count, int32_t* indices, uint16_t* values,
                   void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_li_topk("dsa_li_topk_ws", scores, score_ld, io_dtype, row_start, act_q, act_k, batch,
                               total_rows, n2, s2, sparse_mode, sparse_count, indices);
  if (st != DSA_OK) return st;
  LiTopkArgs a{scores, score_ld, io_dtype, row_start, act_q, act_k, batch, total_rows, n2, s2,
               sparse_mode, sparse_count, indices, values};
  if (sparse_count <= LI_TOPK_MAX_K)
    return hip_status(launch_li_topk(a, (hipStream_t)stream), "dsa_li_topk_ws launch");
  const size_t need = li_topk_workspace_bytes(total_rows, n2, s2, sparse_count);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(DSA_ERR_INVALID, "dsa_li_topk_ws: workspace of %zu bytes < %zu", workspace_bytes, need);
  return hip_status(launch_li_topk_big(a, workspace, (hipStream_t)stream), "dsa_li_topk_ws launch");
}

size_t dsa_sfa_workspace_bytes(int total_rows, int n1, int d, int sparse_count,
                               int sparse_block_size, int kv_splits) {
  if (total_rows <= 0 || sparse_count <= 0 || sparse_block_size <= 0) return 0;
  return sfa_workspace_bytes(total_rows, n1, d, sparse_count, sparse_block_size, kv_splits);
}

size_t dsa_sfa_workspace_zero_bytes(void) { return sfa_workspace_zero_bytes(); }

namespace {
// Argument checks of dsa_sfa_fwd (the reference's conditions, sparse_flash_attention_triton.py
// :1341-1351, :1391-1398) shared with dsa_sfa_fwd_noalloc; DSA_OK when the call may proceed.
int check_sfa_fwd(const char* fn, const void* query, const void* query_rope, const void* key,
                  const void* key_rope, int io_dtype, const int32_t* sparse_indices, int sparse_count,
                  int sparse_block_size, const int32_t* block_table, int max_blocks, int page_block_size,
                  const int32_t* row_start, const int32_t* key_start, const int32_t* act_q,
                  const int32_t* act_k, int batch, int total_rows, int n1, int d, int dr, int64_t key_rows,
                  int sparse_mode, void* out, float* sm_max, float* sm_sum, int kv_splits) {
  if (!query || !query_rope || !key || !key_rope || !sparse_indices || !row_start || !act_q ||
      !act_k || !out)
    return fail(DSA_ERR_INVALID, "%s: null pointer argument", fn);
  if (!block_table && !key_start)
    return fail(DSA_ERR_INVALID, "%s: key_start required without block_table", fn);
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "%s: io_dtype must be fp16 or bf16", fn);
  if (sparse_mode != 0 && sparse_mode != 3)
    return fail(DSA_ERR_INVALID, "Only sparse_mode 0 (full) / 3 (rightDownCausal) supported");
  if (sparse_block_size < 1 || (sparse_block_size & (sparse_block_size - 1)) != 0 ||
      sparse_block_size > 128)
    return fail(DSA_ERR_INVALID, "sparse_block_size must be a power of 2 in [1,128]");
  if (d != 128 && d != 256 && d != 512)
    return fail(DSA_ERR_INVALID, "D must be one of (128, 256, 512), got %d", d);
  if (dr != 64) return fail(DSA_ERR_INVALID, "rope dim must be 64, got %d", dr);
  if (n1 < 1 || n1 > 128 || (n1 & (n1 - 1)) != 0)
    return fail(DSA_ERR_INVALID, "N1 must be one of (1, 2, 4, 8, 16, 32, 64, 128), got %d", n1);
  if (batch <= 0 || total_rows < 0 || sparse_count <= 0 || key_rows < 0)
    return fail(DSA_ERR_INVALID, "%s: non-positive shape", fn);
  if (block_table && (max_blocks <= 0 || page_block_size <= 0))
    return fail(DSA_ERR_INVALID, "%s: PA_BSND needs max_blocks and block_size > 0", fn);
  if ((sm_max == nullptr) != (sm_sum == nullptr))
    return fail(DSA_ERR_INVALID, "%s: sm_max and sm_sum must both be given or both NULL", fn);
  if ((int64_t)sparse_count * sparse_block_size > (1 << 20))
    return fail(DSA_ERR_UNSUPPORTED, "%s: sparse_count*sparse_block_size > 2^20 tokens", fn);
  if (kv_splits > 16) return fail(DSA_ERR_UNSUPPORTED, "%s: kv_splits=%d > 16", fn, kv_splits);
  return DSA_OK;
}
}  // namespace

int dsa_sfa_fwd_noalloc(const void* query, const void* query_rope, const void* key, const void* key_rope,
                        int io_dtype, const int32_t* sparse_indices, int sparse_count, int sparse_block_size,
                        const int32_t* block_table, int max_blocks, int page_block_size,
                        const int32_t* row_start, const int32_t* key_start, const int32_t* act_q,
                        const int32_t* act_k, int batch, int total_rows, int n1, int d, int dr, int s2,
                        int64_t key_rows, int sparse_mode, float scale, void* out, float* sm_max,
                        float* sm_sum, int kv_splits, void* stream) {
  const int st = check_sfa_fwd("dsa_sfa_fwd_noalloc", query, query_rope, key, key_rope, io_dtype,
                               sparse_indices, sparse_count, sparse_block_size, block_table, max_blocks,
                               page_block_size, row_start, key_start, act_q, act_k, batch, total_rows, n1,
                               d, dr, key_rows, sparse_mode, out, sm_max, sm_sum, kv_splits);
  if (st != DSA_OK) return st;
  if (total_rows == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  const size_t need = sfa_workspace_bytes(total_rows, n1, d, sparse_count, sparse_block_size, kv_splits);
  if (need > DSA_SFA_NOALLOC_SCRATCH_BYTES)
    return fail(DSA_ERR_UNSUPPORTED,
                "dsa_sfa_fwd_noalloc: the problem needs %zu bytes of workspace, the static scratch holds %zu "
                "(use dsa_sfa_fwd with a caller workspace)", need, (size_t)DSA_SFA_NOALLOC_SCRATCH_BYTES);
  void* ws = nullptr;
  const hipError_t e = sfa_noalloc_workspace((hipStream_t)stream, &ws);
  if (e != hipSuccess) return hip_status(e, "dsa_sfa_fwd_noalloc scratch set-up");
  SfaArgs a{query, query_rope, key, key_rope, io_dtype, sparse_indices, sparse_count,
            sparse_block_size, block_table, max_blocks, page_block_size, row_start, key_start,
            act_q, act_k, batch, total_rows, n1, d, dr, s2, key_rows, sparse_mode, scale, out, sm_max,
            sm_sum, ws, (size_t)DSA_SFA_NOALLOC_SCRATCH_BYTES, kv_splits};
  return hip_status(launch_sfa_fwd(a, (hipStream_t)stream), "dsa_sfa_fwd_noalloc launch");
}

int dsa_sfa_fwd(const void* query, const void* query_rope, const void* key, const void* key_rope,
                int io_dtype, const int32_t* sparse_indices, int sparse_count,
                int sparse_block_size, const int32_t* block_table, int max_blocks,
                int page_block_size, const int32_t* row_start, const int32_t* key_start,
                const int32_t* act_q, const int32_t* act_k, int batch, int total_rows, int n1,
                int d, int dr, int s2, int64_t key_rows, int sparse_mode, float scale, void* out,
                float* sm_max,
                float* sm_sum, void* workspace, size_t workspace_bytes, int kv_splits,
                void* stream) {
  const int st = check_sfa_fwd("dsa_sfa_fwd", query, query_rope, key, key_rope, io_dtype, sparse_indices,
                               sparse_count, sparse_block_size, block_table, max_blocks, page_block_size,
                               row_start, key_start, act_q, act_k, batch, total_rows, n1, d, dr, key_rows,
                               sparse_mode, out, sm_max, sm_sum, kv_splits);
  if (st != DSA_OK) return st;
  const size_t need = sfa_workspace_bytes(total_rows, n1, d, sparse_count, sparse_block_size, kv_splits);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(DSA_ERR_INVALID, "dsa_sfa_fwd: workspace of %zu bytes required, %zu given", need,
                workspace_bytes);
  SfaArgs a{query, query_rope, key, key_rope, io_dtype, sparse_indices, sparse_count,
            sparse_block_size, block_table, max_blocks, page_block_size, row_start, key_start,
            act_q, act_k, batch, total_rows, n1, d, dr, s2, key_rows, sparse_mode, scale, out, sm_max,
            sm_sum, workspace, workspace_bytes, kv_splits};
  return hip_status(launch_sfa_fwd(a, (hipStream_t)stream), "dsa_sfa_fwd launch");
}

size_t dsa_sfa_bwd_workspace_bytes(int batch, const int32_t* host_row_start,
                                   const int32_t* host_act_k, int s2, int total_rows, int n1, int d,
                                   int sparse_count, int sparse_block_size, int64_t key_rows) {
  if (batch <= 0 || !host_row_start || !host_act_k || total_rows < 0 || n1 <= 0 || sparse_count <= 0 ||
      sparse_block_size <= 0 || key_rows < 0 || (d != 128 && d != 256 && d != 512))
    return 0;
  return sfa_bwd_workspace_bytes(batch, host_row_start, host_act_k, s2, total_rows, n1, d, sparse_count,
                                 sparse_block_size, key_rows);
}

int dsa_sfa_bwd(const void* query, const void* query_rope, const void* key, const void* key_rope,
                int io_dtype, const int32_t* sparse_indices, int sparse_count,
                int sparse_block_size, const int32_t* row_start, const int32_t* key_start,
                const int32_t* act_q, const int32_t* act_k, const int32_t* host_row_start,
                const int32_t* host_act_k, int batch, int total_rows, int n1, int d, int dr, int s2,
                int64_t key_rows, int sparse_mode, float scale, const void* d_out, const void* out,
                const float* sm_max, const float* sm_sum, void* d_query, void* d_query_rope,
                void* d_key, void* d_key_rope, void* d_value, void* workspace,
                size_t workspace_bytes, void* stream) {
  if (!query || !query_rope || !key || !key_rope || !sparse_indices || !row_start || !key_start ||
      !act_q || !act_k || !d_out || !out || !sm_max || !sm_sum || !d_query || !d_query_rope ||
      !d_key || !d_key_rope || !d_value || !workspace || !host_row_start || !host_act_k)
    return fail(DSA_ERR_INVALID, "dsa_sfa_bwd: null pointer argument");
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "dsa_sfa_bwd: io_dtype must be fp16 or bf16");
  if (sparse_mode != 0 && sparse_mode != 3)
    return fail(DSA_ERR_INVALID, "Only sparse_mode 0 (full) / 3 (rightDownCausal) supported");
  if (sparse_block_size < 1 || (sparse_block_size & (sparse_block_size - 1)) != 0 ||
      sparse_block_size > 128)
    return fail(DSA_ERR_INVALID, "sparse_block_size must be a power of 2 in [1,128]");
  if (d != 128 && d != 256 && d != 512)
    return fail(DSA_ERR_INVALID, "D must be one of (128, 256, 512), got %d", d);
  if (dr != 64) return fail(DSA_ERR_INVALID, "rope dim must be 64, got %d", dr);
  if (n1 < 1 || n1 > 128 || (n1 & (n1 - 1)) != 0)
    return fail(DSA_ERR_INVALID, "N1 must be one of (1, 2, 4, 8, 16, 32, 64, 128), got %d", n1);
  if (batch <= 0 || total_rows < 0 || sparse_count <= 0 || key_rows < 0)
    return fail(DSA_ERR_INVALID, "dsa_sfa_bwd: non-positive shape");
  if ((int64_t)sparse_count * sparse_block_size > (1 << 20))
    return fail(DSA_ERR_UNSUPPORTED, "dsa_sfa_bwd: sparse_count*sparse_block_size > 2^20 tokens");
  if (key_rows > INT32_MAX) return fail(DSA_ERR_UNSUPPORTED, "dsa_sfa_bwd: key_rows > 2^31-1");
  if (batch > 65535) return fail(DSA_ERR_UNSUPPORTED, "dsa_sfa_bwd: batch > 65535");
  if (host_row_start[0] != 0 || host_row_start[batch] > total_rows)
    return fail(DSA_ERR_INVALID, "dsa_sfa_bwd: host_row_start must start at 0 and end within total_rows");
  for (int b = 0; b < batch; ++b)   // the host copies size and place the library GEMMs
    if (host_row_start[b + 1] < host_row_start[b])
      return fail(DSA_ERR_INVALID, "dsa_sfa_bwd: host_row_start must be non-decreasing");
  const size_t need = sfa_bwd_workspace_bytes(batch, host_row_start, host_act_k, s2, total_rows, n1, d,
                                              sparse_count, sparse_block_size, key_rows);
  if (workspace_bytes < need)
    return fail(DSA_ERR_INVALID, "dsa_sfa_bwd: workspace of %zu bytes required, %zu given", need,
                workspace_bytes);
  SfaBwdArgs a{};
  a.f = SfaArgs{query, query_rope, key, key_rope, io_dtype, sparse_indices, sparse_count,
                sparse_block_size, nullptr, 0, 0, row_start, key_start, act_q, act_k, batch,
                total_rows, n1, d, dr, s2, key_rows, sparse_mode, scale, nullptr, nullptr, nullptr,
                workspace, workspace_bytes, 1};
  a.d_out = d_out;
  a.out = out;
  a.sm_max = sm_max;
  a.sm_sum = sm_sum;
  a.dq = d_query;
  a.dqr = d_query_rope;
  a.dk = d_key;
  a.dkr = d_key_rope;
  a.dv = d_value;
  a.h_row_start = host_row_start;
  a.h_act_k = host_act_k;
  const hipError_t e = launch_sfa_bwd(a, (hipStream_t)stream);
  if (e == hipErrorSharedObjectInitFailed)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_sfa_bwd: %s", sfa_bwd_library_error());
  if (e == hipErrorStreamCaptureUnsupported)
    return fail(DSA_ERR_UNSUPPORTED,
                "dsa_sfa_bwd: the first call on a device creates its hipBLASLt handle and must run "
                "outside stream capture");
  return hip_status(e, "dsa_sfa_bwd launch");
}

size_t dsa_sli_grad_workspace_bytes(int batch, int s1, int s2, int sparse_count, int d_idx) {
  if (batch <= 0 || s1 < 0 || s2 <= 0 || sparse_count <= 0 || d_idx <= 0) return 0;
  return sli_grad_workspace_bytes(batch * s1, sparse_count, (int64_t)batch * s2, d_idx,
                                  sli_km_sparse_ld(batch * s1, sparse_count, s2, d_idx));
}

int dsa_sli_grad_kl_loss(const void* query, const void* key, const void* query_rope, const void* key_rope,
                         const void* query_index, const void* key_index, const void* weights, int io_dtype,
                         int w_dtype, const int32_t* sparse_indices, int sparse_count, const float* sm_max,
                         const float* sm_sum, const int32_t* act_q, const int32_t* act_k, int batch, int s1,
                         int s2, int n1, int d, int dr, int nidx1, int d_idx, float scale,
                         void* d_query_index, void* d_key_index, void* d_weights, float* loss,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (!query || !key || !query_index || !key_index || !weights || !sparse_indices || !sm_max || !sm_sum ||
      !act_q || !act_k || !d_query_index || !d_key_index || !d_weights || !loss || !workspace ||
      (dr > 0 && (!query_rope || !key_rope)))
    return fail(DSA_ERR_INVALID, "dsa_sli_grad_kl_loss: null pointer argument");
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "dsa_sli_grad_kl_loss: io_dtype must be fp16 or bf16");
  if (!is16(w_dtype) && w_dtype != DSA_DTYPE_F32)
    return fail(DSA_ERR_INVALID, "dsa_sli_grad_kl_loss: weights dtype must be fp16, bf16 or fp32");
  if (batch <= 0 || s1 < 0 || s2 <= 0 || n1 <= 0 || sparse_count <= 0)
    return fail(DSA_ERR_INVALID, "dsa_sli_grad_kl_loss: non-positive shape");
  if (n1 > 128) return fail(DSA_ERR_UNSUPPORTED, "dsa_sli_grad_kl_loss: N1=%d > 128", n1);
  if (dr != 0 && dr != 64) return fail(DSA_ERR_INVALID, "rope dim must be 64 (or 0 without rope), got %d", dr);
  if (!sli_grad_supported(d, dr, nidx1, d_idx, sparse_count))
    return fail(DSA_ERR_UNSUPPORTED,
                "dsa_sli_grad_kl_loss: D=%d (+%d), Nidx1=%d, D_idx=%d, topK=%d outside D in {128,256,512}, "
                "D_idx in {128,256,512}, Nidx1 <= 128, topK <= 2048",
                d, dr, nidx1, d_idx, sparse_count);
  if (batch > 65535 || (int64_t)batch * s1 > INT32_MAX)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_sli_grad_kl_loss: too many rows");
  const size_t need = sli_grad_workspace_bytes(batch * s1, sparse_count, (int64_t)batch * s2, d_idx,
                                               sli_km_sparse_ld(batch * s1, sparse_count, s2, d_idx));
  if (workspace_bytes < need)
    return fail(DSA_ERR_INVALID, "dsa_sli_grad_kl_loss: workspace of %zu bytes required, %zu given", need,
                workspace_bytes);
  if (batch * s1 == 0) return DSA_OK;
  return hip_status(launch_sli_grad(query, key, query_rope ? query_rope : query, key_rope ? key_rope : key,
                                    query_index, key_index, weights, io_dtype, w_dtype, sparse_indices,
                                    sparse_count, sm_max, sm_sum, act_q, act_k, batch, s1, s2, n1, d, dr,
                                    nidx1, d_idx, scale, d_query_index, d_key_index, d_weights, loss,
                                    workspace, (hipStream_t)stream),
                    "dsa_sli_grad_kl_loss launch");
}

size_t dsa_dense_li_grad_workspace_bytes(int batch, int s1, int s2, int d_idx) {
  if (batch <= 0 || s1 < 0 || s2 <= 0 || d_idx <= 0) return 0;
  return sli_grad_workspace_bytes(batch * s1, s2, (int64_t)batch * s2, d_idx, 0);
}

int dsa_dense_li_softmax_lse(const void* query_index, const void* key_index, const void* weights, int io_dtype,
                             int w_dtype, const int32_t* act_q, const int32_t* act_k, int batch, int s1, int s2,
                             int nidx1, int d_idx, float* softmax_max_index, float* softmax_sum_index,
                             void* stream) {
  if (!query_index || !key_index || !weights || !act_q || !act_k || !softmax_max_index || !softmax_sum_index)
    return fail(DSA_ERR_INVALID, "dsa_dense_li_softmax_lse: null pointer argument");
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "dsa_dense_li_softmax_lse: io_dtype must be fp16 or bf16");
  if (!is16(w_dtype) && w_dtype != DSA_DTYPE_F32)
    return fail(DSA_ERR_INVALID, "dsa_dense_li_softmax_lse: weights dtype must be fp16, bf16 or fp32");
  if (batch <= 0 || s1 < 0 || s2 <= 0) return fail(DSA_ERR_INVALID, "dsa_dense_li_softmax_lse: non-positive shape");
  if (!dense_li_grad_supported(1, 1, 128, 0, nidx1, d_idx, s2))
    return fail(DSA_ERR_UNSUPPORTED,
                "dsa_dense_li_softmax_lse: Nidx1=%d, D_idx=%d outside D_idx in {128,256,512}, Nidx1 <= 128",
                nidx1, d_idx);
  if (batch > 65535 || (int64_t)batch * s1 > INT32_MAX)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_dense_li_softmax_lse: too many rows");
  if (batch * s1 == 0) return DSA_OK;
  return hip_status(launch_dense_li_lse(query_index, key_index, weights, io_dtype, w_dtype, act_q, act_k, batch,
                                        s1, s2, nidx1, d_idx, softmax_max_index, softmax_sum_index,
                                        (hipStream_t)stream),
                    "dsa_dense_li_softmax_lse launch");
}

int dsa_dense_li_grad_kl_loss(const void* query, const void* key, const void* query_rope, const void* key_rope,
                              const void* query_index, const void* key_index, const void* weights, int io_dtype,
                              int w_dtype, const float* sm_max, const float* sm_sum, const float* max_index,
                              const float* sum_index, const int32_t* act_q, const int32_t* act_k, int batch,
                              int s1, int s2, int n1, int n2, int d, int dr, int nidx1, int d_idx, float scale,
                              void* d_query_index, void* d_key_index, void* d_weights, float* loss,
                              void* workspace, size_t workspace_bytes, void* stream) {
  if (!query || !key || !query_index || !key_index || !weights || !sm_max || !sm_sum || !act_q || !act_k ||
      !d_query_index || !d_key_index || !d_weights || !loss || !workspace ||
      (dr > 0 && (!query_rope || !key_rope)) || (!max_index != !sum_index))
    return fail(DSA_ERR_INVALID, "dsa_dense_li_grad_kl_loss: null pointer argument");
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "dsa_dense_li_grad_kl_loss: io_dtype must be fp16 or bf16");
  if (!is16(w_dtype) && w_dtype != DSA_DTYPE_F32)
    return fail(DSA_ERR_INVALID, "dsa_dense_li_grad_kl_loss: weights dtype must be fp16, bf16 or fp32");
  if (batch <= 0 || s1 < 0 || s2 <= 0 || n1 <= 0 || n2 <= 0)
    return fail(DSA_ERR_INVALID, "dsa_dense_li_grad_kl_loss: non-positive shape");
  if (n1 % n2 != 0) return fail(DSA_ERR_INVALID, "dsa_dense_li_grad_kl_loss: N1=%d not divisible by N2=%d", n1, n2);
  if (n1 > 128) return fail(DSA_ERR_UNSUPPORTED, "dsa_dense_li_grad_kl_loss: N1=%d > 128", n1);
  if (dr != 0 && dr != 64) return fail(DSA_ERR_INVALID, "rope dim must be 64 (or 0 without rope), got %d", dr);
  if (!dense_li_grad_supported(n1, n2, d, dr, nidx1, d_idx, s2))
    return fail(DSA_ERR_UNSUPPORTED,
                "dsa_dense_li_grad_kl_loss: D=%d (+%d), N1=%d, N2=%d, Nidx1=%d, D_idx=%d outside D, D_idx in "
                "{128,256,512}, Nidx1 <= 128", d, dr, n1, n2, nidx1, d_idx);
  if (batch > 65535 || (int64_t)batch * s1 > INT32_MAX)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_dense_li_grad_kl_loss: too many rows");
  const size_t need = sli_grad_workspace_bytes(batch * s1, s2, (int64_t)batch * s2, d_idx, 0);
  if (workspace_bytes < need)
    return fail(DSA_ERR_INVALID, "dsa_dense_li_grad_kl_loss: workspace of %zu bytes required, %zu given", need,
                workspace_bytes);
  if (batch * s1 == 0) return DSA_OK;
  return hip_status(launch_dense_li_grad(query, key, query_rope ? query_rope : query, key_rope ? key_rope : key,
                                         query_index, key_index, weights, io_dtype, w_dtype, sm_max, sm_sum,
                                         max_index, sum_index, act_q, act_k, batch, s1, s2, n1, n2, d, dr, nidx1,
                                         d_idx, scale, d_query_index, d_key_index, d_weights, loss, workspace,
                                         (hipStream_t)stream),
                    "dsa_dense_li_grad_kl_loss launch");
}

namespace {
// Positions, sections and rotary dimensions, shared by the rotation and the appends
int check_rotation(const char* fn, int axes, const int32_t* sections, const float* inv_freq, int rotary_start,
                   int rotary_dim, int width) {
  if (!inv_freq) return fail(DSA_ERR_INVALID, "%s: null pointer argument", fn);
  if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > 1024 || rotary_start < 0 || rotary_start + rotary_dim > width)
    return fail(DSA_ERR_INVALID, "%s: rotary dimensions [%d, %d + %d) of a width of %d (an even count, at most 1024)", fn,
                rotary_start, rotary_start, rotary_dim, width);
  if (axes < 1 || axes > 4) return fail(DSA_ERR_INVALID, "%s: 1 to 4 position axes, got %d", fn, axes);
  if (axes > 1 && !sections) return fail(DSA_ERR_INVALID, "%s: several axes need sections", fn);
  if (sections) {
    int64_t sum = 0;
    for (int a = 0; a < axes; ++a) {
      if (sections[a] < 0) return fail(DSA_ERR_INVALID, "%s: negative section", fn);
      sum += sections[a];
    }
    if (sum != rotary_dim / 2)
      return fail(DSA_ERR_INVALID, "%s: sections add up to %lld, not to the %d pairs", fn, (long long)sum, rotary_dim / 2);
  }
  return DSA_OK;
}

int check_append(const char* fn, const void* x, int io_dtype, const void* norm_weight, int w_dtype,
                 const int32_t* row_start, const int32_t* act_q, const int32_t* act_k, int lengths_host,
                 const int32_t* block_table, int batch, int total_rows, int rows_per_batch, int max_blocks, int page_block_size, int64_t num_blocks,
                 const void* cache) {
  if (!x || !row_start || !act_q || !act_k || !block_table || !cache)
    return fail(DSA_ERR_INVALID, "%s: null pointer argument", fn);
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "%s: io_dtype must be fp16 or bf16", fn);
  if (norm_weight && !is16(w_dtype) && w_dtype != DSA_DTYPE_F32)
    return fail(DSA_ERR_INVALID, "%s: norm weights must be fp16, bf16 or fp32", fn);
  if (batch <= 0 || total_rows < 0 || rows_per_batch < 1 || max_blocks <= 0 || page_block_size <= 0 || num_blocks <= 0)
    return fail(DSA_ERR_INVALID, "%s: non-positive shape", fn);
  if (total_rows > INT_MAX - 4096) return fail(DSA_ERR_UNSUPPORTED, "%s: %d rows, 2^31 - 4096 or more", fn, total_rows);
  if (((uintptr_t)cache & 15) != 0) return fail(DSA_ERR_INVALID, "%s: caches must be 16-byte aligned", fn);
  if (lengths_host && batch > (APPEND_ARG_LENGTHS - 1) / 3)
    return fail(DSA_ERR_UNSUPPORTED, "%s: host lengths of at most %d sequences, got %d", fn, (APPEND_ARG_LENGTHS - 1) / 3, batch);
  return DSA_OK;
}
}  // namespace

int dsa_rotary(const void* x, int64_t batch_stride, int64_t row_stride, int64_t head_stride, int dtype,
               const void* positions, int positions_64, int axes, const int32_t* sections, const float* inv_freq,
               int rows, int rows_per_batch, int heads, int width, int rotary_start, int rotary_dim, int interleaved,
               int inverse, void* out, void* stream) {
  if (!x || !positions || !out) return fail(DSA_ERR_INVALID, "dsa_rotary: null pointer argument");
  if (!is16(dtype) && dtype != DSA_DTYPE_F32) return fail(DSA_ERR_INVALID, "dsa_rotary: dtype must be fp16, bf16 or fp32");
  if (rows < 0 || rows_per_batch < 1 || heads <= 0 || width <= 0)
    return fail(DSA_ERR_INVALID, "dsa_rotary: non-positive shape");
  const int st = check_rotation("dsa_rotary", axes, sections, inv_freq, rotary_start, rotary_dim, width);
  if (st != DSA_OK) return st;
  if (width > 4096 || (int64_t)heads * width > (1 << 20))
    return fail(DSA_ERR_UNSUPPORTED, "dsa_rotary: width %d > 4096, or heads * width > 2^20", width);
  if (rows > INT_MAX - 4096) return fail(DSA_ERR_UNSUPPORTED, "dsa_rotary: %d rows, 2^31 - 4096 or more", rows);
  if (rows == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  RotaryArgs a{x, batch_stride, row_stride, head_stride, dtype, positions, positions_64, axes, sections, inv_freq, rows,
               rows_per_batch, heads, width, rotary_start, rotary_dim, interleaved, inverse, out};
  return hip_status(launch_rotary(a, (hipStream_t)stream), "dsa_rotary launch");
}

int dsa_row_positions(const int32_t* row_start, int batch, int rows, int32_t* positions, void* stream) {
  if (!row_start || !positions) return fail(DSA_ERR_INVALID, "dsa_row_positions: null pointer argument");
  if (batch <= 0 || rows < 0) return fail(DSA_ERR_INVALID, "dsa_row_positions: non-positive shape");
  if (rows == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  return hip_status(launch_row_positions(row_start, batch, rows, positions, (hipStream_t)stream), "dsa_row_positions launch");
}

int dsa_latent_append(const void* latent, int64_t batch_stride, int64_t row_stride, const void* key_rope,
                      int64_t rope_batch_stride, int64_t rope_row_stride, int io_dtype, int d, const void* norm_weight,
                      int w_dtype, float eps, const void* positions, int positions_64, int axes, const int32_t* sections,
                      const float* inv_freq, int interleaved, const int32_t* row_start, const int32_t* act_q,
                      const int32_t* act_k, int lengths_host, const int32_t* block_table, int batch, int total_rows,
                      int rows_per_batch, int max_blocks, int page_block_size, int64_t num_blocks, void* key_cache, void* key_rope_cache,
                      void* stream) {
  int st = check_append("dsa_latent_append", latent, io_dtype, norm_weight, w_dtype, row_start, act_q, act_k,
                        lengths_host, block_table, batch, total_rows, rows_per_batch, max_blocks, page_block_size, num_blocks, key_cache);
  if (st != DSA_OK) return st;
  if (!key_rope || !key_rope_cache) return fail(DSA_ERR_INVALID, "dsa_latent_append: null pointer argument");
  if (((uintptr_t)key_rope_cache & 15) != 0)
    return fail(DSA_ERR_INVALID, "dsa_latent_append: caches must be 16-byte aligned");
  if (d != 128 && d != 256 && d != 512) return fail(DSA_ERR_INVALID, "D must be one of (128, 256, 512), got %d", d);
  st = check_rotation("dsa_latent_append", axes, sections, inv_freq, 0, 64, 64);
  if (st != DSA_OK) return st;
  if (total_rows == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  AppendArgs a{latent, batch_stride, row_stride, 0, io_dtype, 1, d, key_rope, rope_batch_stride, rope_row_stride,
               norm_weight ? 1 : 0, norm_weight, nullptr, w_dtype, eps, positions, positions_64, axes, sections, inv_freq,
               0, 64, interleaved, row_start, act_q, act_k, lengths_host, block_table, batch, total_rows,
               rows_per_batch, max_blocks, page_block_size, num_blocks, key_cache, key_rope_cache};
  return hip_status(launch_cache_append(a, (hipStream_t)stream), "dsa_latent_append launch");
}

int dsa_index_append(const void* index_key, int64_t batch_stride, int64_t row_stride, int64_t head_stride, int io_dtype,
                     int n2, int w, const void* norm_weight, const void* norm_bias, int w_dtype, float eps,
                     const void* positions, int positions_64, int axes, const int32_t* sections, const float* inv_freq,
                     int rotary_start, int rotary_dim, int interleaved, const int32_t* row_start, const int32_t* act_q,
                     const int32_t* act_k, int lengths_host, const int32_t* block_table, int batch, int total_rows,
                     int rows_per_batch, int max_blocks, int page_block_size, int64_t num_blocks, void* index_cache, void* stream) {
  int st = check_append("dsa_index_append", index_key, io_dtype, norm_weight, w_dtype, row_start, act_q, act_k,
                        lengths_host, block_table, batch, total_rows, rows_per_batch, max_blocks, page_block_size, num_blocks, index_cache);
  if (st != DSA_OK) return st;
  if (n2 <= 0 || n2 > 65535) return fail(DSA_ERR_INVALID, "dsa_index_append: 1 to 65535 key heads, got %d", n2);
  if (!li_score_supported_d(w))
    return fail(DSA_ERR_UNSUPPORTED, "dsa_index_append: D=%d not in {64, 96, 128, 256, 512}", w);
  if (norm_bias && !norm_weight) return fail(DSA_ERR_INVALID, "dsa_index_append: norm_bias without norm_weight");
  st = check_rotation("dsa_index_append", axes, sections, inv_freq, rotary_start, rotary_dim, w);
  if (st != DSA_OK) return st;
  if (rotary_start % 8 != 0 || rotary_dim % 16 != 0)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_index_append: rotary_start %d is no multiple of 8, or rotary_dim %d of 16",
                rotary_start, rotary_dim);
  if (total_rows == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  AppendArgs a{index_key, batch_stride, row_stride, head_stride, io_dtype, n2, w, nullptr, 0, 0, norm_weight ? 2 : 0,
               norm_weight, norm_bias, w_dtype, eps, positions, positions_64, axes, sections, inv_freq, rotary_start,
               rotary_dim, interleaved, row_start, act_q, act_k, lengths_host, block_table, batch, total_rows, rows_per_batch,
               max_blocks, page_block_size, num_blocks, index_cache, nullptr};
  return hip_status(launch_cache_append(a, (hipStream_t)stream), "dsa_index_append launch");
}

size_t dsa_prefix_attn_workspace_bytes(int batch, int total_rows, int n1, int d, int prefix, int max_rows_per_batch,
                                       int max_kv, int64_t total_kv, int kv_splits) {
  if (batch <= 0 || total_rows <= 0 || n1 <= 0 || d <= 0 || prefix < 0 || max_rows_per_batch < 0 || max_kv < 0 || total_kv < 0)
    return 0;
  return prefix_attn_workspace_bytes(batch, total_rows, n1, d, prefix, max_rows_per_batch, max_kv, total_kv, kv_splits);
}

int dsa_prefix_attn(const void* query, const void* query_rope, const void* key, const void* key_rope, int io_dtype,
                    const int32_t* block_table, int max_blocks, int page_block_size, int64_t num_blocks,
                    const int32_t* row_start, const int32_t* act_q, const int32_t* act_k, int batch, int total_rows,
                    int n1, int d, int dr, int prefix, int max_rows_per_batch, int max_kv, int64_t total_kv, int sparse_mode,
                    float scale, void* out, float* sm_max, float* sm_sum, void* workspace, size_t workspace_bytes, int kv_splits,
                    void* stream) {
  if (!query || !query_rope || !key || !key_rope || !block_table || !row_start || !act_q || !act_k || !out)
    return fail(DSA_ERR_INVALID, "dsa_prefix_attn: null pointer argument");
  if (!is16(io_dtype)) return fail(DSA_ERR_INVALID, "dsa_prefix_attn: io_dtype must be fp16 or bf16");
  if (sparse_mode != 0 && sparse_mode != 3)
    return fail(DSA_ERR_INVALID, "Only sparse_mode 0 (full) / 3 (rightDownCausal) supported");
  if (d != 128 && d != 256 && d != 512) return fail(DSA_ERR_INVALID, "D must be one of (128, 256, 512), got %d", d);
  if (dr != 64) return fail(DSA_ERR_INVALID, "rope dim must be 64, got %d", dr);
  if (n1 < 1 || n1 > 128 || (n1 & (n1 - 1)) != 0)
    return fail(DSA_ERR_INVALID, "N1 must be one of (1, 2, 4, 8, 16, 32, 64, 128), got %d", n1);
  if (batch <= 0 || total_rows < 0 || max_blocks <= 0 || page_block_size <= 0 || num_blocks <= 0 || prefix < 0 ||
      max_rows_per_batch < 0 || max_kv < 0 || total_kv < 0)
    return fail(DSA_ERR_INVALID, "dsa_prefix_attn: non-positive shape");
  const int64_t s2 = (int64_t)max_blocks * page_block_size;
  if (prefix > s2 || max_kv > s2)
    return fail(DSA_ERR_INVALID, "dsa_prefix_attn: prefix or max_kv past the %lld tokens of a block-table row", (long long)s2);
  if (s2 > INT_MAX - 4096 || num_blocks > INT_MAX / page_block_size || (int64_t)total_rows * n1 > INT_MAX - 4096)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_prefix_attn: 2^31 tokens, cache rows or head rows");
  // (the join has a work-group of 256 threads for 32 head rows, and a launch fewer than 2^32 threads)
  if ((int64_t)total_rows * n1 > (1 << 29) - 32) return fail(DSA_ERR_UNSUPPORTED, "dsa_prefix_attn: 2^29 head rows");
  if ((((uintptr_t)query | (uintptr_t)query_rope | (uintptr_t)key | (uintptr_t)key_rope | (uintptr_t)out) & 15) != 0)
    return fail(DSA_ERR_INVALID, "dsa_prefix_attn: tensors must be 16-byte aligned");
  if ((sm_max == nullptr) != (sm_sum == nullptr))
    return fail(DSA_ERR_INVALID, "dsa_prefix_attn: sm_max and sm_sum must both be given or both NULL");
  if (kv_splits > 64) return fail(DSA_ERR_UNSUPPORTED, "dsa_prefix_attn: kv_splits=%d > 64", kv_splits);
  if (total_rows == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  PrefixArgs a{query, query_rope, key, key_rope, io_dtype, block_table, max_blocks, page_block_size, num_blocks, row_start,
               act_q, act_k, batch, total_rows, n1, d, prefix, max_rows_per_batch, max_kv, total_kv, sparse_mode, scale, out, sm_max,
               sm_sum, workspace, workspace_bytes, kv_splits};
  size_t lacking = 0;
  const hipError_t e = launch_prefix_attn(a, &lacking, (hipStream_t)stream);
  if (lacking > 0)
    return fail(DSA_ERR_INVALID, "dsa_prefix_attn: a 16-byte aligned workspace of %zu bytes required, %zu given", lacking,
                workspace ? workspace_bytes : (size_t)0);
  return hip_status(e, "dsa_prefix_attn launch");
}

namespace {
int check_norm(const char* fn, const void* x, int64_t row_stride, int dtype, int64_t rows, int width, const void* w, int w_dtype) {
  if (!x) return fail(DSA_ERR_INVALID, "%s: null pointer argument", fn);
  if (!is16(dtype) && dtype != DSA_DTYPE_F32) return fail(DSA_ERR_INVALID, "%s: dtype must be fp16, bf16 or fp32", fn);
  if (w && !is16(w_dtype) && w_dtype != DSA_DTYPE_F32)
    return fail(DSA_ERR_INVALID, "%s: norm weights must be fp16, bf16 or fp32", fn);
  if (rows < 0 || width <= 0) return fail(DSA_ERR_INVALID, "%s: non-positive shape", fn);
  if (width > DSA_NORM_MAX_WIDTH) return fail(DSA_ERR_UNSUPPORTED, "%s: width %d > %d", fn, width, DSA_NORM_MAX_WIDTH);
  if (rows > INT64_MAX / 8 / width || row_stride < 0 || (rows > 1 && row_stride > INT64_MAX / 8 / rows))
    return fail(DSA_ERR_UNSUPPORTED, "%s: rows or strides past 64 bits of bytes", fn);
  return DSA_OK;
}
}  // namespace

int dsa_layer_norm(const void* x, int64_t row_stride, int dtype, int64_t rows, int width, const void* norm_weight,
                   const void* norm_bias, int w_dtype, float eps, void* y, float* mean, float* rstd, void* stream) {
  const int st = check_norm("dsa_layer_norm", x, row_stride, dtype, rows, width, norm_weight, w_dtype);
  if (st != DSA_OK) return st;
  if (!y) return fail(DSA_ERR_INVALID, "dsa_layer_norm: null pointer argument");
  if (norm_bias && !norm_weight) return fail(DSA_ERR_INVALID, "dsa_layer_norm: norm_bias without norm_weight");
  if ((mean == nullptr) != (rstd == nullptr))
    return fail(DSA_ERR_INVALID, "dsa_layer_norm: mean and rstd must both be given or both NULL");
  if (rows == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  NormArgs a{};
  a.x = x, a.x_stride = row_stride, a.io = dtype, a.rows = rows, a.width = width, a.w = norm_weight, a.b = norm_bias;
  a.wdt = w_dtype, a.eps = eps, a.y = y, a.mean = mean, a.rstd = rstd;
  return hip_status(launch_layer_norm(a, (hipStream_t)stream), "dsa_layer_norm launch");
}

size_t dsa_layer_norm_grad_workspace_bytes(int64_t rows, int width) {
  if (rows <= 0 || width <= 0 || width > DSA_NORM_MAX_WIDTH) return 0;
  return layer_norm_grad_workspace_bytes(rows, width);
}

int dsa_layer_norm_grad(const void* d_out, int64_t d_row_stride, const void* x, int64_t row_stride, int dtype, int64_t rows,
                        int width, const float* mean, const float* rstd, const void* norm_weight, int w_dtype, void* d_x,
                        void* d_weight, void* d_bias, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_norm("dsa_layer_norm_grad", x, row_stride, dtype, rows, width, norm_weight, w_dtype);
  if (st != DSA_OK) return st;
  st = check_norm("dsa_layer_norm_grad", d_out, d_row_stride, dtype, rows, width, norm_weight, w_dtype);
  if (st != DSA_OK) return st;
  if (!mean || !rstd || !d_x) return fail(DSA_ERR_INVALID, "dsa_layer_norm_grad: null pointer argument");
  if ((d_weight || d_bias) && !norm_weight)
    return fail(DSA_ERR_INVALID, "dsa_layer_norm_grad: d_weight or d_bias without norm_weight");
  const size_t need = d_weight || d_bias ? dsa_layer_norm_grad_workspace_bytes(rows, width) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0))
    return fail(DSA_ERR_INVALID, "dsa_layer_norm_grad: a 16-byte aligned workspace of %zu bytes required, %zu given", need,
                workspace ? workspace_bytes : (size_t)0);
  if (rows == 0 && !d_weight && !d_bias) {
    g_err[0] = 0;
    return DSA_OK;
  }
  NormArgs a{};
  a.x = x, a.x_stride = row_stride, a.io = dtype, a.rows = rows, a.width = width, a.w = norm_weight, a.wdt = w_dtype;
  a.y = d_x, a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd), a.d = d_out, a.d_stride = d_row_stride;
  a.dw = d_weight, a.db = d_bias, a.part = (float*)workspace;
  return hip_status(launch_layer_norm_grad(a, (hipStream_t)stream), "dsa_layer_norm_grad launch");
}

namespace {
void set_batches(std::initializer_list<DenseTensor*> tensors, const int64_t* strides, DenseArgs& a) {
  for (DenseTensor* t : tensors) t->batch = *strides++;
  a.apart = 1;
}
int check_strides(const char* fn, const DenseTensor& t) {
  if (((uintptr_t)t.p & 15) != 0 || t.row % 8 != 0 || t.head % 8 != 0 || t.batch % 8 != 0)
    return fail(DSA_ERR_INVALID, "%s: sequences, rows and heads must begin on 16-byte borders", fn);
  if (t.row < 0 || t.head < 0 || t.batch < 0 || t.row >= (1 << 24) || t.head >= (1ll << 40) || t.batch >= (1ll << 45))
    return fail(DSA_ERR_UNSUPPORTED, "%s: row strides of 2^24 elements, or sequences 2^45 apart", fn);
  return DSA_OK;
}
int check_dense(const char* fn, const DenseArgs& a) {
  const bool rope = a.dr > 0;
  if (!a.q.p || !a.k.p || !a.v.p || (rope && (!a.qr.p || !a.kr.p)) || !a.row_start || !a.key_start || !a.act_q || !a.act_k)
    return fail(DSA_ERR_INVALID, "%s: null pointer argument", fn);
  if (!is16(a.io)) return fail(DSA_ERR_INVALID, "%s: io_dtype must be fp16 or bf16", fn);
  if (a.sparse_mode != 0 && a.sparse_mode != 3)
    return fail(DSA_ERR_INVALID, "Only sparse_mode 0 (full) / 3 (rightDownCausal) supported");
  if (a.d != 64 && a.d != 128) return fail(DSA_ERR_INVALID, "D must be one of (64, 128), got %d", a.d);
  if (a.dr != 0 && (a.dr != 64 || a.d != 128))
    return fail(DSA_ERR_INVALID, "rope dim must be 0, or 64 beside D = 128, got %d", a.dr);
  if (a.batch <= 0 || a.total_rows < 0 || a.total_keys < 0 || a.n1 <= 0 || a.n2 <= 0 || a.rows_behind < 0 || a.max_rows < 0 || a.max_kv < 0)
    return fail(DSA_ERR_INVALID, "%s: non-positive shape", fn);
  if (a.n1 % a.n2 != 0) return fail(DSA_ERR_INVALID, "%s: N1=%d not divisible by N2=%d", fn, a.n1, a.n2);
  if (a.rows_behind > a.total_rows || a.max_rows > a.total_rows || a.max_kv > a.total_keys)
    return fail(DSA_ERR_INVALID, "%s: rows_behind, max_rows or max_kv past the tensors' rows", fn);
  if (a.stat_padded && a.total_rows % a.batch != 0)
    return fail(DSA_ERR_INVALID, "%s: padded statistics of rows that do not split evenly", fn);
  if (a.apart && (!a.stat_padded || a.rows_behind != 0 || a.total_keys % a.batch != 0))
    return fail(DSA_ERR_INVALID, "%s: batch strides are for padded batches", fn);
  if ((int64_t)a.total_rows * a.n1 >= (1 << 30) || (int64_t)a.total_keys * a.n2 >= (1 << 30) || a.batch > 65535)
    return fail(DSA_ERR_UNSUPPORTED, "%s: 2^30 head rows, or more than 65535 sequences", fn);
  for (const DenseTensor* t : {&a.q, &a.qr, &a.k, &a.kr, &a.v}) {
    if (!rope && (t == &a.qr || t == &a.kr)) continue;
    const int st = check_strides(fn, *t);
    if (st != DSA_OK) return st;
  }
  return DSA_OK;
}
}  // namespace

size_t dsa_dense_attn_workspace_bytes(int batch, int total_rows, int rows_behind, int n1, int n2, int d, int max_rows, int max_kv,
                                      int kv_splits) {
  if (batch <= 0 || total_rows <= 0 || rows_behind < 0 || n1 <= 0 || n2 <= 0 || n1 % n2 != 0 || d <= 0 || max_rows < 0 || max_kv < 0)
    return 0;
  DenseArgs a{};
  a.batch = batch, a.total_rows = total_rows, a.rows_behind = rows_behind, a.n1 = n1, a.n2 = n2, a.d = d;
  a.max_rows = max_rows, a.max_kv = max_kv, a.kv_splits = kv_splits;
  a.sparse_mode = 0;   // either mask's
  const size_t full = dense_attn_workspace_bytes(a);
  a.sparse_mode = 3;
  return std::max(full, dense_attn_workspace_bytes(a));
}

int dsa_dense_attn_batched(const void* query, int64_t q_row, int64_t q_head, const void* query_rope, int64_t qr_row, int64_t qr_head,
                           const void* key, int64_t k_row, int64_t k_head, const void* key_rope, int64_t kr_row, int64_t kr_head,
                           const void* value, int64_t v_row, int64_t v_head, int io_dtype, const int32_t* row_start,
                           const int32_t* key_start, const int32_t* act_q, const int32_t* act_k, int batch, int total_rows,
                           int total_keys, int rows_behind, int n1, int n2, int d, int dr, int max_rows, int max_kv, int sparse_mode,
                           float scale, void* out, int stat_padded, float* sm_max, float* sm_sum, void* workspace,
                           size_t workspace_bytes, int kv_splits, const int64_t* batch_strides, void* stream) {
  DenseArgs a{};
  a.q = {query, q_row, q_head}, a.qr = {query_rope, qr_row, qr_head}, a.k = {key, k_row, k_head};
  a.kr = {key_rope, kr_row, kr_head}, a.v = {value, v_row, v_head}, a.io = io_dtype;
  a.row_start = row_start, a.key_start = key_start, a.act_q = act_q, a.act_k = act_k, a.batch = batch;
  a.total_rows = total_rows, a.total_keys = total_keys, a.rows_behind = rows_behind, a.n1 = n1, a.n2 = n2, a.d = d, a.dr = dr;
  a.max_rows = max_rows, a.max_kv = max_kv, a.sparse_mode = sparse_mode, a.scale = scale, a.out = out;
  a.stat_padded = stat_padded, a.sm_max = sm_max, a.sm_sum = sm_sum, a.ws = workspace, a.ws_bytes = workspace_bytes;
  a.kv_splits = kv_splits;
  if (batch_strides) set_batches({&a.q, &a.qr, &a.k, &a.kr, &a.v}, batch_strides, a);
  const int st = check_dense("dsa_dense_attn", a);
  if (st != DSA_OK) return st;
  if (!out) return fail(DSA_ERR_INVALID, "dsa_dense_attn: null pointer argument");
  if (((uintptr_t)out & 15) != 0) return fail(DSA_ERR_INVALID, "dsa_dense_attn: out must be 16-byte aligned");
  if ((sm_max == nullptr) != (sm_sum == nullptr))
    return fail(DSA_ERR_INVALID, "dsa_dense_attn: sm_max and sm_sum must both be given or both NULL");
  if (kv_splits > 64) return fail(DSA_ERR_UNSUPPORTED, "dsa_dense_attn: kv_splits=%d > 64", kv_splits);
  if (total_rows == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  size_t lacking = 0;
  const hipError_t e = launch_dense_attn(a, &lacking, (hipStream_t)stream);
  if (lacking > 0)
    return fail(DSA_ERR_INVALID, "dsa_dense_attn: a 16-byte aligned workspace of %zu bytes required, %zu given", lacking,
                workspace ? workspace_bytes : (size_t)0);
  if (e == hipErrorInvalidConfiguration)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_dense_attn: 2^32 threads in a launch (sequences times key heads, times kv_splits)");
  return hip_status(e, "dsa_dense_attn launch");
}

int dsa_dense_attn(const void* query, int64_t q_row, int64_t q_head, const void* query_rope, int64_t qr_row, int64_t qr_head,
                   const void* key, int64_t k_row, int64_t k_head, const void* key_rope, int64_t kr_row, int64_t kr_head,
                   const void* value, int64_t v_row, int64_t v_head, int io_dtype, const int32_t* row_start,
                   const int32_t* key_start, const int32_t* act_q, const int32_t* act_k, int batch, int total_rows,
                   int total_keys, int rows_behind, int n1, int n2, int d, int dr, int max_rows, int max_kv, int sparse_mode,
                   float scale, void* out, int stat_padded, float* sm_max, float* sm_sum, void* workspace,
                   size_t workspace_bytes, int kv_splits, void* stream) {
  return dsa_dense_attn_batched(query, q_row, q_head, query_rope, qr_row, qr_head, key, k_row, k_head, key_rope, kr_row,
                                kr_head, value, v_row, v_head, io_dtype, row_start, key_start, act_q, act_k, batch,
                                total_rows, total_keys, rows_behind, n1, n2, d, dr, max_rows, max_kv, sparse_mode, scale,
                                out, stat_padded, sm_max, sm_sum, workspace, workspace_bytes, kv_splits, nullptr, stream);
}

size_t dsa_dense_attn_grad_workspace_bytes(int batch, int total_rows, int total_keys, int rows_behind, int keys_behind, int n1,
                                           int n2, int d, int dr, int max_rows, int max_keys, int max_kv, int splits) {
  if (batch <= 0 || total_rows < 0 || total_keys < 0 || rows_behind < 0 || keys_behind < 0 || n1 <= 0 || n2 <= 0 || n1 % n2 != 0 ||
      d <= 0 || dr < 0 || max_rows < 0 || max_keys < 0 || max_kv < 0)
    return 0;
  DenseGradArgs g{};
  DenseArgs& a = g.f;
  a.batch = batch, a.total_rows = total_rows, a.total_keys = total_keys, a.rows_behind = rows_behind, a.n1 = n1, a.n2 = n2;
  a.d = d, a.dr = dr, a.max_rows = max_rows, a.max_kv = max_kv, a.kv_splits = splits, g.keys_behind = keys_behind, g.max_keys = max_keys;
  return dense_grad_workspace_bytes(g);
}

int dsa_dense_attn_grad_batched(const void* query, int64_t q_row, int64_t q_head, const void* query_rope, int64_t qr_row, int64_t qr_head,
                                const void* key, int64_t k_row, int64_t k_head, const void* key_rope, int64_t kr_row, int64_t kr_head,
                                const void* value, int64_t v_row, int64_t v_head, const void* d_out, int64_t d_row, int64_t d_head,
                                const void* out, int64_t o_row, int64_t o_head, int io_dtype, const int32_t* row_start,
                                const int32_t* key_start, const int32_t* act_q, const int32_t* act_k, int batch, int total_rows,
                                int total_keys, int rows_behind, int keys_behind, int n1, int n2, int d, int dr, int max_rows,
                                int max_keys, int max_kv, int sparse_mode, float scale, int stat_padded, const float* sm_max,
                                const float* sm_sum, void* d_query, void* d_query_rope, void* d_key, void* d_key_rope, void* d_value,
                                void* workspace, size_t workspace_bytes, int splits, const int64_t* batch_strides, void* stream) {
  static const char* fn = "dsa_dense_attn_grad";
  DenseGradArgs g{};
  DenseArgs& a = g.f;
  a.q = {query, q_row, q_head}, a.qr = {query_rope, qr_row, qr_head}, a.k = {key, k_row, k_head};
  a.kr = {key_rope, kr_row, kr_head}, a.v = {value, v_row, v_head}, a.io = io_dtype;
  a.row_start = row_start, a.key_start = key_start, a.act_q = act_q, a.act_k = act_k, a.batch = batch;
  a.total_rows = total_rows, a.total_keys = total_keys, a.rows_behind = rows_behind, a.n1 = n1, a.n2 = n2, a.d = d, a.dr = dr;
  a.max_rows = max_rows, a.max_kv = max_kv, a.sparse_mode = sparse_mode, a.scale = scale, a.stat_padded = stat_padded;
  a.sm_max = const_cast<float*>(sm_max), a.sm_sum = const_cast<float*>(sm_sum), a.ws = workspace, a.ws_bytes = workspace_bytes;
  a.kv_splits = splits, g.d_out = {d_out, d_row, d_head}, g.out = {out, o_row, o_head}, g.keys_behind = keys_behind;
  g.max_keys = max_keys, g.dq = d_query, g.dqr = d_query_rope, g.dk = d_key, g.dkr = d_key_rope, g.dv = d_value;
  if (batch_strides) set_batches({&a.q, &a.qr, &a.k, &a.kr, &a.v, &g.d_out, &g.out}, batch_strides, a);
  const int st = check_dense(fn, a);
  if (st != DSA_OK) return st;
  if (!d_out || !out || !sm_max || !sm_sum || !d_query || !d_key || !d_value || (dr > 0 && (!d_query_rope || !d_key_rope)))
    return fail(DSA_ERR_INVALID, "%s: null pointer argument", fn);
  for (const DenseTensor* t : {&g.d_out, &g.out}) {
    const int of = check_strides(fn, *t);
    if (of != DSA_OK) return of;
  }
  if (a.apart && keys_behind != 0) return fail(DSA_ERR_INVALID, "%s: batch strides are for padded batches", fn);
  if ((((uintptr_t)d_query | (uintptr_t)d_query_rope | (uintptr_t)d_key | (uintptr_t)d_key_rope | (uintptr_t)d_value) & 15) != 0)
    return fail(DSA_ERR_INVALID, "%s: outputs must be 16-byte aligned", fn);
  if (keys_behind < 0 || keys_behind > total_keys || max_keys < 0 || max_keys > total_keys)
    return fail(DSA_ERR_INVALID, "%s: keys_behind or max_keys past the tensors' rows", fn);
  if (splits > 64) return fail(DSA_ERR_UNSUPPORTED, "%s: splits=%d > 64", fn, splits);
  if (total_rows == 0 && total_keys == 0) {
    g_err[0] = 0;
    return DSA_OK;
  }
  size_t lacking = 0;
  const hipError_t e = launch_dense_grad(g, &lacking, (hipStream_t)stream);
  if (lacking > 0)
    return fail(DSA_ERR_INVALID, "%s: a 16-byte aligned workspace of %zu bytes required, %zu given", fn, lacking,
                workspace ? workspace_bytes : (size_t)0);
  if (e == hipErrorInvalidConfiguration)
    return fail(DSA_ERR_UNSUPPORTED, "dsa_dense_attn_grad: 2^32 threads in a launch (sequences times key heads, times splits)");
  return hip_status(e, "dsa_dense_attn_grad launch");
}

int dsa_dense_attn_grad(const void* query, int64_t q_row, int64_t q_head, const void* query_rope, int64_t qr_row, int64_t qr_head,
                        const void* key, int64_t k_row, int64_t k_head, const void* key_rope, int64_t kr_row, int64_t kr_head,
                        const void* value, int64_t v_row, int64_t v_head, const void* d_out, int64_t d_row, int64_t d_head,
                        const void* out, int64_t o_row, int64_t o_head, int io_dtype, const int32_t* row_start,
                        const int32_t* key_start, const int32_t* act_q, const int32_t* act_k, int batch, int total_rows,
                        int total_keys, int rows_behind, int keys_behind, int n1, int n2, int d, int dr, int max_rows,
                        int max_keys, int max_kv, int sparse_mode, float scale, int stat_padded, const float* sm_max,
                        const float* sm_sum, void* d_query, void* d_query_rope, void* d_key, void* d_key_rope, void* d_value,
                        void* workspace, size_t workspace_bytes, int splits, void* stream) {
  return dsa_dense_attn_grad_batched(query, q_row, q_head, query_rope, qr_row, qr_head, key, k_row, k_head, key_rope,
                                     kr_row, kr_head, value, v_row, v_head, d_out, d_row, d_head, out, o_row, o_head,
                                     io_dtype, row_start, key_start, act_q, act_k, batch, total_rows, total_keys,
                                     rows_behind, keys_behind, n1, n2, d, dr, max_rows, max_keys, max_kv, sparse_mode,
                                     scale, stat_padded, sm_max, sm_sum, d_query, d_query_rope, d_key, d_key_rope, d_value,
                                     workspace, workspace_bytes, splits, nullptr, stream);
}

}  // extern "C"
