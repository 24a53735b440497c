// extern "C" entry points of the transformer-layer operators around the depth
// read: argument checks and launches. Declared in include/attnres_b200.h.
#include <stdarg.h>
#include <stdio.h>

#include "common.cuh"
#include "plan.h"
#include "qkrope.h"

namespace {

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return attnres::record_error(code, buf);
}

int launched(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return ATTNRES_OK;
  return fail(ATTNRES_ERR_CUDA, "%s: %s (%s)", where, cudaGetErrorName(e), cudaGetErrorString(e));
}

bool known_dtype(int dtype) {
  return dtype == ATTNRES_DTYPE_F32 || dtype == ATTNRES_DTYPE_F16 || dtype == ATTNRES_DTYPE_BF16;
}

int check_qk_norm_rope(const attnres::QkRopeArgs& a, int dtype) {
  if (!known_dtype(dtype)) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (a.N < 0 || a.T < 1 || a.N % a.T)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope: num_tokens=%lld must be a multiple of seq_len=%lld", a.N, a.T);
  if (a.Hq < 1 || a.Hkv < 1 || a.D < 1 || a.Hq > 4096 || a.Hkv > 4096)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope: heads (%d, %d) in [1, 4096] and head_dim %d must be positive",
                a.Hq, a.Hkv, a.D);
  if (a.D > attnres::kRopeMaxDim)
    return fail(ATTNRES_ERR_UNSUPPORTED, "qk norm rope: head_dim=%d above %d", a.D, attnres::kRopeMaxDim);
  if (a.rot < 0 || a.rot > a.D || a.rot % 2)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope: rotary_dim=%d must be even and in [0, head_dim]", a.rot);
  if (a.qkv_stride < static_cast<long long>(a.Hq + 2 * a.Hkv) * a.D)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope: qkv_row_stride below (q_heads + 2 kv_heads) * head_dim");
  if (a.N > (1LL << 33) / (a.Hq + 2 * a.Hkv))
    return fail(ATTNRES_ERR_UNSUPPORTED, "qk norm rope: num_tokens=%lld is too many for one launch", a.N);
  if (a.N == 0) return ATTNRES_OK;
  if (!a.qkv) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope: qkv is NULL");
  if (a.rot > 0) {
    if (!a.cos || !a.sin) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope: a table is NULL");
    if (!a.positions && a.T > a.table_rows)
      return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope: seq_len=%lld exceeds the tables' %lld rows", a.T,
                  a.table_rows);
  }
  return ATTNRES_OK;
}

attnres::QkRopeArgs qk_rope_args(int64_t num_tokens, int64_t seq_len, int q_heads, int kv_heads, int head_dim,
                                 int rotary_dim, const void* qkv, int64_t qkv_row_stride, const float* cos,
                                 const float* sin, int64_t table_rows, const void* positions, int positions_are_64,
                                 const void* q_weight, const void* k_weight, int normalize, float eps,
                                 int interleaved) {
  attnres::QkRopeArgs a{};
  a.N = num_tokens;
  a.T = seq_len;
  a.Hq = q_heads;
  a.Hkv = kv_heads;
  a.D = head_dim;
  a.rot = rotary_dim;
  a.qkv = qkv;
  a.qkv_stride = qkv_row_stride;
  a.cos = cos;
  a.sin = sin;
  a.table_rows = table_rows;
  a.positions = positions;
  a.positions64 = positions_are_64;
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.normalize = normalize;
  a.interleaved = interleaved;
  a.eps = eps;
  a.inv_D = head_dim > 0 ? 1.f / head_dim : 0.f;
  return a;
}

}  // namespace

extern "C" {

int attnres_qk_norm_rope_forward(int64_t num_tokens, int64_t seq_len, int q_heads, int kv_heads, int head_dim,
                                 int rotary_dim, int dtype, const void* qkv, int64_t qkv_row_stride, const float* cos,
                                 const float* sin, int64_t table_rows, const void* positions, int positions_are_64,
                                 const void* q_weight, const void* k_weight, int normalize, float eps,
                                 int interleaved, void* q, void* k, void* v, void* stream) {
  attnres::QkRopeArgs a = qk_rope_args(num_tokens, seq_len, q_heads, kv_heads, head_dim, rotary_dim, qkv,
                                       qkv_row_stride, cos, sin, table_rows, positions, positions_are_64, q_weight,
                                       k_weight, normalize, eps, interleaved);
  int rc = check_qk_norm_rope(a, dtype);
  if (rc || num_tokens == 0) return rc;
  if (!q || !k || !v) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope: an output is NULL");
  a.out[0] = q;
  a.out[1] = k;
  a.out[2] = v;
  return launched(attnres::qkrope_launch(false, dtype, a, static_cast<cudaStream_t>(stream)),
                  "attnres_qk_norm_rope_forward launch");
}

size_t attnres_qk_norm_rope_backward_workspace_bytes(int head_dim) {
  if (head_dim < 1 || head_dim > attnres::kRopeMaxDim) return 0;
  return attnres::qkrope_workspace_bytes(head_dim);
}

int attnres_qk_norm_rope_backward(int64_t num_tokens, int64_t seq_len, int q_heads, int kv_heads, int head_dim,
                                  int rotary_dim, int dtype, const void* qkv, int64_t qkv_row_stride,
                                  const float* cos, const float* sin, int64_t table_rows, const void* positions,
                                  int positions_are_64, const void* q_weight, const void* k_weight, int normalize,
                                  float eps, int interleaved, const void* grad_q, const void* grad_k,
                                  const void* grad_v, const int64_t* grad_strides, void* grad_qkv,
                                  void* grad_q_weight, void* grad_k_weight, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  attnres::QkRopeArgs a = qk_rope_args(num_tokens, seq_len, q_heads, kv_heads, head_dim, rotary_dim, qkv,
                                       qkv_row_stride, cos, sin, table_rows, positions, positions_are_64, q_weight,
                                       k_weight, normalize, eps, interleaved);
  int rc = check_qk_norm_rope(a, dtype);
  if (rc) return rc;
  if ((grad_q_weight && !q_weight) || (grad_k_weight && !k_weight))
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope backward: a weight gradient without its weight");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (num_tokens == 0) {
    const size_t bytes = static_cast<size_t>(head_dim) * (dtype == ATTNRES_DTYPE_F32 ? 4 : 2);
    cudaError_t e = cudaSuccess;
    if (grad_q_weight) e = cudaMemsetAsync(grad_q_weight, 0, bytes, st);
    if (grad_k_weight && e == cudaSuccess) e = cudaMemsetAsync(grad_k_weight, 0, bytes, st);
    return launched(e, "attnres_qk_norm_rope_backward memset");
  }
  if (!grad_q || !grad_k || !grad_v || !grad_strides || !grad_qkv)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope backward: NULL gradient");
  const void* g[3] = {grad_q, grad_k, grad_v};
  for (int i = 0; i < 3; ++i) {
    a.g[i] = g[i];
    for (int j = 0; j < 3; ++j) a.gs[i][j] = grad_strides[3 * i + j];
  }
  a.dqkv = grad_qkv;
  a.dw[0] = grad_q_weight;
  a.dw[1] = grad_k_weight;
  if (grad_q_weight || grad_k_weight) {
    if (!workspace || workspace_bytes < attnres::qkrope_workspace_bytes(head_dim))
      return fail(ATTNRES_ERR_WORKSPACE, "qk norm rope backward: workspace of %zu bytes, %zu needed", workspace_bytes,
                  attnres::qkrope_workspace_bytes(head_dim));
    a.partials = static_cast<float*>(workspace);
  }
  return launched(attnres::qkrope_launch(true, dtype, a, st), "attnres_qk_norm_rope_backward launch");
}

}  // extern "C"
