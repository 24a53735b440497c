// extern "C" entry points of the transformer-layer operators around the depth
// read: argument checks and launches. Declared in include/attnres_b200.h.
#include <stdarg.h>
#include <stdio.h>

#include "common.cuh"
#include "kv4.h"
#include "plan.h"
#include "qkrope.h"
#include "swiglu.h"

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

// Runs a launch path; nothing it throws (its caches of device facts allocate) crosses the
// C boundary.
template <typename Launch>
int launched(Launch&& launch, const char* where) {
  cudaError_t e = cudaErrorMemoryAllocation;
  try {
    e = launch();
  } catch (...) {
  }
  if (e == cudaSuccess) return ATTNRES_OK;
  return fail(ATTNRES_ERR_CUDA, "%s: %s (%s)", where, cudaGetErrorName(e), cudaGetErrorString(e));
}

bool known_dtype(int dtype) {
  return dtype == ATTNRES_DTYPE_F32 || dtype == ATTNRES_DTYPE_F16 || dtype == ATTNRES_DTYPE_BF16;
}

// Whether dtype asks for fp32 norm weights beside 16-bit data (fp32 data has none other).
int weights_f32(int dtype) { return (dtype & ATTNRES_WEIGHTS_F32) && dtype != (ATTNRES_DTYPE_F32 | ATTNRES_WEIGHTS_F32); }

int check_qk_norm_rope(const attnres::QkRopeArgs& a, int dtype) {
  if (!known_dtype(dtype & ~ATTNRES_WEIGHTS_F32)) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
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
  if (a.N > ((1LL << 33) - 4) / (a.Hq + 2 * a.Hkv))  // blocks of four head rows
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

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_swiglu(int64_t n, int in_dim, int hidden, int dtype, const void* x, int64_t xs, const void* w, int64_t ws) {
  if (n < 0 || in_dim < 1 || hidden < 1)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "swiglu: num_tokens=%lld, in_dim=%d, hidden=%d must be positive",
                (long long)n, in_dim, hidden);
  if (!known_dtype(dtype)) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (dtype == ATTNRES_DTYPE_F32) return fail(ATTNRES_ERR_UNSUPPORTED, "swiglu: float16 and bfloat16 only");
  if (in_dim % 8 || hidden % 8 || hidden > (1 << 28))
    return fail(ATTNRES_ERR_UNSUPPORTED, "swiglu: in_dim=%d and hidden=%d must be multiples of 8", in_dim, hidden);
  // tiles of 256 rows x 64 or 128 columns of h, dx and dW are counted in 32 bits
  if (n > 0x7fffffffLL || in_dim > (1 << 28) || (n / 128 + 1) * (hidden / 128 + 1) > 0x7fffffffLL ||
      (n / 128 + 1) * (in_dim / 128 + 1) > 0x7fffffffLL || (hidden / 128LL + 1) * (in_dim / 128 + 1) > 0x7fffffffLL)
    return fail(ATTNRES_ERR_UNSUPPORTED, "swiglu: num_tokens=%lld is too many for one launch", (long long)n);
  if (xs < in_dim || ws < in_dim) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "swiglu: a row stride below in_dim");
  if (!w || (n > 0 && !x)) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "swiglu: x or weight is NULL");
  if (xs % 8 || ws % 8 || !aligned16(x) || !aligned16(w))
    return fail(ATTNRES_ERR_UNSUPPORTED, "swiglu: rows of x and weight must start on 16-byte boundaries");
  return ATTNRES_OK;
}

constexpr int kKv4MaxGrid = 65535;           // sequences, key heads: a grid's y and z
constexpr int64_t kKv4MaxPlaces = 1LL << 30;  // places of a sequence

bool too_many_query_rows(int batch, int new_tokens, int q_heads) {
  return static_cast<double>(batch) * new_tokens * q_heads > 0x3fffffff;
}

// The pool, the page table and the counts, as every cache entry takes them.
int check_kv4(const attnres::Kv4Cache& c, int max_pages, int64_t table_stride, int batch, int new_tokens) {
  if (c.pages < 0 || c.heads < 1 || c.page < 1 || c.D < 1 || max_pages < 0 || batch < 0 || new_tokens < 0)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "kv4 cache: a size is negative or zero");
  if (c.page % 16 || c.D % attnres::kKv4Group || c.D > attnres::kKv4MaxDim)
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 cache: page_size=%d must be a multiple of 16, head_dim=%d of 32 up to %d",
                c.page, c.D, attnres::kKv4MaxDim);
  if (batch > kKv4MaxGrid || c.heads > kKv4MaxGrid)
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 cache: batch=%d and kv_heads=%d up to %d", batch, c.heads, kKv4MaxGrid);
  if (static_cast<int64_t>(max_pages) * c.page > kKv4MaxPlaces)
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 cache: a sequence of %d pages of %d places is too long", max_pages, c.page);
  if (static_cast<double>(c.pages) * c.heads * (c.page / 16) > 0x7fffffff)
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 cache: a pool of %lld pages is too large", c.pages);
  if (table_stride < max_pages && batch > 1)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "kv4 cache: page_table_stride below max_pages");
  return ATTNRES_OK;
}

int check_kv4_buffers(const attnres::Kv4Cache& c, const int* table, int max_pages, const int* per_sequence) {
  if (c.pages > 0 && (!c.k_codes || !c.k_params || !c.v_codes || !c.v_params))
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "kv4 cache: a buffer of the pool is NULL");
  if (!per_sequence || (max_pages > 0 && !table))
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "kv4 cache: page_table, start or lengths is NULL");
  if (!aligned16(c.k_codes) || !aligned16(c.k_params) || !aligned16(c.v_codes) || !aligned16(c.v_params))
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 cache: the pool's buffers must start on 16-byte boundaries");
  return ATTNRES_OK;
}

attnres::Kv4Cache kv4_cache(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                            int64_t pages, int heads, int page, int D) {
  return {const_cast<void*>(k_codes), const_cast<void*>(k_params), const_cast<void*>(v_codes),
          const_cast<void*>(v_params), pages, heads, page, D};
}

// The kernels count groups of 32 elements in 32 bits.
int check_kv4_rows(const attnres::Kv4RowsArgs& a) {
  if (static_cast<double>(a.B) * a.T * a.c.heads * (a.c.D / 32) > 0x7fffffff)
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 cache: too many tokens for one launch");
  return ATTNRES_OK;
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
  a.w32 = weights_f32(dtype);
  dtype &= ~ATTNRES_WEIGHTS_F32;
  if (!q || !k || !v) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope: an output is NULL");
  a.out[0] = q;
  a.out[1] = k;
  a.out[2] = v;
  return launched([&] { return attnres::qkrope_launch(false, dtype, a, static_cast<cudaStream_t>(stream)); },
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
  a.w32 = weights_f32(dtype);
  dtype &= ~ATTNRES_WEIGHTS_F32;
  if ((grad_q_weight && !q_weight) || (grad_k_weight && !k_weight))
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "qk norm rope backward: a weight gradient without its weight");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (num_tokens == 0) {
    const size_t bytes = static_cast<size_t>(head_dim) * (dtype == ATTNRES_DTYPE_F32 || a.w32 ? 4 : 2);
    cudaError_t e = cudaSuccess;
    if (grad_q_weight) e = cudaMemsetAsync(grad_q_weight, 0, bytes, st);
    if (grad_k_weight && e == cudaSuccess) e = cudaMemsetAsync(grad_k_weight, 0, bytes, st);
    return launched([&] { return e; }, "attnres_qk_norm_rope_backward memset");
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
  return launched([&] { return attnres::qkrope_launch(true, dtype, a, st); },
                  "attnres_qk_norm_rope_backward launch");
}

int attnres_swiglu_forward(int64_t num_tokens, int in_dim, int hidden, int dtype, const void* x, int64_t x_row_stride,
                           const void* weight, int64_t weight_row_stride, void* h, void* stream) {
  int rc = check_swiglu(num_tokens, in_dim, hidden, dtype, x, x_row_stride, weight, weight_row_stride);
  if (rc || num_tokens == 0) return rc;
  if (!h) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "swiglu: h is NULL");
  if (!aligned16(h)) return fail(ATTNRES_ERR_UNSUPPORTED, "swiglu: h must start on a 16-byte boundary");
  attnres::SwigluArgs a{};
  a.N = num_tokens;
  a.C = in_dim;
  a.F = hidden;
  a.x = x;
  a.w = weight;
  a.x_stride = x_row_stride;
  a.w_stride = weight_row_stride;
  a.out = h;
  return launched([&] { return attnres::swiglu_launch(false, dtype, a, static_cast<cudaStream_t>(stream)); },
                  "attnres_swiglu_forward launch");
}

size_t attnres_swiglu_backward_workspace_bytes(int64_t num_tokens, int hidden) {
  return num_tokens < 1 || hidden < 1 ? 0 : static_cast<size_t>(num_tokens) * 4 * hidden;
}

int attnres_swiglu_backward(int64_t num_tokens, int in_dim, int hidden, int dtype, const void* x, int64_t x_row_stride,
                            const void* weight, int64_t weight_row_stride, const void* grad_h,
                            int64_t grad_h_row_stride, void* grad_x, void* grad_weight, void* workspace,
                            size_t workspace_bytes, void* stream) {
  int rc = check_swiglu(num_tokens, in_dim, hidden, dtype, x, x_row_stride, weight, weight_row_stride);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (num_tokens == 0)
    return launched(
        [&] {
          return grad_weight ? cudaMemsetAsync(grad_weight, 0, static_cast<size_t>(hidden) * in_dim * 4, st) : cudaSuccess;
        },
        "attnres_swiglu_backward memset");
  if (!grad_x && !grad_weight) return ATTNRES_OK;
  if (!grad_h) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "swiglu backward: grad_h is NULL");
  if (grad_h_row_stride < hidden)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "swiglu backward: grad_h_row_stride below hidden");
  if (grad_h_row_stride % 8 || !aligned16(grad_h) || !aligned16(grad_x) || !aligned16(grad_weight) ||
      !aligned16(workspace))
    return fail(ATTNRES_ERR_UNSUPPORTED, "swiglu backward: buffers and rows must start on 16-byte boundaries");
  const size_t need = attnres_swiglu_backward_workspace_bytes(num_tokens, hidden);
  if (!workspace || workspace_bytes < need)
    return fail(ATTNRES_ERR_WORKSPACE, "swiglu backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  attnres::SwigluArgs a{};
  a.N = num_tokens;
  a.C = in_dim;
  a.F = hidden;
  a.x = x;
  a.w = weight;
  a.x_stride = x_row_stride;
  a.w_stride = weight_row_stride;
  a.dh = grad_h;
  a.dh_stride = grad_h_row_stride;
  a.dx = grad_x;
  a.dw = grad_weight;
  a.workspace = workspace;
  return launched([&] { return attnres::swiglu_launch(true, dtype, a, st); },
                  "attnres_swiglu_backward launch");
}

int attnres_kv4_append(void* k_codes, void* k_params, void* v_codes, void* v_params, int64_t num_pages, int kv_heads,
                       int page_size, int head_dim, const int* page_table, int64_t page_table_stride, int max_pages,
                       const int* start, const int* counts, int batch, int new_tokens, int dtype, const void* k,
                       const int64_t* k_strides, const void* v, const int64_t* v_strides, void* stream) {
  attnres::Kv4RowsArgs a{};
  a.c = kv4_cache(k_codes, k_params, v_codes, v_params, num_pages, kv_heads, page_size, head_dim);
  int rc = check_kv4(a.c, max_pages, page_table_stride, batch, new_tokens);
  if (rc) return rc;
  if (!known_dtype(dtype)) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (batch == 0 || new_tokens == 0) return ATTNRES_OK;
  if ((rc = check_kv4_buffers(a.c, page_table, max_pages, start))) return rc;
  if (!k || !v || !k_strides || !v_strides) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "kv4 append: k or v is NULL");
  a.table = page_table;
  a.table_stride = page_table_stride;
  a.max_pages = max_pages;
  a.start = start;
  a.counts = counts;
  a.B = batch;
  a.T = new_tokens;
  a.k = k;
  a.v = v;
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = k_strides[i];
    a.vs[i] = v_strides[i];
  }
  if ((rc = check_kv4_rows(a))) return rc;
  return launched([&] { return attnres::kv4_append_launch(dtype, a, static_cast<cudaStream_t>(stream)); },
                  "attnres_kv4_append launch");
}

int attnres_kv4_read(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                     int64_t num_pages, int kv_heads, int page_size, int head_dim, const int* page_table,
                     int64_t page_table_stride, int max_pages, const int* start, const int* counts, int batch,
                     int new_tokens, int dtype, void* k, void* v, void* stream) {
  attnres::Kv4RowsArgs a{};
  a.c = kv4_cache(k_codes, k_params, v_codes, v_params, num_pages, kv_heads, page_size, head_dim);
  int rc = check_kv4(a.c, max_pages, page_table_stride, batch, new_tokens);
  if (rc) return rc;
  if (!known_dtype(dtype)) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (batch == 0 || new_tokens == 0) return ATTNRES_OK;
  if ((rc = check_kv4_buffers(a.c, page_table, max_pages, start))) return rc;
  if (!k || !v) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "kv4 read: k or v is NULL");
  if (!aligned16(k) || !aligned16(v))
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 read: k and v must start on 16-byte boundaries");
  a.table = page_table;
  a.table_stride = page_table_stride;
  a.max_pages = max_pages;
  a.start = start;
  a.counts = counts;
  a.B = batch;
  a.T = new_tokens;
  a.k_out = k;
  a.v_out = v;
  if ((rc = check_kv4_rows(a))) return rc;
  return launched([&] { return attnres::kv4_read_launch(dtype, a, static_cast<cudaStream_t>(stream)); },
                  "attnres_kv4_read launch");
}

size_t attnres_kv4_attention_workspace_bytes(int kv_heads, int page_size, int head_dim, int max_pages, int batch,
                                             int new_tokens, int q_heads) {
  if (kv_heads < 1 || page_size < 1 || head_dim < 1 || max_pages < 0 || batch < 1 || new_tokens < 1 || q_heads < kv_heads)
    return 0;
  // sizes that the call refuses: the plan's numbers would not hold them
  if (batch > kKv4MaxGrid || kv_heads > kKv4MaxGrid || static_cast<int64_t>(max_pages) * page_size > kKv4MaxPlaces ||
      too_many_query_rows(batch, new_tokens, q_heads))
    return 0;
  attnres::Kv4AttnArgs a{};
  a.c = kv4_cache(nullptr, nullptr, nullptr, nullptr, 0, kv_heads, page_size, head_dim);
  a.max_pages = max_pages;
  a.B = batch;
  a.T = new_tokens;
  a.Hq = q_heads;
  return attnres::kv4_attention_workspace_bytes(a);
}

int attnres_kv4_attention(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                          int64_t num_pages, int kv_heads, int page_size, int head_dim, const int* page_table,
                          int64_t page_table_stride, int max_pages, const int* lengths, const int* counts, int batch,
                          int new_tokens, int q_heads, int dtype, const void* q, const int64_t* q_strides, float scale,
                          void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  attnres::Kv4AttnArgs a{};
  a.c = kv4_cache(k_codes, k_params, v_codes, v_params, num_pages, kv_heads, page_size, head_dim);
  int rc = check_kv4(a.c, max_pages, page_table_stride, batch, new_tokens);
  if (rc) return rc;
  if (!known_dtype(dtype)) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (dtype == ATTNRES_DTYPE_F32) return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 attention: float16 and bfloat16 only");
  if (head_dim != 64 && head_dim != 128)
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 attention: head_dim=%d, 64 and 128 are built", head_dim);
  if (q_heads < 1 || q_heads % kv_heads)
    return fail(ATTNRES_ERR_INVALID_ARGUMENT, "kv4 attention: q_heads=%d must be a multiple of kv_heads=%d", q_heads,
                kv_heads);
  if (too_many_query_rows(batch, new_tokens, q_heads))
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 attention: too many query rows for one launch");
  if (batch == 0 || new_tokens == 0) return ATTNRES_OK;
  if ((rc = check_kv4_buffers(a.c, page_table, max_pages, lengths))) return rc;
  if (!q || !q_strides || !out) return fail(ATTNRES_ERR_INVALID_ARGUMENT, "kv4 attention: q or out is NULL");
  if (!aligned16(out) || !aligned16(workspace))
    return fail(ATTNRES_ERR_UNSUPPORTED, "kv4 attention: out and workspace must start on 16-byte boundaries");
  a.table = page_table;
  a.table_stride = page_table_stride;
  a.max_pages = max_pages;
  a.lengths = lengths;
  a.counts = counts;
  a.B = batch;
  a.T = new_tokens;
  a.Hq = q_heads;
  a.q = q;
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i];
  a.scale = scale;
  a.out = out;
  a.lse = lse;
  a.workspace = workspace;
  const size_t need = attnres::kv4_attention_workspace_bytes(a);
  if (need && (!workspace || workspace_bytes < need))
    return fail(ATTNRES_ERR_WORKSPACE, "kv4 attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  return launched([&] { return attnres::kv4_attention_launch(dtype, a, static_cast<cudaStream_t>(stream)); },
                  "attnres_kv4_attention launch");
}

}  // extern "C"
