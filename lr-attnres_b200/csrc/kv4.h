// Launch bundles and format of the 4-bit key/value cache (kv4_cache.cu, kv4_attn.cu).
//
// Groups of 32 elements of a head: element = low + step * code, code 0..15, step and
// low float16. G = head_dim / 32. Per page, kv head and place, for keys and values:
//   params  G pairs (step, low)
//   codes   head_dim / 2 bytes in the order in which the attention's lanes take them:
//           keys    word (c, g), c < 4, at byte 4 (c G + g): elements 32 g + 8 c + 0..7
//           values  half word (r, g), r < 8, at byte 2 (r G + g): elements 32 g + 4 r + 0..3
// the lower element in the lower bits.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace attnres {

constexpr int kKv4Group = 32;
constexpr int kKv4MaxDim = 512;

// Whether either half of a pair of params is an infinity or NaN.
__device__ __forceinline__ bool not_finite(uint32_t p) {
  return (p & 0x7c00u) == 0x7c00u || (p & 0x7c000000u) == 0x7c000000u;
}

struct Kv4Cache {
  void *k_codes, *k_params, *v_codes, *v_params;  // [pages, heads, page, D / 2], [pages, heads, page, G, 2]
  long long pages;
  int heads, page, D;
};

// Tokens 0 .. T of each of B sequences at places start[b] + t of its pages.
struct Kv4RowsArgs {
  Kv4Cache c;
  const int* table;  // [B, max_pages], rows table_stride apart
  long long table_stride;
  int max_pages;
  const int *start, *counts;  // [B]; counts null: T
  int B, T;
  const void *k, *v;     // append: [B, T, heads, D] with strides
  long long ks[3], vs[3];
  void *k_out, *v_out;   // read: dense
};

struct Kv4AttnArgs {
  Kv4Cache c;
  const int* table;
  long long table_stride;
  int max_pages;
  const int *lengths, *counts;  // [B]; counts null: T
  int B, T, Hq;
  const void* q;  // [B, T, Hq, D] with strides
  long long qs[3];
  float scale;
  void* out;   // [B, T, Hq, D]
  float* lse;  // [B, T, Hq] or null
  void* workspace;
};

cudaError_t kv4_append_launch(int dtype, const Kv4RowsArgs& a, cudaStream_t st);
cudaError_t kv4_read_launch(int dtype, const Kv4RowsArgs& a, cudaStream_t st);
cudaError_t kv4_attention_launch(int dtype, const Kv4AttnArgs& a, cudaStream_t st);
size_t kv4_attention_workspace_bytes(const Kv4AttnArgs& a);
cudaError_t read_kv4_status(unsigned* status, bool reset);
cudaError_t read_kv4_attn_status(unsigned* status, bool reset);

}  // namespace attnres
