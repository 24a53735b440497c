// Launch bundle of the q/k norm + rotation kernels (qkrope.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

namespace attnres {

constexpr int kRopeMaxDim = 512;

struct QkRopeArgs {
  long long N, T;  // token rows; tokens of a sequence (row n is token n % T of sequence n / T)
  int Hq, Hkv, D, rot;
  const void* qkv;  // [N, (Hq + 2 Hkv) D], row stride in elements
  long long qkv_stride;
  const float *cos, *sin;  // [table_rows, rot / 2]
  long long table_rows;
  const void* positions;  // [N] int32 / int64, or null: n % T
  int positions64;
  const void* w[2];  // q and k weights [D], or null
  int w32;           // weights and dw are fp32 beside 16-bit data
  int normalize, interleaved;
  float eps, inv_D;
  void* out[3];  // q [N, Hq, D], k, v [N, Hkv, D]
  // backward
  const void* g[3];     // dq, dk, dv
  long long gs[3][3];   // their strides: sequence, token, head
  void* dqkv;           // [N, (Hq + 2 Hkv) D] dense
  void* dw[2];          // [D] or null
  float* partials;      // [blocks][2][D] when a weight gradient is wanted
};

size_t qkrope_workspace_bytes(int D);
cudaError_t qkrope_launch(bool backward, int dtype, const QkRopeArgs& a, cudaStream_t st);

}  // namespace attnres
